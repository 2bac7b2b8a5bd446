// op_xattn_f32.hip — cross attention on float.
#include "op_xattn_kernel.h"

void xa_forward_f32(const OpCtx& c, const XaPlan& p, const XaDev& d) { xa_forward_type<float>(c, p, d); }
void xa_backward_f32(const OpCtx& c, const XaPlan& p, const XaDev& d) { xa_backward_type<float>(c, p, d); }
