// op_xattn_f16.hip — cross attention on half_t.
#include "op_xattn_kernel.h"

void xa_forward_f16(const OpCtx& c, const XaPlan& p, const XaDev& d) { xa_forward_type<half_t>(c, p, d); }
void xa_backward_f16(const OpCtx& c, const XaPlan& p, const XaDev& d) { xa_backward_type<half_t>(c, p, d); }
