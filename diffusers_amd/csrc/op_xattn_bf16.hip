// op_xattn_bf16.hip — cross attention on bf16_t.
#include "op_xattn_kernel.h"

void xa_forward_bf16(const OpCtx& c, const XaPlan& p, const XaDev& d) { xa_forward_type<bf16_t>(c, p, d); }
void xa_backward_bf16(const OpCtx& c, const XaPlan& p, const XaDev& d) { xa_backward_type<bf16_t>(c, p, d); }
