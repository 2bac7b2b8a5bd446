// op_gatedff_f16.hip — the gated feed-forward's products on half_t.
#include "op_gatedff_kernel.h"

void gff_launch_f16(const OpCtx& c, const GffDev& d, int what, int act, int cfg) { gff_launch_type<half_t>(c, d, what, act, cfg); }
