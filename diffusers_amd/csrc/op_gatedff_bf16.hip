// op_gatedff_bf16.hip — the gated feed-forward's products on bf16_t.
#include "op_gatedff_kernel.h"

void gff_launch_bf16(const OpCtx& c, const GffDev& d, int what, int act, int cfg) { gff_launch_type<bf16_t>(c, d, what, act, cfg); }
