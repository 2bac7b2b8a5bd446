// op_gatedff_f32.hip — the gated feed-forward's products on float.
#include "op_gatedff_kernel.h"

void gff_launch_f32(const OpCtx& c, const GffDev& d, int what, int act, int cfg) { gff_launch_type<float>(c, d, what, act, cfg); }
