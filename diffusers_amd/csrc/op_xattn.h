// op_xattn.h — argument block, plan and launchers of cross attention.
#pragma once
#include "ops.h"

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kTile = 64;                       // keys (rows, for dk / dv) of a tile

struct Strided { const char* p; long long b, s, h; };       // bytes
struct XaDev {
    Strided q, k, v, o, dO, dq, dk, dv;
    const int* q_lens; const int* kv_lens; const unsigned char* mask; long long mask_b;
    float* lse; float* delta;                   // [B][Sq][H]
    float* part_o; float* part_ml;              // forward: [splits][B * Hkv][R][D16], [..][2];  dk / dv: part_o = [splits][2][B][Skv][Hkv][D]
    int B, Sq, Skv, H, Hkv, G, D, R;            // R = Sq * G rows of a key head
    int nrb, nkb, splits;
    int rpg;                                    // row blocks of a workgroup (resident kernels)
    int chunk;                                  // dk / dv: tiles of rows of a part
    int ragged;                                 // lengths are given: workgroups go to the XCDs in turn, so that one long sequence does not fill one XCD
    float scale, scale2;                        // scale2 = scale log2(e)
};


// kd: 64-byte steps of the head dimension, nd: 16-column steps of it; nw, qt: waves of a workgroup and 16-row groups of a wave; nrb: row blocks, rpg: of a workgroup that keeps all
// keys (0: they do not fit)
struct XaRows { int nw, qt, nrb, rpg; };
struct XaPlan { int kd, nd; XaRows fwd, dq; int splits, nkb, key_splits, chunk; };
// 16-key groups of a wave that owns keys: two while K, V and both gradients of 32 keys leave its registers room, one past that.  dk, dv, us, one / two groups, 4 sequences of 8 heads: fp16, 4096
// rows and keys, head size 32 253 / 224, 64 360 / 315; 2048 of 96 154 / 123, but with few keys, which leave few workgroups of twice the keys, 34 / 47 (1000 rows on 333); bf16 of 128
// spills.  fp32, 2048 of 32 285 / 284, of 64 555 / 525, but 48 / 59 (333 rows on 1000).
constexpr int xa_ktw(bool f32, int kd) { return f32 ? (kd >= 4 ? 1 : 2) : (kd >= 3 ? 1 : 2); }
// waves of a SIMD the registers are shared out for
constexpr int xa_waves(bool f32, int kd) { return kd >= (f32 ? 8 : 6) ? 1 : 2; }
// 16-row groups of a wave: two where q, o and the scores of 32 rows (dq: do too) fit into 256 registers of every type's kernel.  us, one / two groups, 4 sequences of 8 heads, 2048 rows and keys:
// forward fp16 64 (4096) 220 / 200, 96 93 / 72, bf16 128 116 / 88, fp16 160 133 / 222 (spills), fp32 64 295 / 284, 80 373 / 343 and equal with fewer rows; dq fp16 96 130 / 97, bf16 128 132 / 110,
// but fp16 128 142 / 167 (8 ragged sequences; spills), fp32 64 424 / 402, but 66 / 111 with 333 rows (half the workgroups).
constexpr int xa_qt(int kd, bool dq) { return kd >= (dq ? 4 : 5) ? 1 : 2; }
// Stages of a kernel whose stage holds two tiles (and `extra` bytes).  Two, unless they leave one workgroup to a CU where one stage leaves three (head size 160, fp16, dk / dv with dq 104 us with two
// stages, 87 with one), or do not fit at all (fp32 heads past 128).
constexpr int xa_stage(int kd, int extra) { return 2 * kTile * kd * 64 + extra; }
constexpr int stages_of(int kd, int extra)
{
    const int s = xa_stage(kd, extra), lds = 160 * 1024;
    return 4 * s <= lds ? 2 : 3 * s <= lds ? 1 : 2 * s <= lds - 1024 ? 2 : 1;
}
void xa_forward_f16(const OpCtx& c, const XaPlan& p, const XaDev& d);
void xa_forward_bf16(const OpCtx& c, const XaPlan& p, const XaDev& d);
void xa_forward_f32(const OpCtx& c, const XaPlan& p, const XaDev& d);
void xa_backward_f16(const OpCtx& c, const XaPlan& p, const XaDev& d);
void xa_backward_bf16(const OpCtx& c, const XaPlan& p, const XaDev& d);
void xa_backward_f32(const OpCtx& c, const XaPlan& p, const XaDev& d);
