// op_gatedff.hip — the gated feed-forward block and its gradient as operators of their own.
//
//   a = x Wv^T + bv,  g = x Wg^T + bg,  h = a act(g)                           W = [Wv; Wg] is [2F][K], the value rows first
//   da = dh act(g),  dg = dh a act'(g):  dx = [da dg] W,  dW = [da dg]^T x,  db = column sums of [da dg]
//
// Three products on one tile kernel (op_gatedff_kernel.h): (1) x W^T with value and gate rows of the same columns in one tile, so that both projections, the
// activation and their product never leave the registers; (2) dx; (3) dW.  The backward pass forms a and g again instead of keeping
// them: 4 M K F operations against 4 M F values written by the forward pass and read back, and they stay in fp32.
#include "op_gatedff.h"
#include "ops_device.h"

#include <algorithm>

namespace {

// out[m][n] = sum over the splits, in their order
template <typename T> __global__ __launch_bounds__(256) void gff_join_kernel(const float* part, int splits, long long rows, int cols, T* out, long long ld)
{
    typedef typename VecOf<T, 4>::type T4;
    const long long total = rows * cols;
    for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4; i < total; i += (long long)gridDim.x * 1024) {
        floatx4 s = *(const floatx4*)(part + i);
        for (int k = 1; k < splits; ++k) s += *(const floatx4*)(part + k * total + i);
        const long long m = i / cols;
        T4 o;
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = (T)s[r];
        *(T4*)(out + m * ld + (i - m * cols)) = o;
    }
}

// bias gradient: the row tiles' partial sums, 64 columns to a block, four waves over the rows, joined in order
template <typename T> __global__ __launch_bounds__(256) void gff_cols_kernel(const float* part, int n, int cols, void* out, int out_f32)
{
    __shared__ float s[4][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
    float a = 0.0f;
    if (c < cols)
        for (int i = w; i < n; i += 4) a += part[(long long)i * cols + c];
    s[w][lane] = a;
    __syncthreads();
    if (w == 0 && c < cols) param_put<T>(out, out_f32, c, (s[0][lane] + s[1][lane]) + (s[2][lane] + s[3][lane]));
}

template <typename T> __global__ __launch_bounds__(256) void gff_zero_kernel(T* out, long long rows, int cols, long long ld)
{
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < rows * cols; i += (long long)gridDim.x * 256) out[i / cols * ld + i % cols] = (T)0.0f;
}

void gff_launch(const OpCtx& c, const GffDev& d, int dtype, int what, int act, int cfg)
{
    if (dtype == SDE_F16) gff_launch_f16(c, d, what, act, cfg);
    else if (dtype == SDE_BF16) gff_launch_bf16(c, d, what, act, cfg);
    else gff_launch_f32(c, d, what, act, cfg);
}

constexpr int kTileRows[3] = {256, 128, 64}, kResident[3] = {1, 2, 4};       // workgroups of a CU

// Tile and split of a product, by an estimate of its time: n tiles to a CU take the K-tiles' latency as often as workgroups come one after another, or their
// throughput n times, and n epilogues.  Measured on MI355X (us a K-tile: alone / on a full CU, and an epilogue): 16-bit types 256 x 256 1.4 / 1.75, 7; 128 x 128 0.6 / 0.72,
// 1.6; 64 x 64 0.35 / 0.30, 0.4; fp32, whose matrix instructions take 8 times as long on the same bytes, 7.3 / 7.3, 7; 2.05 / 2.1, 2; 0.66 / 0.575, 0.5.
// E.g. bf16 x W^T with K = 1280, F = 5120, us for the three tiles: 2 rows 28.5, 13.8, 9.1; 1024 rows 36.5, 46.5, 66.1; 8191 rows 217, 276, 472.
// A split of the contraction adds a launch and its parts in fp32, written and read at 4 TB/s.
// `pitch`: bytes from row to row of the first operand.  A tile's rows have to lie inside the 2 GB window of its loads: rows past it would come as zeros.
GffPlan gff_choose(int64_t rows, int64_t cols, int64_t contraction, int dtype, bool may_split, int64_t pitch = 0)
{
    static const double lat[2][3] = {{1.4, 0.6, 0.35}, {7.3, 2.05, 0.66}}, thr[2][3] = {{1.75, 0.72, 0.30}, {7.3, 2.1, 0.575}}, epi[2][3] = {{7.0, 1.6, 0.4}, {7.0, 2.0, 0.5}};
    const int t = dtype == SDE_F32;
    const int64_t nk = cdiv64(contraction * (int64_t)op_esize(dtype), 128);
    GffPlan best{0, 1};
    double least = 1e300;
    for (int c = 0; c < 3; ++c) {
        if ((kTileRows[c] - 1) * pitch + 128 > (int64_t)kOob) continue;
        const int64_t tiles = cdiv64(rows, kTileRows[c]) * cdiv64(cols, kTileRows[c]);
        for (int s = 1; s <= (may_split ? 32 : 1); ++s) {
            if (s > 1 && nk / s < 4) break;
            const double n = (double)cdiv64(tiles * s, 256);
            double us = (double)cdiv64(nk, s) * std::max(lat[t][c] * (double)cdiv64((int64_t)n, kResident[c]), thr[t][c] * n) + epi[t][c] * n;
            if (s > 1) us += 5.0 + (double)rows * cols * (2 * s + 1) * 4.0 / 4.0e6;
            if (us < least) { least = us; best = {c, s}; }
        }
    }
    return best;
}

struct GffWs { size_t dag, cols, part, total; GffPlan first, dx, dw; };
GffWs gff_ws(const sde_gated_ff_args& a)
{
    GffWs w{};
    const size_t e = op_esize(a.dtype);
    w.first = gff_choose(a.M, 2 * a.F, a.K, a.dtype, false);
    w.dx = gff_choose(a.M, a.K, 2 * a.F, a.dtype, true, 2 * a.F * (int64_t)e);
    w.dw = gff_choose(2 * a.F, a.K, a.M, a.dtype, true);
    w.dag = 0;
    w.cols = op_align((size_t)a.M * 2 * a.F * e);
    w.part = w.cols + (a.dbias ? op_align((size_t)cdiv64(a.M, kTileRows[w.first.cfg]) * 2 * 2 * a.F * 4) : 0);
    const int s1 = a.dx ? w.dx.splits : 1, s2 = a.dweight ? w.dw.splits : 1;
    w.total = w.part + op_align(std::max(s1 > 1 ? (size_t)s1 * a.M * a.K * 4 : 0, s2 > 1 ? (size_t)s2 * 2 * a.F * a.K * 4 : 0));
    return w;
}

GffDev gff_first(const sde_gated_ff_args& a)
{
    const int e = (int)op_esize(a.dtype);
    GffDev d{};
    d.A = (const char*)a.x; d.ldA = a.ld_x * e;
    d.B = (const char*)a.weight; d.ldB = a.ld_w * e;
    d.rowsA = (int)a.M; d.rowsB = (int)(2 * a.F); d.Kc = (int)a.K; d.F = (int)a.F;
    d.gate = a.F * a.ld_w * e;
    d.bias = a.bias; d.bias_f32 = a.bias_dtype == SDE_F32;
    d.splits = 1;
    return d;
}

// a product of the backward pass, split and joined where that fills the chip
template <typename T> void gff_product(const OpCtx& c, GffDev d, int dtype, int what, GffPlan plan, float* part)
{
    d.splits = plan.splits;
    d.part = part;
    gff_launch(c, d, dtype, what, 0, plan.cfg);
    if (d.splits == 1) return;
    const long long total = (long long)d.rowsA * d.rowsB;
    gff_join_kernel<T><<<(unsigned)std::min<long long>(cdiv64(total, 1024), 4096), 256, 0, c.stream>>>(part, d.splits, d.rowsA, d.rowsB, (T*)d.out, d.ld_out);
    op_launched("gated feed-forward join");
}

}  // namespace

GffPlan op_gated_ff_plan(const sde_gated_ff_args& a, int product, int64_t* units)
{
    const GffWs w = gff_ws(a);
    const GffPlan p = product == 0 ? w.first : product == 1 ? w.dx : w.dw;
    const int64_t rows = product == 2 ? 2 * a.F : a.M, cols = product == 0 ? 2 * a.F : a.K;
    *units = cdiv64(rows, kTileRows[p.cfg]) * cdiv64(cols, kTileRows[p.cfg]) * p.splits;
    return p;
}

size_t op_gated_ff_ws_bytes(const sde_gated_ff_args& a, bool backward)
{
    return backward && a.M ? gff_ws(a).total : 0;
}

void op_gated_ff_forward(const OpCtx& c, const sde_gated_ff_args& a)
{
    if (a.M == 0) return;
    GffDev d = gff_first(a);
    d.out = (char*)a.h;
    d.ld_out = a.ld_h;
    gff_launch(c, d, a.dtype, GFF_X_WT_FWD, a.activation, gff_choose(a.M, 2 * a.F, a.K, a.dtype, false).cfg);
}

void op_gated_ff_backward(const OpCtx& c, const sde_gated_ff_args& a)
{
    const int e = (int)op_esize(a.dtype);
    op_dispatch(a.dtype, [&](auto t) {
        typedef decltype(t) T;
        if (a.M == 0) {                          // nothing to add up: the parameters' gradients are zero
            if (a.dweight) gff_zero_kernel<T><<<1024, 256, 0, c.stream>>>((T*)a.dweight, 2 * a.F, (int)a.K, a.ld_dw);
            if (a.dbias) gff_cols_kernel<T><<<(unsigned)cdiv64(2 * a.F, 64), 256, 0, c.stream>>>(nullptr, 0, (int)(2 * a.F), a.dbias, a.bias_dtype == SDE_F32);
            op_launched("gated feed-forward zeros");
            return;
        }
        const GffWs w = gff_ws(a);
        char* dag = c.ws + w.dag;
        float* cols = a.dbias ? (float*)(c.ws + w.cols) : nullptr;
        float* part = (float*)(c.ws + w.part);
        GffDev d = gff_first(a);
        d.out = dag; d.ld_out = 2 * a.F;
        d.dh = (const char*)a.dh; d.ld_dh = a.ld_dh;
        d.colsum = cols;
        gff_launch(c, d, a.dtype, GFF_X_WT_BWD, a.activation, w.first.cfg);
        if (a.dbias) {
            gff_cols_kernel<T><<<(unsigned)cdiv64(2 * a.F, 64), 256, 0, c.stream>>>(cols, 2 * (int)cdiv64(a.M, kTileRows[w.first.cfg]), (int)(2 * a.F), a.dbias,
                                                                                    a.bias_dtype == SDE_F32);
            op_launched("gated feed-forward bias gradient");
        }
        if (a.dx) {
            GffDev g{};
            g.A = dag; g.ldA = 2 * a.F * e; g.rowsA = (int)a.M;
            g.B = (const char*)a.weight; g.ldB = a.ld_w * e; g.rowsB = (int)a.K;
            g.Kc = (int)(2 * a.F); g.out = (char*)a.dx; g.ld_out = a.ld_dx;
            gff_product<T>(c, g, a.dtype, GFF_DAG_W, w.dx, part);
        }
        if (a.dweight) {
            GffDev g{};
            g.A = dag; g.ldA = 2 * a.F * e; g.rowsA = (int)(2 * a.F);
            g.B = (const char*)a.x; g.ldB = a.ld_x * e; g.rowsB = (int)a.K;
            g.Kc = (int)a.M; g.out = (char*)a.dweight; g.ld_out = a.ld_dw;
            gff_product<T>(c, g, a.dtype, GFF_DAGT_X, w.dw, part);
        }
    });
}
