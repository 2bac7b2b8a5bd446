// op_layernorm.hip — layer norm and its gradient as operators of their own.
//
//   y = (x - mean) rstd gamma + beta,  mean and var over the C values of a row (two passes over registers: no cancellation)
//   xh = (x - mean) rstd,  g = dy gamma:  dx = rstd (g - mean(g) - xh mean(g xh)),  dgamma = sum dy xh,  dbeta = sum dy
//
// Bound by HBM: forward 2 values per element, backward 3 (x, dy in, dx out).  A row is held in registers by `tpr` lanes (8..64: several
// rows to a wave, reduced by shuffles) or, past 5 chunks a lane, by a block of 256 (reduced through LDS).  A lane keeps its columns for the whole launch, so
// gamma / beta are read once a block and the gradients of the parameters grow in registers; each block leaves one fp32 row of
// partial sums and a second kernel adds those in a fixed order (no atomics: results do not change from run to run).
#include "ops_device.h"

#include <algorithm>

namespace {

constexpr int kThreads = 256;
constexpr int kMaxVplWave = 5, kMaxVplBlock = 8;

// 16 bytes at any element: rows of an odd number of values start anywhere, and the hardware takes a global access at any address
template <typename T, int VEC> struct Loose { typedef typename VecOf<T, VEC>::type type __attribute__((aligned(alignof(T)))); };
template <typename T> struct Loose<T, 1> { typedef T type; };

struct LnPlan {
    int vec;        // elements of an access: 16 bytes' worth, or 1 for rows shorter than that
    int nchunk;     // accesses in a row
    int block;      // 1: a row belongs to the whole block
    int log2tpr;    // lanes of a row (wave variant)
    int vpl;        // accesses a lane; 0: the row does not fit into registers and is read several times
};

struct LnDev {
    const void* x; const void* gamma; const void* beta; const void* dy;
    void* y; void* dx; float* mean; float* rstd; const float* mean_in; const float* rstd_in;
    float* part;                 // [blocks][2][C]
    long long rows, ldx, ldy, lddy, lddx;
    int C, nchunk, log2tpr;
    float eps, inv_c;
    int pf32;                    // parameters are fp32
};

// a lane's VEC parameters from element c on
template <typename T, int VEC> __device__ __forceinline__ void params_at(const LnDev& p, const void* q, int c, bool in, float other, float (&f)[VEC])
{
    if (!q || !in) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) f[i] = other;
        return;
    }
    if constexpr (VEC > 1) {
        if (p.pf32) {
#pragma unroll
            for (int i = 0; i < VEC; i += 4) {
                const floatx4 v = *(const typename Loose<float, 4>::type*)((const float*)q + c + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) f[i + j] = v[j];
            }
        } else vec_get<VEC, T>(*(const typename Loose<T, VEC>::type*)((const T*)q + c), f);
        return;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = param_at<T>(q, p.pf32, c + i);
}

// First element of access `chunk` of a row.  The last one of a row that is not whole accesses ends with the row: its first `again` elements belong to the access before and are left
// out of the sums (their results are written twice, the same both times).
template <int VEC, bool TAIL> __device__ __forceinline__ int first_of(const LnDev& p, int chunk, int& again)
{
    const int c = chunk * VEC, over = c + VEC - p.C;
    again = TAIL && over > 0 ? over : 0;
    return c - again;
}

template <bool BLOCK> __device__ __forceinline__ void row_sum2(float& a, float& b, int log2tpr, float (*red)[4][2], int buf)
{
    if constexpr (BLOCK) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) { a += __shfl_xor(a, o); b += __shfl_xor(b, o); }
        if ((threadIdx.x & 63) == 0) { red[buf][threadIdx.x >> 6][0] = a; red[buf][threadIdx.x >> 6][1] = b; }
        __syncthreads();
        a = (red[buf][0][0] + red[buf][1][0]) + (red[buf][2][0] + red[buf][3][0]);
        b = (red[buf][0][1] + red[buf][1][1]) + (red[buf][2][1] + red[buf][3][1]);
    } else {
        for (int o = 1 << log2tpr >> 1; o > 0; o >>= 1) { a += __shfl_xor(a, o); b += __shfl_xor(b, o); }
    }
}

// TAIL: the row is not whole accesses
template <typename T, int VEC, int VPL, bool BLOCK, bool TAIL>
__global__ __launch_bounds__(kThreads) void ln_fwd_kernel(LnDev p)
{
    typedef typename Loose<T, VEC>::type V;
    __shared__ float red[2][4][2];
    const int tpr = BLOCK ? kThreads : 1 << p.log2tpr;
    const int pos = threadIdx.x & (tpr - 1), slot = BLOCK ? 0 : threadIdx.x >> p.log2tpr;
    const int rows_pb = BLOCK ? 1 : kThreads >> p.log2tpr;
    float gm[VPL][VEC], bt[VPL][VEC];
    bool in[VPL];
    int at[VPL], again[VPL];
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
        in[v] = v * tpr + pos < p.nchunk;
        at[v] = first_of<VEC, TAIL>(p, v * tpr + pos, again[v]);
        if (TAIL && !in[v]) again[v] = VEC;
        params_at<T, VEC>(p, p.gamma, at[v], in[v], 1.0f, gm[v]);
        params_at<T, VEC>(p, p.beta, at[v], in[v], 0.0f, bt[v]);
    }
    const long long step = (long long)gridDim.x * rows_pb;
    const long long first = (long long)blockIdx.x * rows_pb;
    // every lane of a wave goes through the same number of rows: the shuffles of a row stay inside its lanes, rows past the end read nothing
    V raw[VPL];
    auto fetch = [&](long long r) {
#pragma unroll
        for (int v = 0; v < VPL; ++v)
            if (in[v] && r < p.rows) raw[v] = *(const V*)((const T*)p.x + r * p.ldx + at[v]);
            else raw[v] = V{};
    };
    fetch(first + slot);
    for (long long r0 = first; r0 < p.rows; r0 += step) {
        const long long r = r0 + slot;
        float x[VPL][VEC];
#pragma unroll
        for (int v = 0; v < VPL; ++v) vec_get<VEC, T>(raw[v], x[v]);
        fetch(r + step);
        float s = 0.0f, q = 0.0f;
#pragma unroll
        for (int v = 0; v < VPL; ++v)
#pragma unroll
            for (int i = 0; i < VEC; ++i) s += !TAIL || i >= again[v] ? x[v][i] : 0.0f;
        row_sum2<BLOCK>(s, q, p.log2tpr, red, 0);
        const float mean = s * p.inv_c;
        s = 0.0f;
#pragma unroll
        for (int v = 0; v < VPL; ++v)
#pragma unroll
            for (int i = 0; i < VEC; ++i) { x[v][i] -= mean; s = (TAIL ? i >= again[v] : in[v]) ? fmaf(x[v][i], x[v][i], s) : s; }
        row_sum2<BLOCK>(s, q, p.log2tpr, red, 1);
        const float rstd = 1.0f / sqrtf(s * p.inv_c + p.eps);
        if (r < p.rows) {
            if (pos == 0) {
                if (p.mean) p.mean[r] = mean;
                if (p.rstd) p.rstd[r] = rstd;
            }
#pragma unroll
            for (int v = 0; v < VPL; ++v) {
                if (!in[v]) continue;
                float o[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) o[i] = fmaf(x[v][i] * rstd, gm[v][i], bt[v][i]);
                *(V*)((T*)p.y + r * p.ldy + at[v]) = vec_set<VEC, T>(o);
            }
        }
    }
}

template <typename T, int VEC, int VPL, bool BLOCK, bool TAIL>
__global__ __launch_bounds__(kThreads) void ln_bwd_kernel(LnDev p)
{
    typedef typename Loose<T, VEC>::type V;
    __shared__ float red[2][4][2];
    __shared__ float cols[BLOCK ? 1 : 2 * 64 * VPL * VEC];
    const int tpr = BLOCK ? kThreads : 1 << p.log2tpr;
    const int pos = threadIdx.x & (tpr - 1), slot = BLOCK ? 0 : threadIdx.x >> p.log2tpr;
    const int rows_pb = BLOCK ? 1 : kThreads >> p.log2tpr;
    float gm[VPL][VEC], dg[VPL][VEC], db[VPL][VEC];
    bool in[VPL];
    int at[VPL], again[VPL];
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
        in[v] = v * tpr + pos < p.nchunk;
        at[v] = first_of<VEC, TAIL>(p, v * tpr + pos, again[v]);
        if (TAIL && !in[v]) again[v] = VEC;
        params_at<T, VEC>(p, p.gamma, at[v], in[v], 1.0f, gm[v]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            dg[v][i] = 0.0f;
            db[v][i] = 0.0f;
        }
    }
    const long long step = (long long)gridDim.x * rows_pb;
    const long long first = (long long)blockIdx.x * rows_pb;
    V rx[VPL], ry[VPL];
    float mean_n = 0.0f, rstd_n = 0.0f;
    auto fetch = [&](long long r) {
        const bool ok = r < p.rows;
        mean_n = ok ? p.mean_in[r] : 0.0f;
        rstd_n = ok ? p.rstd_in[r] : 0.0f;
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            if (in[v] && ok) {
                rx[v] = *(const V*)((const T*)p.x + r * p.ldx + at[v]);
                ry[v] = *(const V*)((const T*)p.dy + r * p.lddy + at[v]);
            } else { rx[v] = V{}; ry[v] = V{}; }
        }
    };
    fetch(first + slot);
    int buf = 0;
    for (long long r0 = first; r0 < p.rows; r0 += step) {
        const long long r = r0 + slot;
        const float mean = mean_n, rstd = rstd_n;
        float xh[VPL][VEC], d[VPL][VEC];
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            vec_get<VEC, T>(rx[v], xh[v]);
            vec_get<VEC, T>(ry[v], d[v]);
        }
        fetch(r + step);
#pragma unroll
        for (int v = 0; v < VPL; ++v)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                xh[v][i] = (xh[v][i] - mean) * rstd;
                const float g = !TAIL || i >= again[v] ? d[v][i] * gm[v][i] : 0.0f;
                s1 += g;
                s2 = fmaf(g, xh[v][i], s2);
                db[v][i] += d[v][i];
                dg[v][i] = fmaf(d[v][i], xh[v][i], dg[v][i]);
            }
        row_sum2<BLOCK>(s1, s2, p.log2tpr, red, buf);
        buf ^= 1;                       // one barrier a row: the other buffer was read before this row's barrier
        s1 *= p.inv_c;
        s2 *= p.inv_c;
        if (r < p.rows && p.dx) {
#pragma unroll
            for (int v = 0; v < VPL; ++v) {
                if (!in[v]) continue;
                float o[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) o[i] = rstd * (fmaf(d[v][i], gm[v][i], -s1) - xh[v][i] * s2);
                *(V*)((T*)p.dx + r * p.lddx + at[v]) = vec_set<VEC, T>(o);
            }
        }
    }
    if (!p.part) return;
    float* part = p.part + (long long)blockIdx.x * 2 * p.C;
    if constexpr (BLOCK) {
#pragma unroll
        for (int v = 0; v < VPL; ++v) {
            if (!in[v]) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                if (TAIL && i < again[v]) continue;
                part[at[v] + i] = dg[v][i];
                part[p.C + at[v] + i] = db[v][i];
            }
        }
    } else {
        // rows of a wave by shuffles, then the four waves in turn through LDS
        const int wave = threadIdx.x >> 6;
#pragma unroll
        for (int v = 0; v < VPL; ++v)
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                for (int o = tpr; o < 64; o <<= 1) { dg[v][i] += __shfl_xor(dg[v][i], o); db[v][i] += __shfl_xor(db[v][i], o); }
        for (int w = 0; w < 4; ++w) {
            if (wave == w && (threadIdx.x & 63) < tpr) {
#pragma unroll
                for (int v = 0; v < VPL; ++v)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        if (TAIL && i < again[v]) continue;
                        const int c = at[v] + i;                             // < C <= 64 * VPL * VEC: tpr <= 64
                        cols[c] = (w ? cols[c] : 0.0f) + dg[v][i];
                        cols[64 * VPL * VEC + c] = (w ? cols[64 * VPL * VEC + c] : 0.0f) + db[v][i];
                    }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < p.C; c += kThreads) { part[c] = cols[c]; part[p.C + c] = cols[64 * VPL * VEC + c]; }
    }
}

// rows that do not fit into registers: a block to a row, the row is read once for each sum and once more for the result
template <typename T> __global__ __launch_bounds__(kThreads) void ln_fwd_long_kernel(LnDev p)
{
    __shared__ float red[2][4][2];
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* x = (const T*)p.x + r * p.ldx;
        T* y = (T*)p.y + r * p.ldy;
        float s = 0.0f, q = 0.0f;
        for (int c = threadIdx.x; c < p.C; c += kThreads) s += (float)x[c];
        row_sum2<true>(s, q, 0, red, 0);
        const float mean = s * p.inv_c;
        s = 0.0f;
        for (int c = threadIdx.x; c < p.C; c += kThreads) { const float d = (float)x[c] - mean; s = fmaf(d, d, s); }
        row_sum2<true>(s, q, 0, red, 1);
        const float rstd = 1.0f / sqrtf(s * p.inv_c + p.eps);
        if (threadIdx.x == 0) {
            if (p.mean) p.mean[r] = mean;
            if (p.rstd) p.rstd[r] = rstd;
        }
        for (int c = threadIdx.x; c < p.C; c += kThreads) {
            const float g = p.gamma ? param_at<T>(p.gamma, p.pf32, c) : 1.0f, b = p.beta ? param_at<T>(p.beta, p.pf32, c) : 0.0f;
            y[c] = (T)fmaf(((float)x[c] - mean) * rstd, g, b);
        }
    }
}

template <typename T> __global__ __launch_bounds__(kThreads) void ln_bwd_long_kernel(LnDev p)
{
    __shared__ float red[2][4][2];
    float* part = p.part ? p.part + (long long)blockIdx.x * 2 * p.C : nullptr;
    bool fresh = true;                   // a block's first row sets its partial sums, later rows add (each column has one thread)
    int buf = 0;
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x, fresh = false) {
        const T* x = (const T*)p.x + r * p.ldx;
        const T* dy = (const T*)p.dy + r * p.lddy;
        const float mean = p.mean_in[r], rstd = p.rstd_in[r];
        float s1 = 0.0f, s2 = 0.0f;
        for (int c = threadIdx.x; c < p.C; c += kThreads) {
            const float xh = ((float)x[c] - mean) * rstd, d = (float)dy[c];
            const float g = p.gamma ? d * param_at<T>(p.gamma, p.pf32, c) : d;
            s1 += g;
            s2 = fmaf(g, xh, s2);
            if (part) {
                part[c] = (fresh ? 0.0f : part[c]) + d * xh;
                part[p.C + c] = (fresh ? 0.0f : part[p.C + c]) + d;
            }
        }
        row_sum2<true>(s1, s2, 0, red, buf);
        buf ^= 1;
        s1 *= p.inv_c;
        s2 *= p.inv_c;
        if (p.dx)
            for (int c = threadIdx.x; c < p.C; c += kThreads) {
                const float xh = ((float)x[c] - mean) * rstd, d = (float)dy[c];
                const float g = p.gamma ? d * param_at<T>(p.gamma, p.pf32, c) : d;
                ((T*)p.dx)[r * p.lddx + c] = (T)(rstd * (g - s1 - xh * s2));
            }
    }
}

// column sums of part[n][2][C]: a block takes 64 columns, each of its 16 waves every 16th row, four in flight; the waves are added in order
template <typename T> __global__ __launch_bounds__(1024) void ln_cols_kernel(const float* part, int n, int C, void* dgamma, void* dbeta, int pf32)
{
    __shared__ float s[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + lane;                  // of 2C
    const long long pitch = 2ll * C;
    float a[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < pitch) {
        int i = w;
        for (; i + 48 < n; i += 64)
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j] += part[(i + 16 * j) * pitch + c];
        for (; i < n; i += 16) a[0] += part[i * pitch + c];
    }
    s[w][lane] = (a[0] + a[1]) + (a[2] + a[3]);
    __syncthreads();
    if (w == 0 && c < pitch) {
        float t = s[0][lane];
#pragma unroll
        for (int i = 1; i < 16; ++i) t += s[i][lane];
        if (c < C) { if (dgamma) param_put<T>(dgamma, pf32, c, t); }
        else if (dbeta) param_put<T>(dbeta, pf32, c - C, t);
    }
}

// accesses of a lane at most
constexpr int ln_most(int vec, bool block) { return block ? kMaxVplBlock : vec == 8 ? 3 : vec == 4 ? kMaxVplWave : 1; }

LnPlan ln_plan(const sde_layer_norm_args& a)
{
    const int full = 16 / (int)op_esize(a.dtype);
    LnPlan p{a.C >= full ? full : 1, 0, 0, 6, 0};
    if (cdiv64(a.C, p.vec) > (int64_t)kThreads * kMaxVplBlock) return p;
    p.nchunk = (int)cdiv64(a.C, p.vec);
    // few rows: as many lanes as the row has accesses, for the shortest chain of loads; many rows: the split that leaves the fewest lanes idle, with at most 3 accesses of 8 values a
    // lane (more leave too few registers for other waves: fp16 65536 x 320, forward / backward 24.0 / 54.5 us with 5, 18.5 / 33.9 with 3; fp32's 4 values: 5 are as good as 3)
    const int most = ln_most(p.vec, false);
    if (p.nchunk > 64 * most || (a.rows < 512 && p.nchunk > 64)) {
        p.block = 1;
        p.vpl = cdiv(p.nchunk, kThreads);
        if (p.vpl > 5) p.vpl = 8;
        return p;
    }
    int best = 1 << 30;
    for (int l = 3; l <= 6; ++l) {
        const int vpl = cdiv(p.nchunk, 1 << l);
        if (vpl > most) continue;
        const int cost = a.rows < 512 ? -l : (vpl << l);
        if (cost <= best) { best = cost; p.log2tpr = l; p.vpl = vpl; }
    }
    return p;
}

// blocks of the backward pass: two for each CU, fewer when there are few rows or when the rows are so long that the partial sums would take more than 256 MB
int ln_bwd_blocks(const sde_layer_norm_args& a)
{
    const LnPlan p = ln_plan(a);
    const int64_t rows_pb = p.vpl && !p.block ? kThreads >> p.log2tpr : 1;
    return (int)std::min<int64_t>({cdiv64(a.rows, rows_pb), 512, std::max<int64_t>(1, (int64_t(256) << 20) / (8 * a.C))});
}

LnDev ln_dev(const sde_layer_norm_args& a, const LnPlan& p)
{
    LnDev d{};
    d.x = a.x; d.gamma = a.gamma; d.beta = a.beta; d.dy = a.dy; d.y = a.y; d.dx = a.dx;
    d.mean = a.mean; d.rstd = a.rstd; d.mean_in = a.mean; d.rstd_in = a.rstd;
    d.rows = a.rows; d.ldx = a.ld_x; d.ldy = a.ld_y; d.lddy = a.ld_dy; d.lddx = a.ld_dx;
    d.C = (int)a.C; d.nchunk = p.nchunk; d.log2tpr = p.log2tpr;
    d.eps = a.eps; d.inv_c = 1.0f / (float)a.C; d.pf32 = a.param_dtype == SDE_F32;
    return d;
}

template <typename T, int VEC, bool BLOCK, bool BWD> void ln_launch(const LnPlan& p, const LnDev& d, int grid, hipStream_t s)
{
    auto go = [&](auto vpl) {
        constexpr int N = decltype(vpl)::value;
        if constexpr (N <= ln_most(VEC, BLOCK)) {
            auto of = [&](auto tail) {
                if constexpr (BWD) ln_bwd_kernel<T, VEC, N, BLOCK, decltype(tail)::value><<<grid, kThreads, 0, s>>>(d);
                else ln_fwd_kernel<T, VEC, N, BLOCK, decltype(tail)::value><<<grid, kThreads, 0, s>>>(d);
            };
            if constexpr (VEC == 1) of(std::false_type{});
            else if (d.C % VEC) of(std::true_type{});
            else of(std::false_type{});
        }
    };
    switch (p.vpl) {
    case 1: go(std::integral_constant<int, 1>{}); break;
    case 2: go(std::integral_constant<int, 2>{}); break;
    case 3: go(std::integral_constant<int, 3>{}); break;
    case 4: go(std::integral_constant<int, 4>{}); break;
    case 5: go(std::integral_constant<int, 5>{}); break;
    default: go(std::integral_constant<int, 8>{}); break;
    }
}

template <typename T, bool BWD> void ln_run(const LnPlan& p, const LnDev& d, int grid, hipStream_t s)
{
    if (p.vpl == 0) {
        if constexpr (BWD) ln_bwd_long_kernel<T><<<grid, kThreads, 0, s>>>(d);
        else ln_fwd_long_kernel<T><<<grid, kThreads, 0, s>>>(d);
    } else if (p.vec == 1) ln_launch<T, 1, false, BWD>(p, d, grid, s);          // fewer values than an access
    else {
        if (p.block) ln_launch<T, kVec<T>, true, BWD>(p, d, grid, s);
        else ln_launch<T, kVec<T>, false, BWD>(p, d, grid, s);
    }
    op_launched("layer norm");
}

}  // namespace

size_t op_layer_norm_ws_bytes(const sde_layer_norm_args& a)
{
    return a.rows && (a.dgamma || a.dbeta) ? op_align((size_t)ln_bwd_blocks(a) * 2 * a.C * 4) : 0;
}

void op_layer_norm_forward(const OpCtx& c, const sde_layer_norm_args& a)
{
    if (a.rows == 0) return;
    const LnPlan p = ln_plan(a);
    const int64_t rows_pb = p.vpl && !p.block ? kThreads >> p.log2tpr : 1;
    const int grid = (int)std::min<int64_t>(cdiv64(a.rows, rows_pb), 1024);
    const LnDev d = ln_dev(a, p);
    op_dispatch(a.dtype, [&](auto t) { ln_run<decltype(t), false>(p, d, grid, c.stream); });
}

void op_layer_norm_backward(const OpCtx& c, const sde_layer_norm_args& a)
{
    const LnPlan p = ln_plan(a);
    LnDev d = ln_dev(a, p);
    const bool params = a.dgamma || a.dbeta;
    const int grid = a.rows ? ln_bwd_blocks(a) : 0;
    d.part = params ? (float*)c.ws : nullptr;
    op_dispatch(a.dtype, [&](auto t) {
        typedef decltype(t) T;
        if (grid) ln_run<T, true>(p, d, grid, c.stream);
        if (params) {        // without rows the sums are empty: zeros
            ln_cols_kernel<T><<<(unsigned)cdiv64(2 * a.C, 64), 1024, 0, c.stream>>>((const float*)c.ws, grid, (int)a.C, a.dgamma, a.dbeta, d.pf32);
            op_launched("layer norm column sums");
        }
    });
}
