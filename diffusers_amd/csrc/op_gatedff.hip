// op_gatedff.hip — the gated feed-forward block and its gradient as operators of their own.
//
//   a = x Wv^T + bv,  g = x Wg^T + bg,  h = a act(g)                           W = [Wv; Wg] is [2F][K], the value rows first
//   da = dh act(g),  dg = dh a act'(g):  dx = [da dg] W,  dW = [da dg]^T x,  db = column sums of [da dg]
//
// Three products on one tile kernel: (1) x W^T with value and gate rows of the same columns in one tile, so that both projections, the
// activation and their product never leave the registers; (2) dx; (3) dW.  The backward pass forms a and g again instead of keeping
// them: 4 M K F operations against 4 M F values written by the forward pass and read back, and they stay in fp32.
#include "ops_device.h"

#include <algorithm>

namespace {

constexpr int BM = 256, BN = 256, kThreads = 512;
constexpr int kOperandBytes = 256 * 128;        // one K-tile of one operand: 256 rows of 128 bytes
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kSmem = 2 * kStageBytes;

// ---- activations: act(g) and its slope.  exp and 1/x are the hardware's (1 ulp); erf is the library's in fp32.
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
template <int ACT> __device__ __forceinline__ void activation(float g, float& act, float& slope)
{
    if constexpr (ACT == SDE_ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.0f + exp_of(-g));
        act = g * s;
        slope = s * (1.0f + g * (1.0f - s));
    } else if constexpr (ACT == SDE_ACT_GELU) {
        const float cdf = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
        act = g * cdf;
        slope = cdf + g * 0.3989422804014327f * exp_of(-0.5f * g * g);
    } else {
        // 0.5 (1 + tanh u) = 1 / (1 + exp(-2u)),  u = sqrt(2/pi) (g + 0.044715 g^3)
        const float g2 = g * g;
        const float s = __builtin_amdgcn_rcpf(1.0f + exp_of(-1.5957691216057308f * g * (1.0f + 0.044715f * g2)));
        act = g * s;
        slope = s + g * s * (1.0f - s) * 1.5957691216057308f * (1.0f + 0.134145f * g2);
    }
}

enum Epi { EPI_FWD, EPI_BWD, EPI_STORE, EPI_PART };

struct GemmDev {
    const char* A; const char* B;       // first element of row / contraction 0
    long long ldA, ldB;                 // bytes
    int rowsA, rowsB, Kc;               // rows of the output, columns of the output, contraction length
    long long gate;                     // EPI_FWD / EPI_BWD: byte offset of the gate rows in B
    int F;
    const void* bias; int bias_f32;
    char* out; long long ld_out;        // elements
    const char* dh; long long ld_dh;    // EPI_BWD
    float* colsum;                      // EPI_BWD: [2 * row tiles][2F], or null
    float* part;                        // EPI_PART: [splits][rowsA][rowsB]
    int splits, nbm, nbn;
};

// position of 16-byte chunk `c` of LDS row `row`, swizzled so that the reads below spread over all banks.
//   contraction along the row (128-byte rows): 8 chunks, XOR with the row
//   contraction across rows: XOR by 32-byte (16-bit types, transposed reads of 4 rows x 32 bytes) or 64-byte units (fp32)
template <typename T, bool TR> __device__ __forceinline__ int swz(int row)
{
    if constexpr (!TR) return row & 7;
    else if constexpr (sizeof(T) == 2) return ((row & 3) | ((row >> 3) & 1) << 2) << 1;
    else return ((row >> 2) & 3) << 2;
}

template <typename T, bool TR> __device__ __forceinline__ Frag<T> read_frag(const char* tile, int row0, int kk, int lane)
{
    const int r16 = lane & 15, g = lane >> 4;
    Frag<T> f;
    if constexpr (!TR) {
        const int row = row0 + r16;
        f.v = *(const decltype(f.v)*)(tile + row * 128 + (((kk * 4 + g) ^ swz<T, false>(row)) << 4));
    } else if constexpr (sizeof(T) == 2) {
        // a group of 16 lanes reads 4 rows of the contraction x 16 columns and gets them transposed: 4 contraction values of one column a lane
        typedef short short4_t __attribute__((ext_vector_type(4)));
        const int col = row0 + (r16 & 3) * 4;
        short4_t h[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int k = kk * 32 + g * 8 + i * 4 + (r16 >> 2);
            const char* a = tile + k * 512 + (((col >> 3) ^ swz<T, true>(k)) << 4) + (col & 7) * 2;
            h[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)a);
        }
        typedef short short8_t __attribute__((ext_vector_type(8)));
        short8_t w;
#pragma unroll
        for (int i = 0; i < 4; ++i) { w[i] = h[0][i]; w[4 + i] = h[1][i]; }
        f.v = __builtin_bit_cast(decltype(f.v), w);
    } else {
        const int col = row0 + r16;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = kk * 16 + g * 4 + j;
            f.v[j] = *(const float*)(tile + k * 1024 + (((col >> 2) ^ swz<T, true>(k)) << 4) + (col & 3) * 4);
        }
    }
    return f;
}

// One operand's share of a K-tile: 4 loads of 16 bytes a thread.
template <typename T, bool TR> struct Stager {
    unsigned voff[4];       // byte offset from the tile's base; kOob for rows / columns that do not exist
    int kpos[4];            // first contraction index of the chunk within the tile
    const char* base;
    long long step;
    __device__ __forceinline__ void init(const char* p, long long ld, int valid, int tid)
    {
        constexpr int V = kVec<T>;
        base = p;
        step = TR ? (long long)(128 / sizeof(T)) * ld : 128;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int L = j * kThreads + tid;
            if constexpr (!TR) {
                const int row = L >> 3, c = (L & 7) ^ swz<T, false>(row);
                voff[j] = row < valid ? (unsigned)(row * ld) + c * 16 : kOob;
                kpos[j] = c * V;
            } else {
                constexpr int CPR = 256 * sizeof(T) / 16;
                const int k = L / CPR, c = (L % CPR) ^ swz<T, true>(k);
                voff[j] = c * V < valid ? (unsigned)(k * ld) + c * 16 : kOob;
                kpos[j] = k;
            }
        }
    }
    __device__ __forceinline__ void issue(unsigned lds, int left)
    {
        const uintx4 r = make_rsrc(base);
#pragma unroll
        for (int j = 0; j < 4; ++j) dma16(r, kpos[j] < left ? voff[j] : kOob, lds + j * kThreads * 16);
        base += step;
    }
};

template <typename T, bool TRA, bool TRB, int EPI, int ACT>
__global__ __launch_bounds__(kThreads) void gff_gemm_kernel(GemmDev p)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int KT = 128 / sizeof(T);         // contraction elements of a K-tile
    constexpr bool PAIR = EPI == EPI_FWD || EPI == EPI_BWD;
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wid >> 2, wc = wid & 3, fr = lane & 15, fg = lane >> 4;

    // workgroups b, b + 8, ... share an XCD and its L2: each XCD gets a contiguous run of tiles
    int bid = blockIdx.x;
    {
        const int n = p.nbm * p.nbn, q = n >> 3, r = n & 7, xcd = bid & 7, i = bid >> 3;
        bid = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + i;
    }
    const int tm = bid / p.nbn, tn = bid - tm * p.nbn;
    const int m0 = tm * BM, n0 = tn * (PAIR ? BN / 2 : BN);

    const int nk_all = (p.Kc + KT - 1) / KT;
    const int kt0 = (int)((long long)nk_all * blockIdx.y / p.splits), kt1 = (int)((long long)nk_all * (blockIdx.y + 1) / p.splits);

    Stager<T, TRA> sa;
    Stager<T, TRB> sb;
    if constexpr (TRA) sa.init(p.A + (long long)m0 * sizeof(T) + (long long)kt0 * KT * p.ldA, p.ldA, p.rowsA - m0, tid);
    else sa.init(p.A + (long long)m0 * p.ldA + (long long)kt0 * 128, p.ldA, p.rowsA - m0, tid);
    if constexpr (PAIR) {
        // LDS row n of B: wave column n/64, then 32 value rows and the 32 gate rows of the same columns; a wave stages rows of one kind only
        const long long half = ((wid >> 2) & 1) ? p.gate : 0;
        sb.init(p.B + (long long)n0 * p.ldB + half + (long long)kt0 * 128, p.ldB, 0, tid);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int row = (j * kThreads + tid) >> 3, f = (row >> 6) * 32 + (row & 31);
            sb.voff[j] = n0 + f < p.F ? (unsigned)(f * p.ldB) + (((tid & 7) ^ swz<T, false>(row)) << 4) : kOob;
        }
    } else if constexpr (TRB) sb.init(p.B + (long long)n0 * sizeof(T) + (long long)kt0 * KT * p.ldB, p.ldB, p.rowsB - n0, tid);
    else sb.init(p.B + (long long)n0 * p.ldB + (long long)kt0 * 128, p.ldB, p.rowsB - n0, tid);

    const unsigned lds0 = (unsigned)(unsigned long long)(__attribute__((address_space(3))) char*)smem + wid * 1024;
    auto issue = [&](int kt) {
        const unsigned l = lds0 + (kt & 1) * kStageBytes;
        const int left = p.Kc - kt * KT;
        sa.issue(l, left);
        sb.issue(l + kOperandBytes, left);
    };

    floatx4 acc[4][8];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 8; ++b) acc[a][b] = floatx4{0.f, 0.f, 0.f, 0.f};

    if (kt0 < kt1) issue(kt0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int kt = kt0; kt < kt1; ++kt) {
        if (kt + 1 < kt1) issue(kt + 1);         // into the stage that was read before the last barrier
        const char* a = smem + (kt & 1) * kStageBytes;
        const char* b = a + kOperandBytes;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            Frag<T> bf[4], af[8];
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) bf[nt] = read_frag<T, TRB>(b, wc * 64 + nt * 16, kk, lane);
#pragma unroll
            for (int mt = 0; mt < 8; ++mt) af[mt] = read_frag<T, TRA>(a, wr * 128 + mt * 16, kk, lane);
#pragma unroll
            for (int mt = 0; mt < 8; ++mt)
#pragma unroll
                for (int nt = 0; nt < 4; ++nt) acc[nt][mt] = mma(bf[nt], af[mt], acc[nt][mt]);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }

    // a lane holds, for row m = .. + fr, the four columns .. + 4 fg
    typedef typename VecOf<T, 4>::type T4;
    if constexpr (PAIR) {
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
            const int f = n0 + wc * 32 + nt * 16 + fg * 4;
            const bool okf = f < p.F;            // F is a multiple of 4
            float bv[4], bg[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                bv[r] = okf && p.bias ? param_at<T>(p.bias, p.bias_f32, f + r) : 0.0f;
                bg[r] = okf && p.bias ? param_at<T>(p.bias, p.bias_f32, p.F + f + r) : 0.0f;
            }
            float cv[4] = {0.f, 0.f, 0.f, 0.f}, cg[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int mt = 0; mt < 8; ++mt) {
                const long long m = m0 + wr * 128 + mt * 16 + fr;
                if (m >= p.rowsA || !okf) continue;
                T4 dh4{};
                if constexpr (EPI == EPI_BWD) dh4 = *(const T4*)((const T*)p.dh + m * p.ld_dh + f);
                T4 o1, o2;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float a = acc[nt][mt][r] + bv[r], g = acc[nt + 2][mt][r] + bg[r];
                    float act, slope;
                    activation<ACT>(g, act, slope);
                    if constexpr (EPI == EPI_FWD) o1[r] = (T)(a * act);
                    else {
                        // rounded to the inputs' type once: they are operands of the next two products; the bias gradient takes them unrounded
                        const float d = (float)dh4[r], da = d * act, dg = d * a * slope;
                        cv[r] += da;
                        cg[r] += dg;
                        o1[r] = (T)da;
                        o2[r] = (T)dg;
                    }
                }
                T* o = (T*)p.out + m * p.ld_out + f;
                *(T4*)o = o1;
                if constexpr (EPI == EPI_BWD) *(T4*)(o + p.F) = o2;
            }
            if constexpr (EPI == EPI_BWD) {
                if (!p.colsum) continue;
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int o = 1; o < 16; o <<= 1) { cv[r] += __shfl_xor(cv[r], o); cg[r] += __shfl_xor(cg[r], o); }
                if (fr == 0 && okf) {
                    float* c = p.colsum + (long long)(tm * 2 + wr) * 2 * p.F + f;
                    *(floatx4*)c = floatx4{cv[0], cv[1], cv[2], cv[3]};
                    *(floatx4*)(c + p.F) = floatx4{cg[0], cg[1], cg[2], cg[3]};
                }
            }
        }
    } else {
#pragma unroll
        for (int nt = 0; nt < 4; ++nt) {
            const int n = n0 + wc * 64 + nt * 16 + fg * 4;
            if (n >= p.rowsB) continue;          // rowsB is a multiple of 4
#pragma unroll
            for (int mt = 0; mt < 8; ++mt) {
                const long long m = m0 + wr * 128 + mt * 16 + fr;
                if (m >= p.rowsA) continue;
                if constexpr (EPI == EPI_PART) *(floatx4*)(p.part + ((long long)blockIdx.y * p.rowsA + m) * p.rowsB + n) = acc[nt][mt];
                else {
                    T4 o;
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[r] = (T)acc[nt][mt][r];
                    *(T4*)((T*)p.out + m * p.ld_out + n) = o;
                }
            }
        }
    }
}

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

// A product whose tiles do not fill the 256 CUs is split along its contraction, at least 4 K-tiles to a part.
int gff_splits(int64_t rows, int64_t cols, int64_t contraction, int dtype)
{
    const int64_t tiles = cdiv64(rows, BM) * cdiv64(cols, BN), nk = cdiv64(contraction * (int64_t)op_esize(dtype), 128);
    if (tiles >= 192) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>({256 / tiles, nk / 4, 64}));
}

template <typename T, bool TRA, bool TRB, int EPI, int ACT> void gff_gemm(const OpCtx& c, GemmDev d)
{
    constexpr bool PAIR = EPI == EPI_FWD || EPI == EPI_BWD;
    d.nbm = (int)cdiv64(d.rowsA, BM);
    d.nbn = (int)cdiv64(PAIR ? d.F : d.rowsB, PAIR ? BN / 2 : BN);
    auto k = gff_gemm_kernel<T, TRA, TRB, EPI, ACT>;
    op_allow_lds((const void*)k, kSmem);
    k<<<dim3((unsigned)(d.nbm * d.nbn), (unsigned)d.splits), kThreads, kSmem, c.stream>>>(d);
    op_launched("gated feed-forward product");
}

template <typename F> void with_activation(int act, F&& f)
{
    if (act == SDE_ACT_GELU) f(std::integral_constant<int, SDE_ACT_GELU>{});
    else if (act == SDE_ACT_GELU_TANH) f(std::integral_constant<int, SDE_ACT_GELU_TANH>{});
    else f(std::integral_constant<int, SDE_ACT_SILU>{});
}

// out = product of two operands, split and joined where that fills the chip
template <typename T, bool TRA, bool TRB> void gff_product(const OpCtx& c, GemmDev d, float* part, int dtype)
{
    d.splits = gff_splits(d.rowsA, d.rowsB, d.Kc, dtype);
    if (d.splits == 1) { gff_gemm<T, TRA, TRB, EPI_STORE, 0>(c, d); return; }
    d.part = part;
    gff_gemm<T, TRA, TRB, EPI_PART, 0>(c, d);
    const long long total = (long long)d.rowsA * d.rowsB;
    gff_join_kernel<T><<<(unsigned)std::min<long long>(cdiv64(total, 1024), 4096), 256, 0, c.stream>>>(part, d.splits, d.rowsA, d.rowsB, (T*)d.out, d.ld_out);
    op_launched("gated feed-forward join");
}

struct GffWs { size_t dag, cols, part, total; };
GffWs gff_ws(const sde_gated_ff_args& a)
{
    GffWs w{};
    const size_t e = op_esize(a.dtype);
    w.dag = 0;
    w.cols = op_align((size_t)a.M * 2 * a.F * e);
    w.part = w.cols + (a.dbias ? op_align((size_t)cdiv64(a.M, BM) * 2 * 2 * a.F * 4) : 0);
    const int s1 = a.dx ? gff_splits(a.M, a.K, 2 * a.F, a.dtype) : 1, s2 = a.dweight ? gff_splits(2 * a.F, a.K, a.M, a.dtype) : 1;
    w.total = w.part + op_align(std::max(s1 > 1 ? (size_t)s1 * a.M * a.K * 4 : 0, s2 > 1 ? (size_t)s2 * 2 * a.F * a.K * 4 : 0));
    return w;
}

GemmDev gff_first(const sde_gated_ff_args& a)
{
    const int e = (int)op_esize(a.dtype);
    GemmDev d{};
    d.A = (const char*)a.x; d.ldA = a.ld_x * e;
    d.B = (const char*)a.weight; d.ldB = a.ld_w * e;
    d.rowsA = (int)a.M; d.rowsB = (int)(2 * a.F); d.Kc = (int)a.K; d.F = (int)a.F;
    d.gate = a.F * a.ld_w * e;
    d.bias = a.bias; d.bias_f32 = a.bias_dtype == SDE_F32;
    d.splits = 1;
    return d;
}

}  // namespace

size_t op_gated_ff_ws_bytes(const sde_gated_ff_args& a, bool backward)
{
    return backward && a.M ? gff_ws(a).total : 0;
}

void op_gated_ff_forward(const OpCtx& c, const sde_gated_ff_args& a)
{
    if (a.M == 0) return;
    GemmDev d = gff_first(a);
    d.out = (char*)a.h;
    d.ld_out = a.ld_h;
    op_dispatch(a.dtype, [&](auto t) { with_activation(a.activation, [&](auto act) { gff_gemm<decltype(t), false, false, EPI_FWD, decltype(act)::value>(c, d); }); });
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
        GemmDev d = gff_first(a);
        d.out = dag; d.ld_out = 2 * a.F;
        d.dh = (const char*)a.dh; d.ld_dh = a.ld_dh;
        d.colsum = cols;
        with_activation(a.activation, [&](auto act) { gff_gemm<T, false, false, EPI_BWD, decltype(act)::value>(c, d); });
        if (a.dbias) {
            gff_cols_kernel<T><<<(unsigned)cdiv64(2 * a.F, 64), 256, 0, c.stream>>>(cols, 2 * (int)cdiv64(a.M, BM), (int)(2 * a.F), a.dbias, a.bias_dtype == SDE_F32);
            op_launched("gated feed-forward bias gradient");
        }
        if (a.dx) {
            GemmDev g{};
            g.A = dag; g.ldA = 2 * a.F * e; g.rowsA = (int)a.M;
            g.B = (const char*)a.weight; g.ldB = a.ld_w * e; g.rowsB = (int)a.K;
            g.Kc = (int)(2 * a.F); g.out = (char*)a.dx; g.ld_out = a.ld_dx;
            gff_product<T, false, true>(c, g, part, a.dtype);
        }
        if (a.dweight) {
            GemmDev g{};
            g.A = dag; g.ldA = 2 * a.F * e; g.rowsA = (int)(2 * a.F);
            g.B = (const char*)a.x; g.ldB = a.ld_x * e; g.rowsB = (int)a.K;
            g.Kc = (int)a.M; g.out = (char*)a.dweight; g.ld_out = a.ld_dw;
            gff_product<T, true, true>(c, g, part, a.dtype);
        }
    });
}
