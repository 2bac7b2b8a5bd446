// op_gatedff_kernel.h — the tile kernel of the gated feed-forward block and its launcher, for one element type (op_gatedff_{f16,bf16,f32}.hip).
//
// out = A B^T over 128-byte steps of the contraction.  Either operand may lie with its contraction along the rows (the loads of a row are contiguous) or
// across them (TR: LDS keeps the rows and they are read transposed), so that x W^T, [da dg] W and [da dg]^T x need no transposed copies.
//
// Three tiles.  256 x 256, 8 waves of 128 x 64: one workgroup to a CU, 128 KB of LDS, for work that fills the chip with them; per wave 12 LDS reads feed 32 matrix instructions, and a K-tile
// brings 64 KB for 512 of them -- 128 x 128 needs twice the bytes per instruction.  128 x 128 (4 waves of 64 x 64, two workgroups to a CU) and 64 x 64 (4 waves of 32 x 32) are for
// work that would leave CUs idle; gff_choose in op_gatedff.hip holds the rule and what each measured.
//
// A workgroup walks its tiles as one stream of K-tiles: while a K-tile is multiplied the next one -- at a tile's end the first of the next tile -- is on its way into the
// other LDS stage, so that the epilogue hides the next tile's first loads.
#pragma once
#include "op_gatedff.h"
#include "ops_device.h"

namespace {

// ---- activations: act(g) and its slope.  exp and 1 / x are the hardware's (1 ulp).  The erf form takes the tail w = Phi(-|g|) = t Q(t) exp(-g^2 / 2), t = 1 / (1 + p |g|);
// act = max(g, 0) - |g| w has no difference of near values.
// 16-bit types: Abramowitz & Stegun 7.1.26, Q of five terms, w off by at most 7.5e-8 absolutely (relatively 5e-5 at |g| = 3, 1.6e-3 at 5, 1e-2 at 8).  12 plain and 2 transcendental
// instructions; the library's erff took about 40 and made the epilogue of short-K products the bound.
// fp32, whose products leave the epilogue time: Q of nine terms, fitted to erfcx(|g| / sqrt 2) / (2 t) for the least relative error on 0 <= |g| <= 13.3 (1.0e-8; past that w is less
// than fp32's smallest normal value), so that gates far out on the negative side keep their precision: act is off by (g^2 + 32) 2^-24 of itself, the g^2 from the exponential's argument.
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
template <typename T, int ACT> __device__ __forceinline__ void activation(float g, float& act, float& slope)
{
    if constexpr (ACT == SDE_ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.0f + exp_of(-g));
        act = g * s;
        slope = s * (1.0f + g * (1.0f - s));
    } else if constexpr (ACT == SDE_ACT_GELU) {
        const float ax = fabsf(g);
        const float e = __builtin_amdgcn_exp2f(g * g * -0.72134752f);                      // exp(-g^2 / 2)
        float t, w;
        if constexpr (sizeof(T) == 4) {
            t = __builtin_amdgcn_rcpf(fmaf(0.26452443f, ax, 1.0f));
            w = fmaf(0.0310996249f, t, -0.146480367f);
            w = fmaf(w, t, 0.223770157f);
            w = fmaf(w, t, -0.122620679f);
            w = fmaf(w, t, 0.142120138f);
            w = fmaf(w, t, 0.0586104058f);
            w = fmaf(w, t, 0.102940425f);
            w = fmaf(w, t, 0.105005592f);
            w = fmaf(w, t, 0.105554707f);
        } else {
            t = __builtin_amdgcn_rcpf(fmaf(0.23164189f, ax, 1.0f));                        // p / sqrt 2, p = 0.3275911
            w = fmaf(0.5307027145f, t, -0.7265760135f);                                    // a5 / 2 .. a1 / 2
            w = fmaf(w, t, 0.7107068705f);
            w = fmaf(w, t, -0.142248368f);
            w = fmaf(w, t, 0.127414796f);
        }
        w = w * t * e;
        act = fmaf(-fminf(ax, 64.0f), w, fmaxf(g, 0.0f));                              // an infinite gate: infinity times 0 is not wanted here
        slope = fmaf(g * 0.3989422804014327f, e, g >= 0.0f ? 1.0f - w : w);
    } else {
        // 0.5 (1 + tanh u) = 1 / (1 + exp(-2u)),  u = sqrt(2/pi) (g + 0.044715 g^3)
        const float g2 = g * g;
        const float s = __builtin_amdgcn_rcpf(1.0f + exp_of(-1.5957691216057308f * g * (1.0f + 0.044715f * g2)));
        act = g * s;
        slope = s + g * s * (1.0f - s) * 1.5957691216057308f * (1.0f + 0.134145f * g2);
    }
}

template <int WM_, int WN_, int MT_, int NT_> struct Tile {
    static constexpr int WM = WM_, WN = WN_, MT = MT_, NT = NT_;
    static constexpr int threads = WM * WN * 64, BM = WM * MT * 16, BN = WN * NT * 16;
    static constexpr int a_bytes = BM * 128, b_bytes = BN * 128, stage = a_bytes + b_bytes, lds = 2 * stage;
};
template <int CFG> struct TileOf;
template <> struct TileOf<0> { typedef Tile<2, 4, 8, 4> type; };
template <> struct TileOf<1> { typedef Tile<2, 2, 4, 4> type; };
template <> struct TileOf<2> { typedef Tile<2, 2, 2, 2> type; };

// Position of 16-byte chunk c in LDS row `row`: c ^ swz(row), so that the reads below spread over all banks.
//   contraction along the rows: 8 chunks, XOR with the row
//   across them, PITCH bytes a row: XOR by 32-byte units (16-bit types: a transposed read takes 8 rows x 32 bytes) or 64-byte units (fp32)
template <typename T, bool TR, int PITCH> __device__ __forceinline__ int swz(int row)
{
    if constexpr (!TR) return row & 7;
    else if constexpr (sizeof(T) == 4) return ((row >> 2) & 3) << 2;
    else if constexpr (PITCH == 128) return ((row >> 1 & 1) | (row >> 3 & 1) << 1) << 1;
    else return ((row & 3) | (row >> 3 & 1) << 2) << 1;
}

// Fragments of an operand: 16-row group t of a wave's rows, half kk of the K-tile.  The swizzle is an XOR of address bits that no other term but the group's touches, so a
// lane keeps one address and the group is XORed in (TR) or an immediate offset.
template <typename T, bool TR, int ROWS> struct Reader {
    static constexpr int PITCH = TR ? ROWS * (int)sizeof(T) : 128;
    unsigned lane;
    __device__ __forceinline__ void init(int row0, int l)          // first of the wave's rows
    {
        const int r16 = l & 15, g = l >> 4;
        if constexpr (!TR) lane = (row0 + r16) * 128 + ((g ^ swz<T, false, 128>(r16)) << 4);
        else if constexpr (sizeof(T) == 2) {
            const int k = g * 8 + (r16 >> 2);
            lane = k * PITCH + ((row0 * 2) ^ (swz<T, true, PITCH>(k) << 4)) + (r16 & 3) * 8;
        } else lane = g * 4 * PITCH + ((row0 * 4) ^ (swz<T, true, PITCH>(g * 4) << 4)) + r16 * 4;
    }
    __device__ __forceinline__ Frag<T> get(unsigned tile, int t, int kk) const
    {
        Frag<T> f;
        if constexpr (!TR) f.v = at<decltype(f.v)>((tile + lane) ^ (kk << 6), t * 2048);
        else if constexpr (sizeof(T) == 2) {
            // a group of 16 lanes reads 4 rows of the contraction x 16 columns and gets them transposed: 4 contraction values of one column a lane
            typedef short short4_t __attribute__((ext_vector_type(4)));
            const unsigned a = (tile + lane) ^ (t << 5);
            const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(a + kk * 32 * PITCH));
            const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(a + kk * 32 * PITCH + 4 * PITCH));
            f.v = __builtin_bit_cast(decltype(f.v), __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const unsigned a = (tile + lane) ^ (t << 6);
#pragma unroll
            for (int j = 0; j < 4; ++j) f.v[j] = at<float>(a, (kk * 16 + j) * PITCH);
        }
        return f;
    }
    template <typename V> static __device__ __forceinline__ V at(unsigned a, unsigned off) { return *(__attribute__((address_space(3))) V*)(a + off); }
};

// One operand's share of the K-tiles: N loads of 16 bytes a thread.  A lane keeps its offsets for all K-tiles of a tile (rows and columns that do not exist: past the descriptor's
// range, they come as zeros); from K-tile to K-tile only the descriptor's base moves, and lanes are masked in the last K-tile alone -- with the masks and bases of all
// loads formed every time the 107 scalar instructions in front of each K-tile's products cost 15 % of it.
template <typename T, bool TR, int ROWS, int THREADS, bool PAIR, int HALF> struct Stager {
    static constexpr int N = ROWS * 8 / THREADS, CPR = TR ? ROWS * (int)sizeof(T) / 16 : 8, STEP = THREADS / CPR;      // STEP: LDS rows between a thread's loads
    static constexpr int KT = 128 / (int)sizeof(T);
    static constexpr bool MIXED = PAIR && STEP % (2 * HALF) != 0;       // PAIR: a wave's loads alternate between value and gate rows
    unsigned voff[N];
    const char* base;
    const char* base2;         // MIXED: the gate rows'
    long long step;
    __device__ __forceinline__ int k_of(int j, int tid) const           // first contraction index of load j's chunk within the K-tile
    {
        if constexpr (TR) return j * STEP + tid / CPR;
        else return ((tid & 7) ^ swz<T, false, 128>(tid >> 3)) * kVec<T>;       // STEP is a multiple of 8: the same for all j
    }
    template <typename Map> __device__ __forceinline__ void init(const char* p, long long ld, int valid, int tid, int wid, long long gate, Map&& map)
    {
        base = p + (PAIR && !MIXED && wid * 8 % (2 * HALF) >= HALF ? gate : 0);
        base2 = MIXED ? p + gate : nullptr;
        step = TR ? (long long)KT * ld : 128;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if constexpr (!TR) {
                const int lrow = j * STEP + (tid >> 3), row = map(lrow);
                voff[j] = row < valid ? (unsigned)(row * ld) + (((tid & 7) ^ swz<T, false, 128>(lrow)) << 4) : kOob;
            } else {
                const int k = j * STEP + tid / CPR, c = (tid % CPR) ^ swz<T, true, ROWS * (int)sizeof(T)>(k);
                voff[j] = c * kVec<T> < valid ? (unsigned)(k * ld) + c * 16 : kOob;
            }
        }
    }
    // Load j of the next K-tile; `left`: contraction elements from that K-tile on (none: nothing is brought in).  No branch, so that it can stand among the products
    __device__ __forceinline__ void issue(int j, unsigned lds, int left, int tid)
    {
        const bool two = MIXED && j * STEP % (2 * HALF) >= HALF;
        dma16(make_rsrc(two ? base2 : base), k_of(j, tid) < left ? voff[j] : kOob, lds + j * THREADS * 16);
        if (j == N - 1) {
            base += step;
            if constexpr (MIXED) base2 += step;
        }
    }
};

// sum over the 16 lanes of a row
__device__ __forceinline__ float row16_sum(float v)
{
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x128, 0xf, 0xf, true));   // row_ror:8, 4, 2, 1
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x124, 0xf, 0xf, true));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x122, 0xf, 0xf, true));
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x121, 0xf, 0xf, true));
    return v;
}

// the lane, formed anew: values that only a tile's ends need do not take registers from the products in between (kept, they were spilled, and reading them back waited for the next
// tile's loads)
__device__ __forceinline__ int lane_now()
{
    unsigned all;
    asm volatile("s_mov_b32 %0, -1" : "=s"(all));
    return __builtin_amdgcn_mbcnt_hi(all, __builtin_amdgcn_mbcnt_lo(all, 0));
}

template <typename T, bool TRA, bool TRB, int EPI, int ACT, int CFG>
__global__ __launch_bounds__(TileOf<CFG>::type::threads) void gff_gemm_kernel(GffDev p)
{
    typedef typename TileOf<CFG>::type C;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int KT = 128 / sizeof(T);         // contraction elements of a K-tile
    constexpr bool PAIR = EPI == GFF_FWD || EPI == GFF_BWD;
    constexpr int HALF = C::NT * 8;             // PAIR: value columns of a wave, then as many gate columns
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wr = wid / C::WN, wc = wid % C::WN;
    // only the largest tile's pair kernels lack the registers to keep it: 163 -> 156 us for fp16 65536 x 320 -> 1280; a small tile would pay for it (2 x 1280 -> 5120: 10.1 -> 10.8)
    constexpr bool ANEW = PAIR && CFG == 0;
    auto tid_now = [&]() -> int { return ANEW ? wid * 64 + lane_now() : (int)threadIdx.x; };
    const int nk_all = (p.Kc + KT - 1) / KT, units = p.nbm * p.nbn * p.splits;

    int tm = 0, tn = 0, ks = 0, kt0 = 0, kt1 = 0;
    auto unit = [&](int u) {
        // workgroups b, b + 8, ... share an XCD and its L2: each XCD gets a contiguous run of tiles
        const int q = units >> 3, r = units & 7, xcd = u & 7, i = u >> 3;
        u = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + i;
        ks = u % p.splits;
        u /= p.splits;
        tm = u / p.nbn;
        tn = u - tm * p.nbn;
        kt0 = (int)((long long)nk_all * ks / p.splits);
        kt1 = (int)((long long)nk_all * (ks + 1) / p.splits);
    };

    Stager<T, TRA, C::BM, C::threads, false, 0> sa;
    Stager<T, TRB, C::BN, C::threads, PAIR, HALF> sb;
    constexpr int NA = decltype(sa)::N, NB = decltype(sb)::N;
    auto same = [](int r) { return r; };
    auto aim = [&]() {                          // both operands at the unit's first K-tile
        const int tid = tid_now();
        const long long m0 = (long long)tm * C::BM, n0 = (long long)tn * (PAIR ? C::BN / 2 : C::BN);
        if constexpr (TRA) sa.init(p.A + m0 * sizeof(T) + (long long)kt0 * KT * p.ldA, p.ldA, (int)min((long long)C::BM, p.rowsA - m0), tid, wid, 0, same);
        else sa.init(p.A + m0 * p.ldA + (long long)kt0 * 128, p.ldA, (int)min((long long)C::BM, p.rowsA - m0), tid, wid, 0, same);
        if constexpr (PAIR) {
            // LDS rows of a wave column: HALF value rows, then the gate rows of the same columns.  16-row product nt leaves rows 4g .. 4g + 3 with lane group g:
            // operand rows are permuted so that a group's rows of all products are adjacent columns of h (16-byte stores for 16-bit types).
            sb.init(p.B + n0 * p.ldB + (long long)kt0 * 128, p.ldB, (int)min((long long)(C::BN / 2), p.F - n0), tid, wid, p.gate, [](int r) {
                const int w = r / (2 * HALF), v = r % HALF;
                return w * HALF + ((v >> 2) & 3) * (HALF / 4) + (v >> 4) * 4 + (v & 3);
            });
        } else if constexpr (TRB) sb.init(p.B + n0 * sizeof(T) + (long long)kt0 * KT * p.ldB, p.ldB, (int)min((long long)C::BN, p.rowsB - n0), tid, wid, 0, same);
        else sb.init(p.B + n0 * p.ldB + (long long)kt0 * 128, p.ldB, (int)min((long long)C::BN, p.rowsB - n0), tid, wid, 0, same);
    };
    const unsigned smem0 = (unsigned)(unsigned long long)(__attribute__((address_space(3))) char*)smem, lds0 = smem0 + wid * 1024;
    Reader<T, TRA, C::BM> ra;
    Reader<T, TRB, C::BN> rb;
    ra.init(wr * C::MT * 16, ANEW ? lane_now() : (int)threadIdx.x & 63);
    rb.init(wc * C::NT * 16, ANEW ? lane_now() : (int)threadIdx.x & 63);
    auto issue = [&](int j, int left, int slot, int tid) {            // the 2 N loads of a K-tile, A's first
        if (j < NA) sa.issue(j, lds0 + slot * C::stage, left, tid);
        else if (j < NA + NB) sb.issue(j - NA, lds0 + slot * C::stage + C::a_bytes, left, tid);
    };

    int slot = 0;
    bool arrived = false;                       // this thread's share of the K-tile in `slot` has been waited for
    if ((int)blockIdx.x >= units) return;
    unit(blockIdx.x);
    aim();
#pragma unroll
    for (int j = 0; j < NA + NB; ++j) issue(j, p.Kc - kt0 * KT, 0, tid_now());
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
        unit(u);
        const int tm_ = tm, tn_ = tn, ks_ = ks, k0 = kt0, k1 = kt1;
        floatx4 acc[C::NT][C::MT];
#pragma unroll
        for (int a = 0; a < C::NT; ++a)
#pragma unroll
            for (int b = 0; b < C::MT; ++b) acc[a][b] = floatx4{0.f, 0.f, 0.f, 0.f};
        for (int kt = k0; kt < k1; ++kt) {
            if (!arrived) wait_loads();
            arrived = false;
            meet();                        // the K-tile in `slot` is whole, the other stage has been read
            int left = p.Kc - (kt + 1) * KT;
            if (kt + 1 == k1) {
                left = 0;
                if (u + (int)gridDim.x < units) {
                    unit(u + gridDim.x);
                    aim();
                    left = p.Kc - kt0 * KT;
                }
            }
            const unsigned a = smem0 + slot * C::stage, b = a + C::a_bytes;
            slot ^= 1;
            const int tid = tid_now();
            // Four phases of a quarter of the products (half the rows, half the K-tile); each reads the fragments of the next one in front of its own products, the first two
            // bring in half of the next K-tile each, so that the matrix unit has work while both are under way.  All loads in the first phase: 5 % slower, a quarter in each
            // phase: up to 6 % (the last ones are waited for too soon).
            constexpr int MH = C::MT / 2, Q = (NA + NB + 1) / 2;
            Frag<T> bf[2][C::NT], af[2][MH];
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt) bf[0][nt] = rb.get(b, nt, 0);
#pragma unroll
            for (int mt = 0; mt < MH; ++mt) af[0][mt] = ra.get(a, mt, 0);
#pragma unroll
            for (int ph = 0; ph < 4; ++ph) {
                const int kk = ph >> 1, mh = ph & 1;
                if (ph < 3) {
#pragma unroll
                    for (int mt = 0; mt < MH; ++mt) af[(ph + 1) & 1][mt] = ra.get(a, ((ph + 1) & 1) * MH + mt, (ph + 1) >> 1);
                }
                if (ph == 1) {
#pragma unroll
                    for (int nt = 0; nt < C::NT; ++nt) bf[1][nt] = rb.get(b, nt, 1);
                }
#pragma unroll
                for (int j = 0; j < Q; ++j) issue(ph * Q + j, left, slot, tid);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int mt = 0; mt < MH; ++mt)
#pragma unroll
                    for (int nt = 0; nt < C::NT; ++nt) acc[nt][mh * MH + mt] = mma(bf[kk][nt], af[ph & 1][mt], acc[nt][mh * MH + mt]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }

        const int lane = tid_now() & 63, fr = lane & 15, fg = lane >> 4;
        const long long m0 = (long long)tm_ * C::BM + wr * C::MT * 16 + fr;
        typedef typename VecOf<T, 4>::type T4;
        if constexpr (PAIR) {
            // a lane holds W columns f .. f + W - 1 of row m0 + 16 mt, values and gates
            constexpr int P = C::NT / 2, W = P * 4;
            const int f = tn_ * (C::BN / 2) + wc * HALF + fg * W;
            const bool okf = f < p.F;            // F is a multiple of W or the rest of a lane is (16-byte steps)
            float bv[W], bg[W];
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const bool in = p.bias && f + i < p.F;
                bv[i] = in ? param_at<T>(p.bias, p.bias_f32, f + i) : 0.0f;
                bg[i] = in ? param_at<T>(p.bias, p.bias_f32, p.F + f + i) : 0.0f;
            }
            T4 d[EPI == GFF_BWD ? C::MT : 1][P];
            if constexpr (EPI == GFF_BWD) {
#pragma unroll
                for (int mt = 0; mt < C::MT; ++mt)
#pragma unroll
                    for (int q = 0; q < P; ++q)
                        if (m0 + mt * 16 < p.rowsA && f + q * 4 < p.F) d[mt][q] = *(const T4*)((const T*)p.dh + (m0 + mt * 16) * p.ld_dh + f + q * 4);
                        else d[mt][q] = T4{};
            }
            float cv[W], cg[W];
#pragma unroll
            for (int i = 0; i < W; ++i) cv[i] = cg[i] = 0.0f;
            T4 o1[C::MT][P], o2[EPI == GFF_BWD ? C::MT : 1][P];
#pragma unroll
            for (int mt = 0; mt < C::MT; ++mt)
#pragma unroll
                for (int q = 0; q < P; ++q)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int i = q * 4 + r;
                        const float a = acc[q][mt][r] + bv[i], g = acc[q + P][mt][r] + bg[i];
                        float act, slope;
                        activation<T, ACT>(g, act, slope);
                        if constexpr (EPI == GFF_FWD) o1[mt][q][r] = (T)(a * act);
                        else {
                            // rounded to the inputs' type once: they are operands of the next two products; the bias gradient takes them unrounded
                            const float dd = (float)d[mt][q][r], da = dd * act, dg = dd * a * slope;
                            if (m0 + mt * 16 < p.rowsA) { cv[i] += da; cg[i] += dg; }
                            o1[mt][q][r] = (T)da;
                            o2[mt][q][r] = (T)dg;
                        }
                    }
            // the next tile's first loads have had the time of the arithmetic above; the stores need not be waited for
            wait_loads();
            arrived = true;
            if (okf) {
#pragma unroll
                for (int mt = 0; mt < C::MT; ++mt) {
                    if (m0 + mt * 16 >= p.rowsA) continue;
                    T* o = (T*)p.out + (m0 + mt * 16) * p.ld_out + f;
                    if constexpr (P == 2 && sizeof(T) == 2) {
                        typedef typename VecOf<T, 8>::type T8;
                        *(T8*)o = __builtin_shufflevector(o1[mt][0], o1[mt][1], 0, 1, 2, 3, 4, 5, 6, 7);
                        if constexpr (EPI == GFF_BWD) *(T8*)(o + p.F) = __builtin_shufflevector(o2[mt][0], o2[mt][1], 0, 1, 2, 3, 4, 5, 6, 7);
                    } else {
#pragma unroll
                        for (int q = 0; q < P; ++q)
                            if (f + q * 4 < p.F) {
                                *(T4*)(o + q * 4) = o1[mt][q];
                                if constexpr (EPI == GFF_BWD) *(T4*)(o + p.F + q * 4) = o2[mt][q];
                            }
                    }
                }
            }
            if constexpr (EPI == GFF_BWD) {
                if (p.colsum) {
#pragma unroll
                    for (int i = 0; i < W; ++i) { cv[i] = row16_sum(cv[i]); cg[i] = row16_sum(cg[i]); }
                    if (fr == 0) {
                        float* c = p.colsum + ((long long)tm_ * C::WM + wr) * 2 * p.F + f;
#pragma unroll
                        for (int q = 0; q < P; ++q)
                            if (f + q * 4 < p.F) {
                                *(floatx4*)(c + q * 4) = floatx4{cv[q * 4], cv[q * 4 + 1], cv[q * 4 + 2], cv[q * 4 + 3]};
                                *(floatx4*)(c + p.F + q * 4) = floatx4{cg[q * 4], cg[q * 4 + 1], cg[q * 4 + 2], cg[q * 4 + 3]};
                            }
                    }
                }
            }
        } else {
            wait_loads();
            arrived = true;
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt) {
                const int n = tn_ * C::BN + wc * C::NT * 16 + nt * 16 + fg * 4;
                if (n >= p.rowsB) continue;          // rowsB is a multiple of 4
#pragma unroll
                for (int mt = 0; mt < C::MT; ++mt) {
                    const long long m = m0 + mt * 16;
                    if (m >= p.rowsA) continue;
                    if constexpr (EPI == GFF_PART) *(floatx4*)(p.part + ((long long)ks_ * p.rowsA + m) * p.rowsB + n) = acc[nt][mt];
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
}

template <typename T, bool TRA, bool TRB, int EPI, int ACT, int CFG> void launch(const OpCtx& c, GffDev& d)
{
    typedef typename TileOf<CFG>::type C;
    constexpr bool PAIR = EPI == GFF_FWD || EPI == GFF_BWD;
    d.nbm = (int)cdiv64(d.rowsA, C::BM);
    d.nbn = (int)cdiv64(PAIR ? d.F : d.rowsB, PAIR ? C::BN / 2 : C::BN);
    auto k = gff_gemm_kernel<T, TRA, TRB, EPI, ACT, CFG>;
    op_allow_lds((const void*)k, C::lds);
    const long long units = (long long)d.nbm * d.nbn * d.splits, fit = CFG == 0 ? 256 : CFG == 1 ? 512 : 1024;     // workgroups that run at once
    k<<<(unsigned)(units < fit ? units : fit), C::threads, C::lds, c.stream>>>(d);
    op_launched("gated feed-forward product");
}
template <typename T, bool TRA, bool TRB, int EPI, int ACT> void by_tile(const OpCtx& c, GffDev& d, int cfg)
{
    if (cfg == 0) launch<T, TRA, TRB, EPI, ACT, 0>(c, d);
    else if (cfg == 1) launch<T, TRA, TRB, EPI, ACT, 1>(c, d);
    else launch<T, TRA, TRB, EPI, ACT, 2>(c, d);
}
template <typename T, int EPI> void by_activation(const OpCtx& c, GffDev& d, int act, int cfg)
{
    if (act == SDE_ACT_GELU) by_tile<T, false, false, EPI, SDE_ACT_GELU>(c, d, cfg);
    else if (act == SDE_ACT_GELU_TANH) by_tile<T, false, false, EPI, SDE_ACT_GELU_TANH>(c, d, cfg);
    else by_tile<T, false, false, EPI, SDE_ACT_SILU>(c, d, cfg);
}
template <typename T> void gff_launch_type(const OpCtx& c, GffDev d, int what, int act, int cfg)
{
    if (what == GFF_X_WT_FWD) by_activation<T, GFF_FWD>(c, d, act, cfg);
    else if (what == GFF_X_WT_BWD) by_activation<T, GFF_BWD>(c, d, act, cfg);
    else if (what == GFF_DAG_W) {
        if (d.splits > 1) by_tile<T, false, true, GFF_PART, 0>(c, d, cfg);
        else by_tile<T, false, true, GFF_STORE, 0>(c, d, cfg);
    } else {
        if (d.splits > 1) by_tile<T, true, true, GFF_PART, 0>(c, d, cfg);
        else by_tile<T, true, true, GFF_STORE, 0>(c, d, cfg);
    }
}

}  // namespace
