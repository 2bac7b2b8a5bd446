// op_xattn.hip — attention of queries to another sequence's keys and values (an encoder's states), and its gradient, as operators of their own.
//
//   s = scale q k^T,  p = softmax of s over the keys that count,  o = p v,  lse = log of the softmax's denominator
//   delta = rowsum(do o),  dp = do v^T,  ds = p (dp - delta):  dq = scale ds k,  dk = scale ds^T q,  dv = p^T do
//
// A key counts if it lies before its sequence's kv_len and its mask byte is not zero; a row counts if it lies before its sequence's q_len.  A row
// without a key that counts gives zeros and no gradient.  What does not count is never brought in (its loads are turned into zeros by the buffer
// range check), so infinities or NaN there cannot spread.
//
// The query heads of one key head are rows of one problem: row rr is query rr / G of head rr % G, so that shared heads read K and V once.
//   forward, dq:  a wave owns 16 QT rows and walks the keys; K and V tiles go from global memory to LDS two stages deep.  s^T = k q^T leaves the
//                 probabilities in the registers as the second operand of the next product; V (K for dq) is read from LDS transposed.
//   dk, dv:       a wave owns 16 KTW keys, K and V stay in registers, tiles of rows pass through LDS in the same way.
// Few rows: the keys are split over blocks, each leaves (o, max, sum) in fp32 and a second kernel joins them.  Few keys: dk and dv are split over
// rows and their fp32 parts joined in order.  No atomics.
#include "ops_device.h"

#include <algorithm>

namespace {

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
    int ragged;                                 // lengths are given: workgroups go to the XCDs in turn, so that one long sequence does not fill one XCD
    float scale, scale2;                        // scale2 = scale log2(e)
};

// bytes of LDS and stages of a kernel whose stage holds two tiles (and `extra` bytes): one stage where two do not fit into 160 KB (fp32 heads past 128)
constexpr int stages_of(int kd, int extra) { return 2 * (2 * kTile * kd * 64 + extra) <= 160 * 1024 - 1024 ? 2 : 1; }

template <typename T> struct Cfg { static constexpr int frag = 64 / (int)sizeof(T); };   // elements of a 64-byte step of a contraction

__device__ __forceinline__ int xcd_chunk(int bid, int n)
{
    const int q = n >> 3, r = n & 7, x = bid & 7, i = bid >> 3;
    return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + i;
}

// LDS tiles: rows of KD x 64 bytes, 16-byte chunks swizzled inside aligned groups so that 8 rows read at one chunk (and 8 rows x 32 bytes in the
// transposed reads) fall on different banks
template <int KD> __device__ __forceinline__ int swz(int row)
{
    if constexpr (KD % 4 == 0) return (row & 7) << 1;
    else if constexpr (KD % 2 == 0) return row & 7;
    else return (row >> 2) & 3;
}
template <typename T, int KD> __device__ __forceinline__ Frag<T> read_rows(const char* tile, int row0, int kk, int lane)
{
    const int row = row0 + (lane & 15);
    Frag<T> f;
    f.v = *(const decltype(f.v)*)(tile + row * (KD * 64) + (((kk * 4 + (lane >> 4)) ^ swz<KD>(row)) << 4));
    return f;
}
// Columns d0 .. d0+15 of the tile as the first operand, contraction over rows in the order the accumulators of a 16-row product leave them:
// 16-bit: element j of lane group g is row 32 s + 16 (j / 4) + 4 g + j % 4; fp32: row 16 s + 4 g + j.
template <typename T, int KD> __device__ __forceinline__ Frag<T> read_cols(const char* tile, int d0, int s, int lane)
{
    const int r16 = lane & 15, g = lane >> 4;
    Frag<T> f;
    if constexpr (sizeof(T) == 2) {
        typedef short short4_t __attribute__((ext_vector_type(4)));
        typedef short short8_t __attribute__((ext_vector_type(8)));
        const int col = d0 + (r16 & 3) * 4;
        short8_t w;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = s * 32 + i * 16 + g * 4 + (r16 >> 2);
            const char* a = tile + row * (KD * 64) + (((col >> 3) ^ swz<KD>(row)) << 4) + (col & 7) * 2;
            const short4_t h = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)a);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[i * 4 + e] = h[e];
        }
        f.v = __builtin_bit_cast(decltype(f.v), w);
    } else {
        const int col = d0 + r16;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int row = s * 16 + g * 4 + j;
            f.v[j] = *(const float*)(tile + row * (KD * 64) + (((col >> 2) ^ swz<KD>(row)) << 4) + (col & 3) * 4);
        }
    }
    return f;
}

// tile of `kTile` rows; `words` says which rows count; row r starts at base + offset(r)
template <typename T, int KD, int NW, typename Off>
__device__ __forceinline__ void stage_tile(const char* base, unsigned lds, unsigned long long words, int D, int tid, Off&& offset)
{
    constexpr int CPR = KD * 4, N = kTile * CPR / (64 * NW);
    static_assert(kTile * CPR % (64 * NW) == 0, "tile divides into whole loads");
    const uintx4 r = make_rsrc(base);
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int L = i * 64 * NW + tid, row = L / CPR, c = (L % CPR) ^ swz<KD>(row);
        const bool ok = ((words >> row) & 1) && c * kVec<T> < D;
        dma16(r, ok ? offset(row) + c * 16 : kOob, lds + (i * NW + wid) * 1024);
    }
}

// the operand of 16 rows a wave keeps in registers; rows that do not count read nothing
template <typename T, int KD> __device__ __forceinline__ void load_rows(Frag<T> (&f)[KD], const char* p, bool ok, int D, int lane)
{
#pragma unroll
    for (int kk = 0; kk < KD; ++kk) {
        const int c = kk * 4 + (lane >> 4);
        if (ok && c * kVec<T> < D) f[kk].v = *(const decltype(f[kk].v)*)(p + c * 16);
        else f[kk].v = decltype(f[kk].v){};
    }
}

__device__ __forceinline__ unsigned long long low_bits(long long n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; }

// second operands from accumulators: kTile contraction values of a wave's 16 columns
template <typename T> struct Probs {
    static constexpr int N = kTile / Cfg<T>::frag;
    Frag<T> f[N];
    __device__ __forceinline__ void set(int t16, int r, float v)          // 16-row product t16, register r
    {
        if constexpr (sizeof(T) == 2) f[t16 >> 1].v[(t16 & 1) * 4 + r] = (T)v;
        else f[t16].v[r] = v;
    }
};

// MODE 0: forward; 1: forward, a part of the keys (splits); 2: dq
template <typename T, int KD, int ND, int NW, int QT, int MODE>
__global__ __launch_bounds__(NW * 64) void xa_rows_kernel(XaDev p)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int TB = kTile * KD * 64;                  // bytes of a tile
    constexpr int STAGES = stages_of(KD, 0);
    constexpr int ROWS = NW * QT * 16;
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int fr = lane & 15, fg = lane >> 4;
    int id = p.ragged ? blockIdx.x : xcd_chunk(blockIdx.x, gridDim.x);
    const int split = id % p.splits; id /= p.splits;
    const int rb = id % p.nrb; id /= p.nrb;
    const int hk = id % p.Hkv, b = id / p.Hkv;

    const int kv_len = p.kv_lens ? min(max(p.kv_lens[b], 0), p.Skv) : p.Skv;
    const int q_len = p.q_lens ? min(max(p.q_lens[b], 0), p.Sq) : p.Sq;
    const int ntiles = (kv_len + kTile - 1) / kTile;
    const int t0 = (int)((long long)ntiles * split / p.splits), t1 = (int)((long long)ntiles * (split + 1) / p.splits);
    const int row0 = rb * ROWS + wid * QT * 16;
    const bool any_rows = rb * ROWS < q_len * p.G;

    int rr[QT], rs[QT], rh[QT];
    bool row_in[QT], row_ok[QT];
    Frag<T> qf[QT][KD], of[MODE == 2 ? QT : 1][KD];
    float lse2[QT], dlt[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        rr[t] = row0 + t * 16 + fr;
        row_in[t] = rr[t] < p.R;
        rs[t] = rr[t] / p.G;
        rh[t] = hk * p.G + (rr[t] - rs[t] * p.G);
        row_ok[t] = row_in[t] && rs[t] < q_len;
        load_rows<T, KD>(qf[t], p.q.p + b * p.q.b + rs[t] * p.q.s + rh[t] * p.q.h, row_ok[t], p.D, lane);
        lse2[t] = 0.0f;
        dlt[t] = 0.0f;
        if constexpr (MODE == 2) {
            Frag<T> out[KD];
            load_rows<T, KD>(of[t], p.dO.p + b * p.dO.b + rs[t] * p.dO.s + rh[t] * p.dO.h, row_ok[t], p.D, lane);
            load_rows<T, KD>(out, p.o.p + b * p.o.b + rs[t] * p.o.s + rh[t] * p.o.h, row_ok[t], p.D, lane);
#pragma unroll
            for (int kk = 0; kk < KD; ++kk)
#pragma unroll
                for (int e = 0; e < kVec<T>; ++e) dlt[t] = fmaf((float)of[t][kk].v[e], (float)out[kk].v[e], dlt[t]);
            dlt[t] += __shfl_xor(dlt[t], 16);
            dlt[t] += __shfl_xor(dlt[t], 32);
            const long long at = ((long long)b * p.Sq + rs[t]) * p.H + rh[t];
            const float l = row_ok[t] ? p.lse[at] : INFINITY;
            lse2[t] = l == -INFINITY ? INFINITY : l * kLog2e;              // a row without keys: every probability becomes 0
            if (row_in[t] && fg == 0) p.delta[at] = dlt[t];
        }
    }

    floatx4 acc[ND][QT];
    float m[QT], l[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        m[t] = -INFINITY;
        l[t] = 0.0f;
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d][t] = floatx4{0.f, 0.f, 0.f, 0.f};
    }

    const char* kb = p.k.p + b * p.k.b + hk * p.k.h;
    const char* vb = p.v.p + b * p.v.b + hk * p.v.h;
    const unsigned char* mb = p.mask ? p.mask + b * p.mask_b : nullptr;
    const unsigned lds0 = (unsigned)(unsigned long long)(__attribute__((address_space(3))) char*)smem;
    auto mask_byte = [&](int t) -> int {          // of key 64 t + lane
        const long long key = (long long)t * kTile + lane;
        return mb && t < t1 && key < kv_len ? mb[key] : 1;
    };
    auto word_of = [&](int t, int byte) { return __ballot(byte != 0) & low_bits((long long)kv_len - (long long)t * kTile); };
    auto issue = [&](int t, int slot, unsigned long long w) {
        const unsigned lds = lds0 + slot * 2 * TB;
        stage_tile<T, KD, NW>(kb + (long long)t * kTile * p.k.s, lds, w, p.D, tid, [&](int r) { return (unsigned)(r * p.k.s); });
        stage_tile<T, KD, NW>(vb + (long long)t * kTile * p.v.s, lds + TB, w, p.D, tid, [&](int r) { return (unsigned)(r * p.v.s); });
    };

    if constexpr (MODE == 2) {
        if (!p.dq.p) return;                      // dk / dv alone: delta is all they need from here
    }
    if (any_rows && t0 < t1) {
        unsigned long long word = word_of(t0, mask_byte(t0)), next = 0;
        int byte = mask_byte(t0 + 1);
        issue(t0, 0, word);
        for (int t = t0; t < t1; ++t) {
            wait_loads();
            meet();
            if (t + 1 < t1) {
                next = word_of(t + 1, byte);
                byte = mask_byte(t + 2);
                if constexpr (STAGES == 2) issue(t + 1, (t + 1 - t0) & 1, next);
            }
            const char* tk = smem + (STAGES == 2 ? ((t - t0) & 1) * 2 * TB : 0);
            const char* tv = tk + TB;
            if (word) {
                floatx4 s[4][QT];
#pragma unroll
                for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
                    for (int q = 0; q < QT; ++q) s[kt][q] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int kk = 0; kk < KD; ++kk) {
                        const Frag<T> kf = read_rows<T, KD>(tk, kt * 16, kk, lane);
#pragma unroll
                        for (int q = 0; q < QT; ++q) s[kt][q] = mma(kf, qf[q][kk], s[kt][q]);
                    }
                }
                Probs<T> pf[QT];
                if constexpr (MODE < 2) {
                    if (word != ~0ull) {
#pragma unroll
                        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const bool on = (word >> (kt * 16 + fg * 4 + r)) & 1;
#pragma unroll
                                for (int q = 0; q < QT; ++q) s[kt][q][r] = on ? s[kt][q][r] : -INFINITY;
                            }
                    }
#pragma unroll
                    for (int q = 0; q < QT; ++q) {
                        float top = -INFINITY;
#pragma unroll
                        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                            for (int r = 0; r < 4; ++r) top = fmaxf(top, s[kt][q][r] * p.scale2);
                        top = fmaxf(top, __shfl_xor(top, 16));
                        top = fmaxf(top, __shfl_xor(top, 32));
                        const float mn = fmaxf(m[q], top);
                        const float use = mn == -INFINITY ? 0.0f : mn;
                        const float alpha = __builtin_amdgcn_exp2f(m[q] - use);
                        m[q] = mn;
                        float sum = 0.0f;
#pragma unroll
                        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const float e = __builtin_amdgcn_exp2f(fmaf(s[kt][q][r], p.scale2, -use));
                                sum += e;
                                pf[q].set(kt, r, e);      // rounded to the inputs' type: the operand of the product with v; the sum takes it unrounded
                            }
                        l[q] = fmaf(l[q], alpha, sum);
#pragma unroll
                        for (int d = 0; d < ND; ++d) acc[d][q] *= alpha;
                    }
                } else {
#pragma unroll
                    for (int kt = 0; kt < 4; ++kt) {
                        floatx4 dp[QT];
#pragma unroll
                        for (int q = 0; q < QT; ++q) dp[q] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int kk = 0; kk < KD; ++kk) {
                            const Frag<T> vf = read_rows<T, KD>(tv, kt * 16, kk, lane);
#pragma unroll
                            for (int q = 0; q < QT; ++q) dp[q] = mma(vf, of[q][kk], dp[q]);
                        }
#pragma unroll
                        for (int q = 0; q < QT; ++q)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const bool on = (word >> (kt * 16 + fg * 4 + r)) & 1;
                                const float e = __builtin_amdgcn_exp2f(fmaf(s[kt][q][r], p.scale2, -lse2[q]));
                                pf[q].set(kt, r, on ? e * (dp[q][r] - dlt[q]) : 0.0f);
                            }
                    }
                }
                const char* tc = MODE == 2 ? tk : tv;
#pragma unroll
                for (int s2 = 0; s2 < Probs<T>::N; ++s2)
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        const Frag<T> cf = read_cols<T, KD>(tc, d * 16, s2, lane);
#pragma unroll
                        for (int q = 0; q < QT; ++q) acc[d][q] = mma(cf, pf[q].f[s2], acc[d][q]);
                    }
            }
            word = next;
            if constexpr (STAGES == 1) {
                meet();
                if (t + 1 < t1) issue(t + 1, 0, word);
            }
        }
    }

    // a lane holds columns d = 16 i + 4 fg .. + 3 of row rr
    typedef typename VecOf<T, 4>::type T4;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        if constexpr (MODE < 2) {
            l[t] += __shfl_xor(l[t], 16);
            l[t] += __shfl_xor(l[t], 32);
        }
        if (!row_in[t]) continue;
        if constexpr (MODE == 1) {
            const long long at = ((long long)split * p.B * p.Hkv + (long long)b * p.Hkv + hk) * p.R + rr[t];
            if (fg == 0) { p.part_ml[at * 2] = m[t]; p.part_ml[at * 2 + 1] = l[t]; }
#pragma unroll
            for (int d = 0; d < ND; ++d) *(floatx4*)(p.part_o + at * (ND * 16) + d * 16 + fg * 4) = acc[d][t];
        } else {
            float by = p.scale;
            if constexpr (MODE == 0) {
                by = l[t] > 0.0f ? 1.0f / l[t] : (l[t] == 0.0f ? 0.0f : l[t]);      // a NaN stays one
                if (p.lse && fg == 0) p.lse[((long long)b * p.Sq + rs[t]) * p.H + rh[t]] = l[t] == 0.0f || !row_ok[t] ? -INFINITY : (m[t] + __builtin_amdgcn_logf(l[t])) * kLn2;
            }
            const Strided& out = MODE == 0 ? p.o : p.dq;
            T* o = (T*)(out.p + b * out.b + rs[t] * out.s + rh[t] * out.h);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const int c = d * 16 + fg * 4;
                if (c >= p.D) continue;                  // D is a multiple of 4
                T4 w;
#pragma unroll
                for (int r = 0; r < 4; ++r) w[r] = (T)(row_ok[t] ? acc[d][t][r] * by : 0.0f);
                *(T4*)(o + c) = w;
            }
        }
    }
}

// joins the parts of a row: a wave to a row
template <typename T> __global__ __launch_bounds__(256) void xa_join_kernel(XaDev p, int dpad)
{
    const long long total = (long long)p.B * p.Hkv * p.R;
    const int lane = threadIdx.x & 63;
    for (long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); i < total; i += (long long)gridDim.x * 4) {
        const int rr = (int)(i % p.R), hk = (int)(i / p.R % p.Hkv), b = (int)(i / p.R / p.Hkv);
        const int s = rr / p.G, h = hk * p.G + rr % p.G;
        const bool ok = !p.q_lens || s < p.q_lens[b];
        float m = -INFINITY;
        for (int k = lane; k < p.splits; k += 64) m = fmaxf(m, p.part_ml[(k * total + i) * 2]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        const float use = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, acc[4] = {0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < p.splits; ++k) {
            const float* ml = p.part_ml + (k * total + i) * 2;
            const float w = __builtin_amdgcn_exp2f(ml[0] - use);
            l = fmaf(ml[1], w, l);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (lane + j * 64 < p.D) acc[j] = fmaf(p.part_o[(k * total + i) * dpad + lane + j * 64], w, acc[j]);
        }
        const float by = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
        T* o = (T*)(p.o.p + b * p.o.b + s * p.o.s + h * p.o.h);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (lane + j * 64 < p.D) o[lane + j * 64] = (T)(ok ? acc[j] * by : 0.0f);
        if (p.lse && lane == 0) p.lse[((long long)b * p.Sq + s) * p.H + h] = l == 0.0f || !ok ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kLn2;
    }
}

template <typename T, int KD, int ND, int NW, int KTW>
__global__ __launch_bounds__(NW * 64) void xa_keys_kernel(XaDev p)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int TB = kTile * KD * 64, STAGE = 2 * TB + 2 * kTile * 4, STAGES = stages_of(KD, 2 * kTile * 4);      // Q and dO tiles, then lse and delta of the rows
    constexpr int KEYS = NW * KTW * 16;
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int fr = lane & 15, fg = lane >> 4;
    int id = p.ragged ? blockIdx.x : xcd_chunk(blockIdx.x, gridDim.x);
    const int split = id % p.splits; id /= p.splits;
    const int kbk = id % p.nkb; id /= p.nkb;
    const int hk = id % p.Hkv, b = id / p.Hkv;
    const int kv_len = p.kv_lens ? min(max(p.kv_lens[b], 0), p.Skv) : p.Skv;
    const int q_len = p.q_lens ? min(max(p.q_lens[b], 0), p.Sq) : p.Sq;
    const int rows = q_len * p.G, ntiles = (rows + kTile - 1) / kTile;
    const int t0 = (int)((long long)ntiles * split / p.splits), t1 = (int)((long long)ntiles * (split + 1) / p.splits);

    int key[KTW];
    bool key_ok[KTW];
    Frag<T> kf[KTW][KD], vf[KTW][KD];
    floatx4 ak[ND][KTW], av[ND][KTW];
#pragma unroll
    for (int j = 0; j < KTW; ++j) {
        key[j] = kbk * KEYS + (wid * KTW + j) * 16 + fr;
        key_ok[j] = key[j] < kv_len && (!p.mask || p.mask[b * p.mask_b + key[j]]);
        load_rows<T, KD>(kf[j], p.k.p + b * p.k.b + key[j] * p.k.s + hk * p.k.h, key_ok[j], p.D, lane);
        load_rows<T, KD>(vf[j], p.v.p + b * p.v.b + key[j] * p.v.s + hk * p.v.h, key_ok[j], p.D, lane);
#pragma unroll
        for (int d = 0; d < ND; ++d) { ak[d][j] = floatx4{0.f, 0.f, 0.f, 0.f}; av[d][j] = floatx4{0.f, 0.f, 0.f, 0.f}; }
    }

    const char* qb = p.q.p + b * p.q.b + (long long)hk * p.G * p.q.h;
    const char* ob = p.dO.p + b * p.dO.b + (long long)hk * p.G * p.dO.h;
    const unsigned lds0 = (unsigned)(unsigned long long)(__attribute__((address_space(3))) char*)smem;
    float row_lse = 0.0f, row_delta = 0.0f;
    auto issue = [&](int t, int slot) {
        const unsigned lds = lds0 + slot * STAGE;
        const int r0 = t * kTile, s0 = r0 / p.G;
        const unsigned long long w = low_bits((long long)rows - r0);
        auto off = [&](const Strided& x) { return [&](int r) { const int s = (r0 + r) / p.G; return (unsigned)((s - s0) * x.s + (r0 + r - s * p.G) * x.h); }; };
        stage_tile<T, KD, NW>(qb + s0 * p.q.s, lds, w, p.D, tid, off(p.q));
        stage_tile<T, KD, NW>(ob + s0 * p.dO.s, lds + TB, w, p.D, tid, off(p.dO));
        if (tid < kTile) {
            const int rr = r0 + tid, s = rr / p.G;
            row_lse = INFINITY;
            row_delta = 0.0f;
            if (rr < rows) {
                const long long at = ((long long)b * p.Sq + s) * p.H + hk * p.G + (rr - s * p.G);
                row_lse = p.lse[at] * kLog2e;
                if (row_lse == -INFINITY) row_lse = INFINITY;
                row_delta = p.delta[at];
            }
        }
    };
    auto settle = [&](int slot) {                // lse and delta of the tile that `issue` asked for
        if (tid < kTile) {
            float* x = (float*)(smem + slot * STAGE + 2 * TB);
            x[tid] = row_lse;
            x[kTile + tid] = row_delta;
        }
    };

    if (kbk * KEYS < kv_len && t0 < t1) {
        issue(t0, 0);
        for (int t = t0; t < t1; ++t) {
            const int slot = STAGES == 2 ? (t - t0) & 1 : 0;
            settle(slot);
            wait_loads();
            meet();
            if constexpr (STAGES == 2) if (t + 1 < t1) issue(t + 1, slot ^ 1);
            const char* tq = smem + slot * STAGE;
            const char* to = tq + TB;
            const float* rl = (const float*)(tq + 2 * TB);
            Probs<T> pp[KTW], ps[KTW];
#pragma unroll
            for (int rt = 0; rt < 4; ++rt) {
                floatx4 s[KTW], dp[KTW];
#pragma unroll
                for (int j = 0; j < KTW; ++j) { s[j] = floatx4{0.f, 0.f, 0.f, 0.f}; dp[j] = floatx4{0.f, 0.f, 0.f, 0.f}; }
#pragma unroll
                for (int kk = 0; kk < KD; ++kk) {
                    const Frag<T> a = read_rows<T, KD>(tq, rt * 16, kk, lane), c = read_rows<T, KD>(to, rt * 16, kk, lane);
#pragma unroll
                    for (int j = 0; j < KTW; ++j) { s[j] = mma(a, kf[j][kk], s[j]); dp[j] = mma(c, vf[j][kk], dp[j]); }
                }
                const floatx4 ls = *(const floatx4*)(rl + rt * 16 + fg * 4), dl = *(const floatx4*)(rl + kTile + rt * 16 + fg * 4);
#pragma unroll
                for (int j = 0; j < KTW; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float e = __builtin_amdgcn_exp2f(fmaf(s[j][r], p.scale2, -ls[r]));
                        pp[j].set(rt, r, key_ok[j] ? e : 0.0f);
                        ps[j].set(rt, r, key_ok[j] ? e * (dp[j][r] - dl[r]) : 0.0f);
                    }
            }
#pragma unroll
            for (int s2 = 0; s2 < Probs<T>::N; ++s2)
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const Frag<T> oc = read_cols<T, KD>(to, d * 16, s2, lane), qc = read_cols<T, KD>(tq, d * 16, s2, lane);
#pragma unroll
                    for (int j = 0; j < KTW; ++j) { av[d][j] = mma(oc, pp[j].f[s2], av[d][j]); ak[d][j] = mma(qc, ps[j].f[s2], ak[d][j]); }
                }
            if constexpr (STAGES == 1) {
                meet();
                if (t + 1 < t1) issue(t + 1, 0);
            }
        }
    }

    typedef typename VecOf<T, 4>::type T4;
#pragma unroll
    for (int j = 0; j < KTW; ++j) {
        if (key[j] >= p.Skv) continue;
        const long long n = (long long)p.B * p.Skv * p.Hkv * p.D;
        float* part = p.part_o ? p.part_o + (long long)split * 2 * n + (((long long)b * p.Skv + key[j]) * p.Hkv + hk) * p.D : nullptr;
        T* ok = (T*)(p.dk.p + b * p.dk.b + key[j] * p.dk.s + hk * p.dk.h);
        T* ov = (T*)(p.dv.p + b * p.dv.b + key[j] * p.dv.s + hk * p.dv.h);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const int c = d * 16 + fg * 4;
            if (c >= p.D) continue;
            const floatx4 gk = ak[d][j] * p.scale, gv = av[d][j];
            if (part) { *(floatx4*)(part + c) = gk; *(floatx4*)(part + n + c) = gv; }
            else {
                T4 wk, wv;
#pragma unroll
                for (int r = 0; r < 4; ++r) { wk[r] = (T)gk[r]; wv[r] = (T)gv[r]; }
                if (p.dk.p) *(T4*)(ok + c) = wk;
                if (p.dv.p) *(T4*)(ov + c) = wv;
            }
        }
    }
}

// dk / dv from their parts, in the order of the splits; blockIdx.y: dk, dv
template <typename T> __global__ __launch_bounds__(256) void xa_keys_join_kernel(XaDev p)
{
    typedef typename VecOf<T, 4>::type T4;
    const Strided& out = blockIdx.y ? p.dv : p.dk;
    if (!out.p) return;
    const long long n = (long long)p.B * p.Skv * p.Hkv * p.D;
    for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (long long)gridDim.x * 1024) {
        floatx4 s = *(const floatx4*)(p.part_o + blockIdx.y * n + i);
        for (int k = 1; k < p.splits; ++k) s += *(const floatx4*)(p.part_o + ((long long)k * 2 + blockIdx.y) * n + i);
        const int d = (int)(i % p.D), hk = (int)(i / p.D % p.Hkv);
        const long long bk = i / p.D / p.Hkv;
        T4 w;
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] = (T)s[r];
        *(T4*)((T*)(out.p + bk / p.Skv * out.b + bk % p.Skv * out.s + hk * out.h) + d) = w;
    }
}

// rows without keys (or no keys at all): zeros, lse -inf
template <typename T> __global__ __launch_bounds__(256) void xa_zero_kernel(Strided x, int S, int H, int D, long long n, float* lse)
{
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        const long long bs = i / D / H;
        const int h = (int)(i / D % H), d = (int)(i % D);
        if (x.p) ((T*)(x.p + bs / S * x.b + bs % S * x.s + h * x.h))[d] = (T)0.0f;
        if (lse && d == 0) lse[bs * H + h] = -INFINITY;
    }
}
template <typename T> void xa_zero(const OpCtx& c, const Strided& x, int B, int S, int H, int D, float* lse)
{
    const long long n = (long long)B * S * H * D;
    if (n == 0 || (!x.p && !lse)) return;
    xa_zero_kernel<T><<<(unsigned)std::min<long long>(cdiv64(n, 256), 4096), 256, 0, c.stream>>>(x, S, H, D, n, lse);
    op_launched("cross attention zeros");
}

// ---- variants.  KD: 64-byte steps of the head dimension, ND: 16-column steps of it.  The fp32 head dimension needs twice the bytes, so its waves own half the rows.
struct XaShape { int kd, nd; };
XaShape xa_shape(const sde_cross_attention_args& a)
{
    const int step = a.dtype == SDE_F32 ? 16 : 32;
    int kd = cdiv((int)a.D, step), nd = cdiv((int)a.D, 16);
    if (a.dtype == SDE_F32) {
        kd = nd = nd <= 2 ? 2 : nd <= 4 ? 4 : nd <= 5 ? 5 : nd <= 8 ? 8 : nd <= 10 ? 10 : 16;
    } else {
        kd = kd <= 5 ? kd : kd <= 6 ? 6 : 8;
        nd = nd == 3 || nd == 5 ? nd : 2 * kd;
    }
    return {kd, nd};
}
template <typename F> void xa_with_shape(const sde_cross_attention_args& a, F&& f)
{
    const XaShape s = xa_shape(a);
#define XA_CASE(T, KD, ND) if (s.kd == KD && s.nd == ND) { f(T{}, std::integral_constant<int, KD>{}, std::integral_constant<int, ND>{}); return; }
#define XA_16(T) XA_CASE(T, 1, 2) XA_CASE(T, 2, 3) XA_CASE(T, 2, 4) XA_CASE(T, 3, 5) XA_CASE(T, 3, 6) XA_CASE(T, 4, 8) XA_CASE(T, 5, 10) XA_CASE(T, 6, 12) XA_CASE(T, 8, 16)
    if (a.dtype == SDE_F16) { XA_16(half_t) }
    else if (a.dtype == SDE_BF16) { XA_16(bf16_t) }
    else { XA_CASE(float, 2, 2) XA_CASE(float, 4, 4) XA_CASE(float, 5, 5) XA_CASE(float, 8, 8) XA_CASE(float, 10, 10) XA_CASE(float, 16, 16) }
#undef XA_16
#undef XA_CASE
    sde_fail(SDE_ERR_INVALID_ARGUMENT, "cross attention: no kernel for this head size");
}

struct XaPlan { int nw, qt, nrb, splits; int ktw, nkb, key_splits; XaShape shape; };
XaPlan xa_plan(const sde_cross_attention_args& a)
{
    XaPlan p{};
    p.shape = xa_shape(a);
    const int64_t R = a.Sq * (a.H / a.Hkv), heads = a.B * a.Hkv, ktiles = cdiv64(a.Skv, kTile);
    p.nw = R <= 32 ? 1 : 4;
    p.qt = p.nw == 1 ? (R <= 16 ? 1 : 2) : 2;
    if (p.shape.kd >= 8) p.qt = 1;
    p.nrb = (int)cdiv64(R, p.nw * p.qt * 16);
    // the keys are split when the rows leave CUs idle: to about 8 waves for each CU, at least 2 tiles a part
    const int64_t blocks = heads * p.nrb, want = p.nw == 1 ? 2048 : 512;
    p.splits = 1;
    if (blocks < 256 || (p.nw == 1 && blocks < want)) p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({want / blocks, ktiles / 2, 64}));
    p.ktw = p.shape.kd >= 5 ? 1 : 2;
    if (a.dtype == SDE_F32 && p.shape.kd >= 4) p.ktw = 1;
    p.nkb = (int)cdiv64(a.Skv, 4 * p.ktw * 16);
    const int64_t kblocks = heads * p.nkb, rtiles = cdiv64(R, kTile);
    p.key_splits = kblocks >= 512 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>({cdiv64(512, kblocks), rtiles, 64}));
    return p;
}

Strided strided(const void* p, const int64_t* s, int e) { return Strided{(const char*)p, s[0] * e, s[1] * e, s[2] * e}; }

XaDev xa_dev(const sde_cross_attention_args& a)
{
    const int e = (int)op_esize(a.dtype);
    XaDev d{};
    d.q = strided(a.q, a.q_stride, e); d.k = strided(a.k, a.k_stride, e); d.v = strided(a.v, a.v_stride, e); d.o = strided(a.o, a.o_stride, e);
    d.dO = strided(a.d_o, a.do_stride, e); d.dq = strided(a.dq, a.dq_stride, e); d.dk = strided(a.dk, a.dk_stride, e); d.dv = strided(a.dv, a.dv_stride, e);
    d.q_lens = a.q_lens; d.kv_lens = a.kv_lens; d.mask = a.key_mask; d.mask_b = a.key_mask_stride;
    d.lse = a.lse;
    d.B = (int)a.B; d.Sq = (int)a.Sq; d.Skv = (int)a.Skv; d.H = (int)a.H; d.Hkv = (int)a.Hkv; d.G = (int)(a.H / a.Hkv); d.D = (int)a.D; d.R = d.Sq * d.G;
    d.scale = a.scale; d.scale2 = a.scale * kLog2e;
    d.splits = 1;
    d.ragged = a.q_lens || a.kv_lens;
    return d;
}

template <typename T, int KD, int ND, int NW, int QT, int MODE> void xa_rows(const OpCtx& c, const XaDev& d)
{
    constexpr int smem = stages_of(KD, 0) * 2 * kTile * KD * 64;
    auto k = xa_rows_kernel<T, KD, ND, NW, QT, MODE>;
    op_allow_lds((const void*)k, smem);
    k<<<(unsigned)((long long)d.B * d.Hkv * d.nrb * d.splits), NW * 64, smem, c.stream>>>(d);
    op_launched("cross attention");
}
template <typename T, int KD, int ND, int MODE> void xa_rows_by(const OpCtx& c, const XaPlan& p, const XaDev& d)
{
    if (p.nw == 1) {
        if (p.qt == 1) xa_rows<T, KD, ND, 1, 1, MODE>(c, d);
        else if constexpr (KD < 8) xa_rows<T, KD, ND, 1, 2, MODE>(c, d);
    } else {
        if (p.qt == 1) { if constexpr (KD >= 8) xa_rows<T, KD, ND, 4, 1, MODE>(c, d); }
        else if constexpr (KD < 8) xa_rows<T, KD, ND, 4, 2, MODE>(c, d);
    }
}

}  // namespace

size_t op_cross_attention_ws_bytes(const sde_cross_attention_args& a, bool backward)
{
    const int64_t rows = a.B * a.Sq * a.H;
    if (!rows || !a.Skv) return 0;
    const XaPlan p = xa_plan(a);
    if (!backward) return p.splits > 1 ? op_align((size_t)p.splits * rows * p.shape.nd * 16 * 4) + op_align((size_t)p.splits * rows * 2 * 4) : 0;
    return op_align((size_t)rows * 4) + (p.key_splits > 1 ? op_align((size_t)p.key_splits * 2 * a.B * a.Skv * a.Hkv * a.D * 4) : 0);
}

void op_cross_attention_forward(const OpCtx& c, const sde_cross_attention_args& a)
{
    if (a.B * a.Sq * a.H == 0) return;
    XaDev d = xa_dev(a);
    if (a.Skv == 0) {
        op_dispatch(a.dtype, [&](auto t) { xa_zero<decltype(t)>(c, d.o, d.B, d.Sq, d.H, d.D, d.lse); });
        return;
    }
    const XaPlan p = xa_plan(a);
    d.nrb = p.nrb;
    d.splits = p.splits;
    xa_with_shape(a, [&](auto t, auto kd, auto nd) {
        typedef decltype(t) T;
        constexpr int KD = decltype(kd)::value, ND = decltype(nd)::value;
        if (p.splits == 1) { xa_rows_by<T, KD, ND, 0>(c, p, d); return; }
        const long long rows = (long long)a.B * a.Sq * a.H;
        d.part_o = (float*)c.ws;
        d.part_ml = (float*)(c.ws + op_align((size_t)p.splits * rows * ND * 16 * 4));
        xa_rows_by<T, KD, ND, 1>(c, p, d);
        xa_join_kernel<T><<<(unsigned)std::min<long long>(cdiv64(rows, 4), 8192), 256, 0, c.stream>>>(d, ND * 16);
        op_launched("cross attention join");
    });
}

void op_cross_attention_backward(const OpCtx& c, const sde_cross_attention_args& a)
{
    XaDev d = xa_dev(a);
    if (a.B * a.Sq * a.H == 0 || a.Skv == 0) {
        op_dispatch(a.dtype, [&](auto t) {
            xa_zero<decltype(t)>(c, d.dq, d.B, d.Sq, d.H, d.D, nullptr);
            xa_zero<decltype(t)>(c, d.dk, d.B, d.Skv, d.Hkv, d.D, nullptr);
            xa_zero<decltype(t)>(c, d.dv, d.B, d.Skv, d.Hkv, d.D, nullptr);
        });
        return;
    }
    const XaPlan p = xa_plan(a);
    const long long rows = (long long)a.B * a.Sq * a.H;
    d.delta = (float*)c.ws;
    d.nrb = p.nrb;
    xa_with_shape(a, [&](auto t, auto kd, auto nd) {
        typedef decltype(t) T;
        constexpr int KD = decltype(kd)::value, ND = decltype(nd)::value;
        constexpr int KTW = (sizeof(T) == 4 ? KD >= 4 : KD >= 5) ? 1 : 2;
        xa_rows_by<T, KD, ND, 2>(c, p, d);
        if (!a.dk && !a.dv) return;
        d.nkb = p.nkb;
        d.splits = p.key_splits;
        if (p.key_splits > 1) d.part_o = (float*)(c.ws + op_align((size_t)rows * 4));
        constexpr int smem = stages_of(KD, 2 * kTile * 4) * (2 * kTile * KD * 64 + 2 * kTile * 4);
        auto k = xa_keys_kernel<T, KD, ND, 4, KTW>;
        op_allow_lds((const void*)k, smem);
        k<<<(unsigned)((long long)d.B * d.Hkv * d.nkb * d.splits), 256, smem, c.stream>>>(d);
        op_launched("cross attention key gradients");
        if (p.key_splits > 1) {
            const long long n = (long long)a.B * a.Skv * a.Hkv * a.D;
            xa_keys_join_kernel<T><<<dim3((unsigned)std::min<long long>(cdiv64(n, 1024), 4096), 2), 256, 0, c.stream>>>(d);
            op_launched("cross attention key gradients' join");
        }
    });
}
