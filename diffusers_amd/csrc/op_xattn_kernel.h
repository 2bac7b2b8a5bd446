// op_xattn_kernel.h — cross attention's kernels and their launchers, for one element type (op_xattn_{f16,bf16,f32}.hip).
#pragma once
#include "op_xattn.h"
#include "ops_device.h"

#include <algorithm>
#include <type_traits>

namespace {

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
// A lane's LDS addresses.  Where rows are a power of two long the swizzle and the column are XORed into one address per read, on top of the tile's own (which changes from
// tile to tile): the compiler cannot keep an address for every read of the loop in a register of its own, which cost more registers than the fragments.
template <typename T, int KD> struct Reader {
    static constexpr int RB = KD * 64;
    static constexpr bool POW2 = KD == 2 || KD == 4 || KD == 8 || KD == 16;
    unsigned rows_, cols_;
    int r16, g;
    template <typename V> static __device__ __forceinline__ V at(unsigned a) { return *(__attribute__((address_space(3))) V*)a; }
    __device__ __forceinline__ void init(int lane)
    {
        r16 = lane & 15;
        g = lane >> 4;
        rows_ = r16 * RB + ((g ^ swz<KD>(r16)) << 4);
        if constexpr (sizeof(T) == 2) {
            const int row = g * 4 + (r16 >> 2);
            cols_ = row * RB + ((((r16 & 3) >> 1) ^ swz<KD>(row)) << 4) + (r16 & 1) * 8;
        } else cols_ = g * 4 * RB + (((r16 >> 2) ^ swz<KD>(g * 4)) << 4) + (r16 & 3) * 4;
    }
    // 16 rows from 16 t on, 64-byte step kk of them
    __device__ __forceinline__ Frag<T> rows(unsigned tile, int t, int kk) const
    {
        Frag<T> f;
        unsigned a;
        if constexpr (POW2) a = ((tile + rows_) ^ (kk << 6)) + t * 16 * RB;
        else if constexpr (KD % 2) a = tile + rows_ + kk * 64 + t * 16 * RB;
        else a = tile + r16 * RB + (((kk * 4 + g) ^ swz<KD>(r16)) << 4) + t * 16 * RB;
        f.v = at<decltype(f.v)>(a);
        return f;
    }
    // Columns 16 d .. + 15 as the first operand, contraction over rows in the order the accumulators of 16-row products leave them:
    // 16-bit: element j of lane group g is row 32 s + 16 (j / 4) + 4 g + j % 4 (transposed reads); fp32: row 16 s + 4 g + j.
    __device__ __forceinline__ Frag<T> cols(unsigned tile, int d, int s) const
    {
        Frag<T> f;
        if constexpr (sizeof(T) == 2) {
            typedef short short4_t __attribute__((ext_vector_type(4)));
            unsigned a;
            if constexpr (POW2) a = (tile + cols_) ^ (d << 5);
            else {
                const int row = g * 4 + (r16 >> 2);
                constexpr int M = KD % 2 ? 1 : 3;                            // columns the swizzle mixes; the rest is an immediate offset
                a = tile + row * RB + ((((d & M) * 2 + ((r16 & 3) >> 1)) ^ swz<KD>(row)) << 4) + (r16 & 1) * 8 + (d & ~M) * 32;
            }
            const short4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(a + s * 32 * RB));
            const short4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)(a + s * 32 * RB + 16 * RB));
            f.v = __builtin_bit_cast(decltype(f.v), __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (POW2) f.v[j] = at<float>(((tile + cols_) ^ (d << 6) ^ (KD == 2 ? j << 4 : j << 5)) + (s * 16 + j) * RB);
                else if constexpr (KD % 2) f.v[j] = at<float>(tile + cols_ + d * 64 + (s * 16 + j) * RB);
                else f.v[j] = at<float>(tile + (g * 4 + j) * RB + (((d * 4 + (r16 >> 2)) ^ swz<KD>(g * 4 + j)) << 4) + (r16 & 3) * 4 + s * 16 * RB);
            }
        }
        return f;
    }
};

// Brings a tile of kTile rows into LDS.  A lane's offsets are the same for every tile (rows a fixed stride apart); rows that `word` leaves out come as zeros.
template <typename T, int KD, int NW> struct Stager {
    static constexpr int CPR = KD * 4, N = kTile * CPR / (64 * NW);
    static_assert(kTile * CPR % (64 * NW) == 0, "a tile is whole loads");
    unsigned voff[N];
    static __device__ __forceinline__ int row_of(int i, int tid) { return (i * 64 * NW + tid) / CPR; }
    template <typename Off> __device__ __forceinline__ void init(int D, int tid, Off&& offset)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = row_of(i, tid), c = ((i * 64 * NW + tid) % CPR) ^ swz<KD>(row);
            voff[i] = c * kVec<T> < D ? offset(row) + c * 16 : kOob;
        }
    }
    __device__ __forceinline__ void issue(const char* base, unsigned lds, unsigned long long word, int tid, int wid) const
    {
        const uintx4 r = make_rsrc(base);
        if (word == ~0ull) {
#pragma unroll
            for (int i = 0; i < N; ++i) dma16(r, voff[i], lds + (i * NW + wid) * 1024);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) dma16(r, (word >> row_of(i, tid)) & 1 ? voff[i] : kOob, lds + (i * NW + wid) * 1024);
        }
    }
};

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

// Score gradients ds = p (dp - delta) as fp16 operands.  p is about 1 / Skv and the upstream gradient any size, so ds itself lies where fp16 has few bits or none (2^-24 and less: with 8000 keys
// and do of 1e-3 the products with it were 1 % off) or past its largest value.  They go in as 2^n ds, each column of the product (a row for dq, a key for dk) with an n of its own: it starts
// high and comes down, with the sums so far, when a value passes 2^15, to put that value at 2^8 .. 2^9.  Powers of two: exact.  bf16 and fp32 have the range.
// dk / dv: starts at 2^72, the first tile brings it down.  Backward pass of fp16, us before / with: 8 x 2047 x 16 heads of 128 (4 shared) on 1500 keys 908 / 890, 16 x 4096 x 8 of 40 on 77
// 96 / 100, 2 x 4096 x 8 of 40 on 4096 257 / 259.
template <typename T> constexpr bool kScaled = std::is_same_v<T, half_t>;
constexpr float kUpStart = 4.722366482869645e21f, kUpLimit = 32768.0f;       // 2^72: times 2^8 p (dk / dv) and the largest |dp - delta|, twice 256 products of 65504^2, it is still finite
__device__ __forceinline__ unsigned exponent(float m) { return __builtin_bit_cast(unsigned, m) >> 23; }          // of m >= 0: 127 and up from 1, 255 for infinity
__device__ __forceinline__ float to_2_8(unsigned e) { return __builtin_bit_cast(float, (127 + 8 + 127 - e) << 23); }      // brings a value of this exponent to 2^8 .. 2^9
// what a column is multiplied with so that its largest magnitude (this lane's is `m`; a column is lanes l, l + 16, + 32, + 48) fits
__device__ __forceinline__ float fit(float m)
{
    m = fmaxf(m, __shfl_xor(m, 16));
    m = fmaxf(m, __shfl_xor(m, 32));
    return m > kUpLimit ? to_2_8(exponent(m)) : 1.0f;
}

// The sequence with the rank-th most keys (none for sequences without queries).  A workgroup's time goes with its sequence's keys; with the longest first, none starts late: bf16, 8
// ragged sequences of up to 2047 x 16 rows and 1500 keys, forward 107 us in the given order, 100 in this one, 93 with a key head's workgroups on one XCD (below).
__device__ __forceinline__ int by_length(const XaDev& p, int rank, int lane)
{
    int w = 0;
    if (lane < p.B) {
        w = p.kv_lens ? min(max(p.kv_lens[lane], 0), p.Skv) : p.Skv;
        if (p.q_lens && p.q_lens[lane] <= 0) w = 0;
    }
    int at = 0;
    for (int j = 0; j < p.B; ++j) {
        const int other = __builtin_amdgcn_readlane(w, j);
        at += other > w || (other == w && j < lane);
    }
    return __builtin_ctzll(__ballot(lane < p.B && at == rank));          // ranks of the B lanes are all different: one lane has it
}

// MODE 0: forward; 1: forward, a part of the keys (splits); 2: dq.  RES: all keys fit into the stages; they are brought in once and the workgroup walks `rpg` blocks of rows
// over them without another barrier (a prompt of 77 tokens under thousands of image tokens).
// Two waves to a SIMD: with more registers allowed the compiler keeps o in accumulation registers and copies all of it back and forth in every tile.
template <typename T, int KD, int ND, int NW, int QT, int MODE, bool RES>
__global__ __launch_bounds__(NW * 64, xa_waves(sizeof(T) == 4, KD)) void xa_rows_kernel(XaDev p)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    typedef typename VecOf<T, 4>::type T4;
    constexpr int TB = kTile * KD * 64;                  // bytes of a tile
    constexpr int STAGES = stages_of(KD, 0);
    constexpr int ROWS = NW * QT * 16;
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int fr = lane & 15, fg = lane >> 4;
    const int ngroups = RES ? (p.nrb + p.rpg - 1) / p.rpg : p.nrb, per_head = ngroups * p.splits;
    // Workgroups of one key head share its keys through an XCD's L2.  All alike: an XCD gets a contiguous run of them.  Lengths given: key heads go to the XCDs in turn (workgroups
    // i, i + 8, ... share an XCD), the last few that do not make a round of eight one workgroup to an XCD after the other.
    int id = blockIdx.x;
    if (!p.ragged) id = xcd_chunk(id, gridDim.x);
    else if (id < p.B * p.Hkv / 8 * 8 * per_head) {
        const int round = id / (8 * per_head), i = id % (8 * per_head);
        id = (round * 8 + (i & 7)) * per_head + (i >> 3);
    }
    const int split = id % p.splits; id /= p.splits;
    const int group = id % ngroups; id /= ngroups;
    const int hk = id % p.Hkv, b = p.ragged && p.B <= 64 ? by_length(p, id / p.Hkv, lane) : id / p.Hkv;
    const int rb0 = RES ? group * p.rpg : group, rb1 = RES ? min(rb0 + p.rpg, p.nrb) : rb0 + 1;

    const int kv_len = p.kv_lens ? min(max(p.kv_lens[b], 0), p.Skv) : p.Skv;
    const int q_len = p.q_lens ? min(max(p.q_lens[b], 0), p.Sq) : p.Sq;
    const int ntiles = (kv_len + kTile - 1) / kTile;
    const int t0 = (int)((long long)ntiles * split / p.splits), t1 = (int)((long long)ntiles * (split + 1) / p.splits);

    const char* kb = p.k.p + b * p.k.b + hk * p.k.h;
    const char* vb = p.v.p + b * p.v.b + hk * p.v.h;
    const unsigned char* mb = p.mask ? p.mask + b * p.mask_b : nullptr;
    const unsigned lds0 = (unsigned)(unsigned long long)(__attribute__((address_space(3))) char*)smem;
    Reader<T, KD> rd;
    rd.init(lane);
    Stager<T, KD, NW> sk, sv;
    sk.init(p.D, tid, [&](int r) { return (unsigned)(r * p.k.s); });
    sv.init(p.D, tid, [&](int r) { return (unsigned)(r * p.v.s); });
    auto mask_byte = [&](int t) -> int {          // of key 64 t + lane
        const long long key = (long long)t * kTile + lane;
        return mb && t < t1 && key < kv_len ? mb[key] : 1;
    };
    auto word_of = [&](int t, int byte) { return __ballot(byte != 0) & low_bits((long long)kv_len - (long long)t * kTile); };
    auto issue = [&](int t, int slot, unsigned long long w) {
        const unsigned lds = lds0 + slot * 2 * TB;
        sk.issue(kb + (long long)t * kTile * p.k.s, lds, w, tid, wid);
        sv.issue(vb + (long long)t * kTile * p.v.s, lds + TB, w, tid, wid);
    };

    unsigned long long word = 0, next = 0;
    int byte = 1;
    const bool any_rows = rb0 * ROWS < q_len * p.G;
    bool walk = any_rows && t0 < t1;
    if constexpr (MODE == 2) walk = walk && (p.dq.p || ntiles == 1);        // dk / dv alone need delta only, which a single tile of keys gives (below)
    if (walk) {
        word = word_of(t0, mask_byte(t0));
        byte = mask_byte(t0 + 1);
        issue(t0, 0, word);
        if constexpr (RES) {
            if (t0 + 1 < t1) {
                next = word_of(t0 + 1, byte);
                issue(t0 + 1, 1, next);
            }
            wait_loads();
            meet();
        }
    }

    for (int rb = rb0; rb < rb1; ++rb) {
        const int row0 = rb * ROWS + wid * QT * 16;
        int rr[QT], rs[QT], rh[QT];
        bool row_in[QT], row_ok[QT];
        Frag<T> qf[QT][KD], of[MODE == 2 ? QT : 1][KD];
        float lse2[QT], dlt[QT], up[QT];          // up: kScaled
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            rr[t] = row0 + t * 16 + fr;
            row_in[t] = rr[t] < p.R;
            rs[t] = p.G == 1 ? rr[t] : rr[t] / p.G;
            rh[t] = hk * p.G + (rr[t] - rs[t] * p.G);
            row_ok[t] = row_in[t] && rs[t] < q_len;
            load_rows<T, KD>(qf[t], p.q.p + b * p.q.b + rs[t] * p.q.s + rh[t] * p.q.h, row_ok[t], p.D, lane);
            lse2[t] = 0.0f;
            dlt[t] = 0.0f;
            if constexpr (MODE == 2) {
                Frag<T> out[KD];
                load_rows<T, KD>(of[t], p.dO.p + b * p.dO.b + rs[t] * p.dO.s + rh[t] * p.dO.h, row_ok[t], p.D, lane);
                load_rows<T, KD>(out, p.o.p + b * p.o.b + rs[t] * p.o.s + rh[t] * p.o.h, row_ok[t], p.D, lane);
                float size = 0.0f;
#pragma unroll
                for (int kk = 0; kk < KD; ++kk)
#pragma unroll
                    for (int e = 0; e < kVec<T>; ++e) {
                        dlt[t] = fmaf((float)of[t][kk].v[e], (float)out[kk].v[e], dlt[t]);
                        if constexpr (kScaled<T>) size += fabsf((float)of[t][kk].v[e]);
                    }
                if constexpr (kScaled<T>) {
                    // |ds| is at most sum |do| times twice the largest |v|: right at once unless values pass 2^6, when a tile is formed twice
                    size += __shfl_xor(size, 16);
                    size += __shfl_xor(size, 32);
                    up[t] = to_2_8(max(exponent(size), 127u - 24u));
                }
                dlt[t] += __shfl_xor(dlt[t], 16);
                dlt[t] += __shfl_xor(dlt[t], 32);
                const float l = row_ok[t] ? p.lse[((long long)b * p.Sq + rs[t]) * p.H + rh[t]] : INFINITY;
                lse2[t] = l == -INFINITY ? INFINITY : l * kLog2e;              // a row without keys: every probability becomes 0
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

        // One tile.  FULL: all its keys count; otherwise 16-key groups without one are left out and the rest is masked key by key.
        auto tile = [&](auto full_, unsigned long long w, unsigned tk, unsigned tv) __attribute__((always_inline)) {
            constexpr bool FULL = decltype(full_)::value;
            auto group_on = [&](int kt) { return FULL || ((w >> (kt * 16)) & 0xffff) != 0; };
            const unsigned mine[2] = {(unsigned)w >> (fg * 4), (unsigned)(w >> 32) >> (fg * 4)};        // this lane group's keys: bits 0..3 and 16..19
            auto key_on = [&](int kt, int r) { return FULL || ((mine[kt >> 1] >> ((kt & 1) * 16 + r)) & 1) != 0; };
            // 16 keys by the wave's rows: key (value) rows of the tile times q (do)
            auto scores = [&](unsigned tile_, int kt, const Frag<T> (&rows)[QT][KD], floatx4 (&x)[QT]) __attribute__((always_inline)) {
#pragma unroll
                for (int q = 0; q < QT; ++q) x[q] = floatx4{0.f, 0.f, 0.f, 0.f};
                if (group_on(kt)) {
#pragma unroll
                    for (int kk = 0; kk < KD; ++kk) {
                        const Frag<T> f = rd.rows(tile_, kt, kk);
#pragma unroll
                        for (int q = 0; q < QT; ++q) x[q] = mma(f, rows[q][kk], x[q]);
                    }
                }
            };
            // few rows: their time is that of reading the keys, so the probabilities go in as two operands, the rounded value and what rounding took away
            constexpr bool SPLIT = sizeof(T) == 2 && NW == 1 && MODE < 2;
            Probs<T> pf[QT], pl[SPLIT ? QT : 1];
            if constexpr (MODE < 2) {
                floatx4 s[4][QT];
#pragma unroll
                for (int kt = 0; kt < 4; ++kt) {
                    scores(tk, kt, qf, s[kt]);
                    if (kt == 1) __builtin_amdgcn_sched_barrier(0);         // not all fragments of the tile at once: they would push o out of the registers
                }
                float top[QT];
#pragma unroll
                for (int q = 0; q < QT; ++q) top[q] = -INFINITY;
#pragma unroll
                for (int kt = 0; kt < 4; ++kt) {
                    if (!group_on(kt)) continue;
#pragma unroll
                    for (int q = 0; q < QT; ++q)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            if constexpr (!FULL) s[kt][q][r] = key_on(kt, r) ? s[kt][q][r] : -INFINITY;
                            top[q] = fmaxf(top[q], s[kt][q][r]);
                        }
                }
#pragma unroll
                for (int q = 0; q < QT; ++q) {
                    top[q] = fmaxf(top[q], __shfl_xor(top[q], 16));
                    top[q] = fmaxf(top[q], __shfl_xor(top[q], 32)) * p.scale2;
                }
                // The running maximum follows only when a row's has grown by more than 2^8: the terms stay below 2^8 (fp16 holds them) and the sums are
                // right for any reference value; scaling o in every tile was a quarter of the vector instructions.
                bool grow = false;
#pragma unroll
                for (int q = 0; q < QT; ++q) grow = grow || top[q] > m[q] + 8.0f;
                if (__any(grow)) {
#pragma unroll
                    for (int q = 0; q < QT; ++q) {
                        const float mn = fmaxf(m[q], top[q]);
                        const float alpha = mn == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[q] - mn);
                        m[q] = mn;
                        l[q] *= alpha;
#pragma unroll
                        for (int d = 0; d < ND; ++d) acc[d][q] *= alpha;
                    }
                }
                float use[QT];
#pragma unroll
                for (int q = 0; q < QT; ++q) use[q] = m[q] == -INFINITY ? 0.0f : m[q];
#pragma unroll
                for (int kt = 0; kt < 4; ++kt) {
                    if (group_on(kt)) {
                        if constexpr (!FULL) asm volatile("");        // a branch, not 16 exponentials thrown away
#pragma unroll
                        for (int q = 0; q < QT; ++q) {
                            float sum = 0.0f;
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const float e = __builtin_amdgcn_exp2f(fmaf(s[kt][q][r], p.scale2, -use[q]));
                                sum += e;
                                pf[q].set(kt, r, e);      // rounded to the inputs' type: the operand of the product with v; the sum takes it unrounded
                                if constexpr (SPLIT) pl[q].set(kt, r, e - (float)(T)e);
                            }
                            l[q] += sum;
                        }
                    } else {
#pragma unroll
                        for (int q = 0; q < QT; ++q)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                pf[q].set(kt, r, 0.0f);
                                if constexpr (SPLIT) pl[q].set(kt, r, 0.0f);
                            }
                    }
                }
            } else {
                auto prob = [&](const floatx4 (&x)[QT], int kt, int q, int r) { return key_on(kt, r) ? __builtin_amdgcn_exp2f(fmaf(x[q][r], p.scale2, -lse2[q])) : 0.0f; };
                if (ntiles == 1) {
                    // All keys are here: delta = sum of p dp, without the rounding of o.  With few keys that rounding, u |do| |o|, is as large as those of the products'
                    // operands; with many keys o is a mean and it is small, unless one key takes most of a row (bf16, 300 keys: dq is 2.4e-3 off for N(0, 1) scores, 4.6e-3 where the
                    // largest probability is 0.65 on average, 5.9e-3 at 0.83; fp16 3.0e-4, 5.8e-4, 7.7e-4).  A second walk over the keys would take it away, for half as much time again.
                    float d[QT];
#pragma unroll
                    for (int q = 0; q < QT; ++q) d[q] = 0.0f;
#pragma unroll
                    for (int kt = 0; kt < 4; ++kt) {
                        floatx4 s[QT], dp[QT];
                        scores(tk, kt, qf, s);
                        scores(tv, kt, of, dp);
#pragma unroll
                        for (int q = 0; q < QT; ++q)
#pragma unroll
                            for (int r = 0; r < 4; ++r) d[q] = key_on(kt, r) ? fmaf(prob(s, kt, q, r), dp[q][r], d[q]) : d[q];
                    }
#pragma unroll
                    for (int q = 0; q < QT; ++q) {
                        d[q] += __shfl_xor(d[q], 16);
                        dlt[q] = d[q] + __shfl_xor(d[q], 32);
                    }
                }
                float top[QT];
                auto gradients = [&]() __attribute__((always_inline)) {
#pragma unroll
                    for (int q = 0; q < QT; ++q) top[q] = 0.0f;
#pragma unroll
                    for (int kt = 0; kt < 4; ++kt) {
                        if (!group_on(kt)) {
#pragma unroll
                            for (int q = 0; q < QT; ++q)
#pragma unroll
                                for (int r = 0; r < 4; ++r) pf[q].set(kt, r, 0.0f);
                            continue;
                        }
                        floatx4 s[QT], dp[QT];
                        scores(tk, kt, qf, s);
                        scores(tv, kt, of, dp);
#pragma unroll
                        for (int q = 0; q < QT; ++q)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                float x;
                                if constexpr (kScaled<T>) {
                                    x = key_on(kt, r) ? prob(s, kt, q, r) * fmaf(dp[q][r], up[q], -dlt[q] * up[q]) : 0.0f;
                                    top[q] = fmaxf(top[q], fabsf(x));
                                } else x = key_on(kt, r) ? prob(s, kt, q, r) * (dp[q][r] - dlt[q]) : 0.0f;
                                pf[q].set(kt, r, x);
                            }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                };
                if constexpr (kScaled<T>) {
#pragma unroll 1
                    for (int turn = 0; turn < 2; ++turn) {          // a tile with a value that does not fit is formed again; infinities do not fit the second time either
                        gradients();
                        bool past = false;
#pragma unroll
                        for (int q = 0; q < QT; ++q) past = past || top[q] > kUpLimit;
                        if (!__any(past)) break;
#pragma unroll
                        for (int q = 0; q < QT; ++q) {
                            const float by = fit(top[q]);
                            up[q] *= by;
#pragma unroll
                            for (int d = 0; d < ND; ++d) acc[d][q] *= by;
                        }
                    }
                } else gradients();
            }
            const unsigned tc = MODE == 2 ? tk : tv;
#pragma unroll
            for (int s2 = 0; s2 < Probs<T>::N; ++s2) {
                constexpr int GK = 4 / Probs<T>::N;                          // 16-key groups of a step
                bool on = false;
#pragma unroll
                for (int g = 0; g < GK; ++g) on = on || group_on(s2 * GK + g);
                if (on) {
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        const Frag<T> cf = rd.cols(tc, d, s2);
#pragma unroll
                        for (int q = 0; q < QT; ++q) {
                            acc[d][q] = mma(cf, pf[q].f[s2], acc[d][q]);
                            if constexpr (SPLIT) acc[d][q] = mma(cf, pl[q].f[s2], acc[d][q]);
                        }
                    }
                }
            }
        };
        auto one = [&](unsigned long long w, int slot) __attribute__((always_inline)) {
            const unsigned tk = lds0 + slot * 2 * TB;
            if (w == ~0ull) tile(std::true_type{}, w, tk, tk + TB);
            else if (w) tile(std::false_type{}, w, tk, tk + TB);
        };

        if (walk) {
            if constexpr (RES) {
#pragma unroll 1
                for (int slot = 0; slot < 2; ++slot) one(slot ? next : word, slot);
            } else {
                for (int t = t0; t < t1; ++t) {
                    wait_loads();
                    meet();
                    if (t + 1 < t1) {
                        next = word_of(t + 1, byte);
                        byte = mask_byte(t + 2);
                        if constexpr (STAGES == 2) issue(t + 1, (t + 1 - t0) & 1, next);
                    }
                    one(word, STAGES == 2 ? (t - t0) & 1 : 0);
                    word = next;
                    if constexpr (STAGES == 1) {
                        meet();
                        if (t + 1 < t1) issue(t + 1, 0, word);
                    }
                }
            }
        }

        // a lane holds columns d = 16 i + 4 fg .. + 3 of row rr
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            if constexpr (MODE < 2) {
                l[t] += __shfl_xor(l[t], 16);
                l[t] += __shfl_xor(l[t], 32);
            }
            if (!row_in[t]) continue;
            const long long flat = ((long long)b * p.Sq + rs[t]) * p.H + rh[t];
            if constexpr (MODE == 1) {
                const long long at = ((long long)split * p.B * p.Hkv + (long long)b * p.Hkv + hk) * p.R + rr[t];
                if (fg == 0) { p.part_ml[at * 2] = m[t]; p.part_ml[at * 2 + 1] = l[t]; }
#pragma unroll
                for (int d = 0; d < ND; ++d) *(floatx4*)(p.part_o + at * (ND * 16) + d * 16 + fg * 4) = acc[d][t];
            } else {
                float by = p.scale;
                if constexpr (MODE == 0) {
                    by = l[t] > 0.0f ? 1.0f / l[t] : (l[t] == 0.0f ? 0.0f : l[t]);      // a NaN stays one
                    if (p.lse && fg == 0) p.lse[flat] = l[t] == 0.0f || !row_ok[t] ? -INFINITY : (m[t] + __builtin_amdgcn_logf(l[t])) * kLn2;
                } else {
                    if (fg == 0) p.delta[flat] = dlt[t];
                    if (!p.dq.p) continue;
                    if constexpr (kScaled<T>) {
#pragma unroll
                        for (int d = 0; d < ND; ++d) acc[d][t] *= 1.0f / up[t];
                    }
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
__global__ __launch_bounds__(NW * 64, xa_waves(sizeof(T) == 4, KD)) void xa_keys_kernel(XaDev p)
{
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int TB = kTile * KD * 64, STAGE = 2 * TB + 2 * kTile * 4, STAGES = stages_of(KD, 2 * kTile * 4);      // Q and dO tiles, then lse and delta of the rows
    constexpr int KEYS = NW * KTW * 16;
    // fp16 holds probabilities below 2^-14 with fewer bits, and with thousands of keys most are: dv is formed from 2^8 times them (8 less in the exponent's lse)
    constexpr float kUpLog = kScaled<T> ? 8.0f : 0.0f, kDown = kScaled<T> ? 1.0f / 256.0f : 1.0f;
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int fr = lane & 15, fg = lane >> 4;
    int id = p.ragged ? blockIdx.x : xcd_chunk(blockIdx.x, gridDim.x);
    const int split = id % p.splits; id /= p.splits;
    const int kbk = id % p.nkb; id /= p.nkb;
    const int hk = id % p.Hkv, b = id / p.Hkv;
    const int kv_len = p.kv_lens ? min(max(p.kv_lens[b], 0), p.Skv) : p.Skv;
    const int q_len = p.q_lens ? min(max(p.q_lens[b], 0), p.Sq) : p.Sq;
    const int rows = q_len * p.G, ntiles = (rows + kTile - 1) / kTile;
    // a part takes a fixed number of tiles of rows: parts of long and short sequences cost the same, and parts past a sequence's rows are empty (nothing is written, the
    // joining kernel knows)
    const int t0 = split * p.chunk, t1 = min(ntiles, t0 + p.chunk);
    if (p.part_o && (kbk * KEYS >= kv_len || t0 >= t1)) return;

    int key[KTW];
    bool key_ok[KTW];
    Frag<T> kf[KTW][KD], vf[KTW][KD];
    floatx4 ak[ND][KTW], av[ND][KTW];
    float up[KTW];                                // kScaled: ps and ak hold up times their values
#pragma unroll
    for (int j = 0; j < KTW; ++j) {
        up[j] = kUpStart;
        key[j] = kbk * KEYS + (wid * KTW + j) * 16 + fr;
        key_ok[j] = key[j] < kv_len && (!p.mask || p.mask[b * p.mask_b + key[j]]);
        load_rows<T, KD>(kf[j], p.k.p + b * p.k.b + key[j] * p.k.s + hk * p.k.h, key_ok[j], p.D, lane);
        load_rows<T, KD>(vf[j], p.v.p + b * p.v.b + key[j] * p.v.s + hk * p.v.h, key_ok[j], p.D, lane);
#pragma unroll
        for (int d = 0; d < ND; ++d) { ak[d][j] = floatx4{0.f, 0.f, 0.f, 0.f}; av[d][j] = floatx4{0.f, 0.f, 0.f, 0.f}; }
    }

    bool active = false;                          // a wave without a key that counts helps to bring the tiles in and leaves its share of zeros
#pragma unroll
    for (int j = 0; j < KTW; ++j) active = active || __any(key_ok[j]);

    const char* qb = p.q.p + b * p.q.b + (long long)hk * p.G * p.q.h;
    const char* ob = p.dO.p + b * p.dO.b + (long long)hk * p.G * p.dO.h;
    const unsigned lds0 = (unsigned)(unsigned long long)(__attribute__((address_space(3))) char*)smem;
    float row_lse = 0.0f, row_delta = 0.0f;
    Reader<T, KD> rd;
    rd.init(lane);
    Stager<T, KD, NW> sq, so;
    auto offsets = [&](int r0) {                  // of the rows from r0 on, from the first of r0's query
        const int s0 = r0 / p.G;
        auto off = [&](const Strided& x) { return [&](int r) { const int s = (r0 + r) / p.G; return (unsigned)((s - s0) * x.s + (r0 + r - s * p.G) * x.h); }; };
        sq.init(p.D, tid, off(p.q));
        so.init(p.D, tid, off(p.dO));
    };
    const bool fixed = kTile % p.G == 0;          // a tile starts at a query's first head: the same offsets for all tiles
    if (fixed) offsets(0);
    auto issue = [&](int t, int slot) {
        const unsigned lds = lds0 + slot * STAGE;
        const int r0 = t * kTile, s0 = r0 / p.G;
        if (!fixed) offsets(r0);
        const unsigned long long w = low_bits((long long)rows - r0);
        sq.issue(qb + s0 * p.q.s, lds, w, tid, wid);
        so.issue(ob + s0 * p.dO.s, lds + TB, w, tid, wid);
        if (tid < kTile) {
            const int rr = r0 + tid, s = rr / p.G;
            row_lse = INFINITY;
            row_delta = 0.0f;
            if (rr < rows) {
                const long long at = ((long long)b * p.Sq + s) * p.H + hk * p.G + (rr - s * p.G);
                row_lse = p.lse[at] * kLog2e - kUpLog;
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
            const unsigned tq = lds0 + slot * STAGE, to = tq + TB;
            const float* rl = (const float*)(smem + slot * STAGE + 2 * TB);
            if (active) {
            Probs<T> pp[KTW], ps[KTW];
            floatx4 ds[kScaled<T> ? 4 : 1][KTW];
            float top = 0.0f;
#pragma unroll
            for (int rt = 0; rt < 4; ++rt) {
                floatx4 s[KTW], dp[KTW];
#pragma unroll
                for (int j = 0; j < KTW; ++j) { s[j] = floatx4{0.f, 0.f, 0.f, 0.f}; dp[j] = floatx4{0.f, 0.f, 0.f, 0.f}; }
#pragma unroll
                for (int kk = 0; kk < KD; ++kk) {
                    const Frag<T> a = rd.rows(tq, rt, kk), c = rd.rows(to, rt, kk);
#pragma unroll
                    for (int j = 0; j < KTW; ++j) { s[j] = mma(a, kf[j][kk], s[j]); dp[j] = mma(c, vf[j][kk], dp[j]); }
                }
                const floatx4 ls = *(const floatx4*)(rl + rt * 16 + fg * 4), dl = *(const floatx4*)(rl + kTile + rt * 16 + fg * 4);
#pragma unroll
                for (int j = 0; j < KTW; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float e = __builtin_amdgcn_exp2f(fmaf(s[j][r], p.scale2, -ls[r]));
                        pp[j].set(rt, r, e);          // a key that does not count has its own column of the results alone: set to zero at the end
                        if constexpr (kScaled<T>) {
                            ds[rt][j][r] = e * up[j] * (dp[j][r] - dl[r]);
                            top = fmaxf(top, fabsf(ds[rt][j][r]));
                        } else ps[j].set(rt, r, e * (dp[j][r] - dl[r]));
                    }
            }
            if constexpr (kScaled<T>) {
                if (__any(top > kUpLimit)) {
#pragma unroll
                    for (int j = 0; j < KTW; ++j) {
                        float m = 0.0f;
#pragma unroll
                        for (int rt = 0; rt < 4; ++rt)
#pragma unroll
                            for (int r = 0; r < 4; ++r) m = fmaxf(m, fabsf(ds[rt][j][r]));
                        const float by = fit(m);
                        up[j] *= by;
#pragma unroll
                        for (int rt = 0; rt < 4; ++rt) ds[rt][j] *= by;
#pragma unroll
                        for (int d = 0; d < ND; ++d) ak[d][j] *= by;
                    }
                }
#pragma unroll
                for (int j = 0; j < KTW; ++j)
#pragma unroll
                    for (int rt = 0; rt < 4; ++rt)
#pragma unroll
                        for (int r = 0; r < 4; ++r) ps[j].set(rt, r, ds[rt][j][r]);
            }
#pragma unroll
            for (int s2 = 0; s2 < Probs<T>::N; ++s2)
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const Frag<T> oc = rd.cols(to, d, s2), qc = rd.cols(tq, d, s2);
#pragma unroll
                    for (int j = 0; j < KTW; ++j) { av[d][j] = mma(oc, pp[j].f[s2], av[d][j]); ak[d][j] = mma(qc, ps[j].f[s2], ak[d][j]); }
                }
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
            if constexpr (kScaled<T>) ak[d][j] *= kDown / up[j];
            const floatx4 none = {0.f, 0.f, 0.f, 0.f}, gk = key_ok[j] ? ak[d][j] * p.scale : none, gv = key_ok[j] ? av[d][j] * kDown : none;
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

// dk / dv from their parts (those that were written), in the order of the splits; blockIdx.y: dk, dv; keys: those of a workgroup
template <typename T> __global__ __launch_bounds__(256) void xa_keys_join_kernel(XaDev p, int keys)
{
    typedef typename VecOf<T, 4>::type T4;
    const Strided& out = blockIdx.y ? p.dv : p.dk;
    if (!out.p) return;
    const long long n = (long long)p.B * p.Skv * p.Hkv * p.D;
    for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (long long)gridDim.x * 1024) {
        const int d = (int)(i % p.D), hk = (int)(i / p.D % p.Hkv);
        const long long bk = i / p.D / p.Hkv;
        const int b = (int)(bk / p.Skv);
        const int kv_len = p.kv_lens ? min(max(p.kv_lens[b], 0), p.Skv) : p.Skv, q_len = p.q_lens ? min(max(p.q_lens[b], 0), p.Sq) : p.Sq;
        const int parts = bk % p.Skv < (kv_len + keys - 1) / keys * keys ? ((q_len * p.G + kTile - 1) / kTile + p.chunk - 1) / p.chunk : 0;
        floatx4 s = {0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < parts; ++k) s += *(const floatx4*)(p.part_o + ((long long)k * 2 + blockIdx.y) * n + i);
        T4 w;
#pragma unroll
        for (int r = 0; r < 4; ++r) w[r] = (T)s[r];
        *(T4*)((T*)(out.p + bk / p.Skv * out.b + bk % p.Skv * out.s + hk * out.h) + d) = w;
    }
}

template <typename T, int KD, int ND, int NW, int QT, int MODE, bool RES> void xa_rows(const OpCtx& c, const XaDev& d)
{
    constexpr int smem = stages_of(KD, 0) * 2 * kTile * KD * 64;
    auto k = xa_rows_kernel<T, KD, ND, NW, QT, MODE, RES>;
    op_allow_lds((const void*)k, smem);
    const long long groups = RES ? (d.nrb + d.rpg - 1) / d.rpg : d.nrb;
    k<<<(unsigned)((long long)d.B * d.Hkv * groups * d.splits), NW * 64, smem, c.stream>>>(d);
    op_launched("cross attention");
}
template <typename T, int KD, int ND, int MODE> void xa_rows_by(const OpCtx& c, const XaRows& r, XaDev d)
{
    constexpr int QT = xa_qt(KD, MODE == 2);
    d.nrb = r.nrb;
    d.rpg = r.rpg;
    if (r.nw == 1) { xa_rows<T, KD, ND, 1, 1, MODE, false>(c, d); return; }
    if constexpr (MODE != 1 && stages_of(KD, 0) == 2) {              // as xa_plan has it
        if (d.rpg) { xa_rows<T, KD, ND, 4, QT, MODE, true>(c, d); return; }
    }
    if constexpr (QT == 2) {
        if (r.qt == 2) { xa_rows<T, KD, ND, 4, 2, MODE, false>(c, d); return; }
    }
    xa_rows<T, KD, ND, 4, 1, MODE, false>(c, d);
}
template <typename T, typename F> void xa_with_shape(int kd, int nd, F&& f)
{
#define XA_CASE(KD, ND) if (kd == KD && nd == ND) { f(std::integral_constant<int, KD>{}, std::integral_constant<int, ND>{}); return; }
    if constexpr (sizeof(T) == 2) {
        XA_CASE(1, 2) XA_CASE(2, 3) XA_CASE(2, 4) XA_CASE(3, 5) XA_CASE(3, 6) XA_CASE(4, 8) XA_CASE(5, 10) XA_CASE(6, 12) XA_CASE(8, 16)
    } else {
        XA_CASE(2, 2) XA_CASE(4, 4) XA_CASE(5, 5) XA_CASE(8, 8) XA_CASE(10, 10) XA_CASE(16, 16)
    }
#undef XA_CASE
    sde_fail(SDE_ERR_INVALID_ARGUMENT, "cross attention: no kernel for this head size");
}
template <typename T> void xa_forward_type(const OpCtx& c, const XaPlan& p, const XaDev& d)
{
    xa_with_shape<T>(p.kd, p.nd, [&](auto kd, auto nd) {
        constexpr int KD = decltype(kd)::value, ND = decltype(nd)::value;
        if (p.splits == 1) { xa_rows_by<T, KD, ND, 0>(c, p.fwd, d); return; }
        xa_rows_by<T, KD, ND, 1>(c, p.fwd, d);
        xa_join_kernel<T><<<(unsigned)std::min<long long>(cdiv64((long long)d.B * d.Sq * d.H, 4), 8192), 256, 0, c.stream>>>(d, ND * 16);
        op_launched("cross attention join");
    });
}
// d.splits / d.part_o: those of dk / dv
template <typename T> void xa_backward_type(const OpCtx& c, const XaPlan& p, const XaDev& d)
{
    xa_with_shape<T>(p.kd, p.nd, [&](auto kd, auto nd) {
        constexpr int KD = decltype(kd)::value, ND = decltype(nd)::value;
        constexpr int KTW = xa_ktw(sizeof(T) == 4, KD);
        XaDev r = d;
        r.splits = 1;
        xa_rows_by<T, KD, ND, 2>(c, p.dq, r);
        if (!d.dk.p && !d.dv.p) return;
        constexpr int smem = stages_of(KD, 2 * kTile * 4) * (2 * kTile * KD * 64 + 2 * kTile * 4);
        auto k = xa_keys_kernel<T, KD, ND, 4, KTW>;
        op_allow_lds((const void*)k, smem);
        k<<<(unsigned)((long long)d.B * d.Hkv * d.nkb * d.splits), 256, smem, c.stream>>>(d);
        op_launched("cross attention key gradients");
        if (d.part_o) {
            const long long n = (long long)d.B * d.Skv * d.Hkv * d.D;
            xa_keys_join_kernel<T><<<dim3((unsigned)std::min<long long>(cdiv64(n, 1024), 4096), 2), 256, 0, c.stream>>>(d, 4 * KTW * 16);
            op_launched("cross attention key gradients' join");
        }
    });
}

}  // namespace
