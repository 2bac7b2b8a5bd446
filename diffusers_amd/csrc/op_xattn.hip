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
#include "op_xattn.h"
#include "ops_device.h"

#include <algorithm>

namespace {

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

void xa_shape(const sde_cross_attention_args& a, XaPlan& p)
{
    const int step = a.dtype == SDE_F32 ? 16 : 32;
    int kd = cdiv((int)a.D, step), nd = cdiv((int)a.D, 16);
    if (a.dtype == SDE_F32) {
        kd = nd = nd <= 2 ? 2 : nd <= 4 ? 4 : nd <= 5 ? 5 : nd <= 8 ? 8 : nd <= 10 ? 10 : 16;
    } else {
        kd = kd <= 5 ? kd : kd <= 6 ? 6 : 8;
        nd = nd == 3 || nd == 5 ? nd : 2 * kd;
    }
    p.kd = kd;
    p.nd = nd;
}

XaPlan xa_plan(const sde_cross_attention_args& a)
{
    XaPlan p{};
    xa_shape(a, p);
    const int64_t R = a.Sq * (a.H / a.Hkv), heads = a.B * a.Hkv, ktiles = cdiv64(a.Skv, kTile);
    // one wave for single tokens; 16 rows a wave up to 64 rows, more past that
    auto rows = [&](bool dq) {
        const int nw = R <= 16 ? 1 : 4, qt = R <= 64 ? 1 : xa_qt(p.kd, dq);
        return XaRows{nw, qt, (int)cdiv64(R, nw * qt * 16), 0};
    };
    p.fwd = rows(false);
    p.dq = rows(true);
    // the keys are split when the rows leave CUs idle: to about 8 waves for each CU, at least 2 tiles a part
    const int64_t blocks = heads * p.fwd.nrb, want = p.fwd.nw == 1 ? 2048 : 512;
    p.splits = 1;
    if (blocks < 256 || (p.fwd.nw == 1 && blocks < want)) p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({want / blocks, ktiles / 2, 64}));
    // two tiles of keys or fewer stay in LDS, where it has two stages, while a workgroup walks blocks of rows over them: as many as leave 4 workgroups to a CU
    if (R > 64 && ktiles <= 2 && stages_of(p.kd, 0) == 2) {
        auto blocks_of = [&](const XaRows& r) { return (int)std::max<int64_t>(1, std::min<int64_t>(heads * r.nrb / 1024, 16)); };
        p.fwd.rpg = p.splits == 1 ? blocks_of(p.fwd) : 0;
        p.dq.rpg = blocks_of(p.dq);
    }
    // dk / dv: parts of equal numbers of row tiles.  Two workgroups to a CU run at once; four times that many parts where lengths are given, so that a long sequence
    // does not keep a few CUs busy alone.
    const int keys = 4 * 16 * xa_ktw(a.dtype == SDE_F32, p.kd);
    p.nkb = (int)cdiv64(a.Skv, keys);
    const int64_t kblocks = heads * p.nkb, rtiles = cdiv64(R, kTile), parts = a.q_lens || a.kv_lens ? 2048 : 512;
    const int64_t splits = kblocks >= parts ? 1 : std::max<int64_t>(1, std::min<int64_t>({cdiv64(parts, kblocks), rtiles, 64}));
    p.chunk = (int)cdiv64(rtiles, splits);
    p.key_splits = (int)cdiv64(rtiles, p.chunk);
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

}  // namespace

int64_t op_cross_attention_threads(const sde_cross_attention_args& a)
{
    if (!a.B || !a.Sq || !a.Skv) return 0;
    const XaPlan p = xa_plan(a);
    auto rows = [&](const XaRows& r, int64_t splits) { return (r.rpg ? cdiv64(r.nrb, r.rpg) : r.nrb) * splits * r.nw * 64; };
    return a.B * a.Hkv * std::max({rows(p.fwd, p.splits), rows(p.dq, 1), (int64_t)p.nkb * p.key_splits * 256});
}

size_t op_cross_attention_ws_bytes(const sde_cross_attention_args& a, bool backward)
{
    const int64_t rows = a.B * a.Sq * a.H;
    if (!rows || !a.Skv) return 0;
    const XaPlan p = xa_plan(a);
    if (!backward) return p.splits > 1 ? op_align((size_t)p.splits * rows * p.nd * 16 * 4) + op_align((size_t)p.splits * rows * 2 * 4) : 0;
    return op_align((size_t)rows * 4) + (p.key_splits > 1 && (a.dk || a.dv) ? op_align((size_t)p.key_splits * 2 * a.B * a.Skv * a.Hkv * a.D * 4) : 0);
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
    d.splits = p.splits;
    if (p.splits > 1) {
        d.part_o = (float*)c.ws;
        d.part_ml = (float*)(c.ws + op_align((size_t)p.splits * a.B * a.Sq * a.H * p.nd * 16 * 4));
    }
    if (a.dtype == SDE_F16) xa_forward_f16(c, p, d);
    else if (a.dtype == SDE_BF16) xa_forward_bf16(c, p, d);
    else xa_forward_f32(c, p, d);
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
    d.delta = (float*)c.ws;
    d.nkb = p.nkb;
    d.splits = p.key_splits;
    d.chunk = p.chunk;
    if (p.key_splits > 1) d.part_o = (float*)(c.ws + op_align((size_t)a.B * a.Sq * a.H * 4));
    if (a.dtype == SDE_F16) xa_backward_f16(c, p, d);
    else if (a.dtype == SDE_BF16) xa_backward_bf16(c, p, d);
    else xa_backward_f32(c, p, d);
}
