"""GPU: ops.cross_attention and its gradient against the formulas in 64 bits.

Bounds, elementwise.  u = half a step of the tensors' type, v = 2^-24.  A score is off by (D + 8) v scale |q| |k| and by its exponent's rounding, 4 v (|s| + |max|); a
probability by twice the row's worst score error, relative, and by the sum's (Skv + 8) v.  Probabilities and score gradients are rounded to the tensors' type once, as
operands of the next product (u of their magnitude); delta = rowsum(do o) takes the rounded result o (u |do| |o|).  A product of contraction length n adds (n + 8) v of the product
of magnitudes."""
import pytest
import torch

from diffusers_amd import ops

pytestmark = pytest.mark.gpu
V = 2.0 ** -24
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
# half a step of fp16's smallest values; a probability below fp32's smallest normal value, 2^-126, comes out of the exponential as 0
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -126}
T = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def within(got, want, bound, what):
    u, tiny = U[got.dtype], TINY[got.dtype]
    off = (got.double() - want).abs() - (u * want.abs() + tiny + (1 + u) * bound)
    assert torch.isfinite(got.double()).all(), what
    assert off.max().item() <= 0, f"{what}: {off.max().item():.3g} past its bound at {off.argmax().item()}, value {want.flatten()[off.argmax()].item():.3g}"


def make(b, sq, skv, h, hkv, d, t, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(t)
    return r(b, sq, h, d), r(b, skv, hkv, d), r(b, skv, hkv, d), r(b, sq, h, d)


def check(q, k, v, do, q_lens=None, kv_lens=None, key_mask=None, scale=None, grad=True):
    leaves = [t.detach().requires_grad_(grad) for t in (q, k, v)]
    o = ops.cross_attention(*leaves, q_lens=q_lens, kv_lens=kv_lens, key_mask=key_mask, scale=scale)
    (b, sq, h, d), (skv, hkv) = q.shape, k.shape[1:3]
    G, u, tiny = h // hkv, U[q.dtype], TINY[q.dtype]
    scale = d ** -0.5 if scale is None else scale
    dev = q.device
    keys, rows = torch.ones(b, skv, dtype=torch.bool, device=dev), torch.ones(b, sq, dtype=torch.bool, device=dev)
    if kv_lens is not None:
        keys &= torch.arange(skv, device=dev) < kv_lens[:, None]
    if key_mask is not None:
        keys &= key_mask.bool()
    if q_lens is not None:
        rows &= torch.arange(sq, device=dev) < q_lens[:, None]
    by_row = lambda x: torch.where(rows[:, :, None, None], x.double(), 0.0).view(b, sq, hkv, G, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, sq * G, d)
    back = lambda x: x.view(b, hkv, sq, G, d).permute(0, 2, 1, 3, 4).reshape(b, sq, h, d)
    Q, D = by_row(q), by_row(do)
    K, W = (torch.where(keys[:, :, None, None], x.double(), 0.0).permute(0, 2, 1, 3).contiguous() for x in (k, v))
    Kt, Wt = K.transpose(2, 3).contiguous(), W.transpose(2, 3).contiguous()
    on = keys[:, None, None, :] & rows.repeat_interleave(G, 1)[:, None, :, None]
    s = torch.where(on, scale * (Q @ Kt), float("-inf"))
    top = s.amax(3, keepdim=True)
    top = torch.where(top.isinf(), 0.0, top)
    p = torch.exp(s - top)
    total = p.sum(3, keepdim=True)
    p = torch.where(total > 0, p / total.clamp_min(1e-300), 0.0)
    e_s = (d + 8) * V * scale * (Q.abs() @ Kt.abs()) + 4 * V * (torch.where(on, s.abs(), 0.0) + top.abs())
    r = 2 * torch.where(on, e_s, 0.0).amax(3, keepdim=True) + (skv + 8) * V          # relative, of a probability
    O = p @ W
    pv = p @ W.abs()
    e_o = (u + r + (skv + 8) * V) * pv + tiny * W.abs().sum(2, keepdim=True)          # the unnormalised probabilities are at most 1: tiny of them is tiny of p times the sum, at least 1
    within(o, back(O), back(e_o), "o")
    if not grad:
        return o
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    Dt, Pt = D.transpose(2, 3).contiguous(), p.transpose(2, 3).contiguous()
    n = sq * G
    e_p = (u + r) * p + tiny
    within(dv, (Pt @ D).permute(0, 2, 1, 3), (e_p.transpose(2, 3).contiguous() @ D.abs() + (n + 8) * V * (Pt @ D.abs())).permute(0, 2, 1, 3), "dv")
    dp = D @ Wt
    delta = (D * O).sum(3, keepdim=True)
    e_dp = (d + 8) * V * (D.abs() @ Wt.abs())
    e_delta = (D.abs() * (u * O.abs() + e_o + tiny)).sum(3, keepdim=True) + (d + 8) * V * (D * O).abs().sum(3, keepdim=True)
    ds = p * (dp - delta)
    e_ds = p * (r * (dp - delta).abs() + e_dp + e_delta + 2 * V * (dp.abs() + delta.abs()))
    e_ds = e_ds + u * (ds.abs() + e_ds) + torch.where(on, tiny, 0.0)
    within(dq, back(scale * (ds @ K)), back(scale * (e_ds @ K.abs() + (skv + 8) * V * (ds.abs() @ K.abs()))), "dq")
    dst, edt = ds.transpose(2, 3).contiguous(), e_ds.transpose(2, 3).contiguous()
    within(dk, (scale * (dst @ Q)).permute(0, 2, 1, 3), (scale * (edt @ Q.abs() + (n + 8) * V * (dst.abs() @ Q.abs()))).permute(0, 2, 1, 3), "dk")
    return o, dq, dk, dv


def lens(*n):
    return torch.tensor(n, dtype=torch.int32, device="cuda")


SIZES = [  # B, Sq, Skv, H, Hkv, D
    (1, 1, 1, 1, 1, 8), (2, 1, 5, 4, 2, 64), (2, 77, 77, 3, 3, 40), (1, 130, 64, 2, 1, 80), (1, 64, 65, 2, 2, 96), (3, 5, 200, 8, 2, 128), (1, 33, 700, 4, 4, 160),
    (1, 17, 129, 2, 1, 256), (2, 300, 33, 5, 5, 32), (1, 9, 1000, 12, 1, 192), (1, 16, 63, 1, 1, 24), (1, 257, 128, 2, 2, 48), (1, 2, 3000, 1, 1, 72)]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("size", SIZES)
def test_cross_attention(size, dtype):
    check(*make(*size, T[dtype], seed=sum(size)))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("d", [40, 128])
def test_cross_attention_of_ragged_sequences(d, dtype):
    q, k, v, do = make(6, 70, 150, 4, 2, d, T[dtype], seed=d)
    q_lens, kv_lens = lens(70, 0, 1, 64, 33, 70), lens(150, 150, 0, 64, 1, 65)
    mask = torch.rand(6, 150, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") < 0.7
    mask[5] = False                                     # a sequence without a key, one with its last keys alone
    mask[3, :60] = False
    for kw in ({"q_lens": q_lens, "kv_lens": kv_lens}, {"key_mask": mask}, {"q_lens": q_lens, "kv_lens": kv_lens, "key_mask": mask}):
        check(q, k, v, do, **kw)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("sq", [1, 40, 300])
def test_what_does_not_count_is_not_read(sq, dtype):
    """Infinities and NaN behind the lengths and under the mask change nothing: not the result, not the gradients."""
    q, k, v, do = make(3, sq, 200, 4, 2, 64, T[dtype], seed=3)
    q_lens, kv_lens = lens(sq, (sq + 1) // 2, 0), lens(200, 77, 100)
    mask = torch.rand(3, 200, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda") < 0.8
    want = check(q, k, v, do, q_lens, kv_lens, mask)
    keys = mask & (torch.arange(200, device="cuda") < kv_lens[:, None])
    rows = torch.arange(sq, device="cuda") < q_lens[:, None]
    bad = [torch.where(on[:, :, None, None], t, torch.full_like(t, f)) for t, on, f in
           ((q, rows, float("nan")), (k, keys, float("inf")), (v, keys, float("nan")), (do, rows, float("-inf")))]
    leaves = [t.requires_grad_() for t in bad[:3]]
    o = ops.cross_attention(*leaves, q_lens=q_lens, kv_lens=kv_lens, key_mask=mask)
    got = (o, *torch.autograd.grad(o, leaves, bad[3]))
    for name, a, w in zip(("o", "dq", "dk", "dv"), got, want):
        assert torch.equal(a, w), name
    assert not o[~rows].any() and not got[1][~rows].any() and not got[2][~keys].any() and not got[3][~keys].any()


def test_lengths_past_the_sequence_are_taken_at_its_end():
    q, k, v, _ = make(2, 20, 30, 2, 2, 64, torch.float16)
    assert torch.equal(ops.cross_attention(q, k, v, q_lens=lens(99, 20), kv_lens=lens(30, 1 << 30)), ops.cross_attention(q, k, v))
    assert not ops.cross_attention(q, k, v, kv_lens=lens(-5, 0)).any()
    assert torch.equal(ops.cross_attention(q, k, v, kv_lens=lens(7, 30).long()), ops.cross_attention(q, k, v, kv_lens=lens(7, 30)))


@pytest.mark.parametrize("sq,h,hkv,skv", [(1, 32, 8, 4100), (1, 8, 8, 2500), (3, 16, 2, 1300), (16, 2, 2, 5000)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_cross_attention_of_few_queries_on_many_keys(sq, h, hkv, skv, dtype):
    q, k, v, do = make(3, sq, skv, h, hkv, 128, T[dtype], seed=sq)
    mask = torch.rand(3, skv, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda") < 0.9
    check(q, k, v, do, kv_lens=lens(skv, skv // 3, 1), key_mask=mask)


def test_cross_attention_of_large_scores():
    """Scores of some hundreds: one key takes nearly all; and a scale of its own."""
    q, k, v, do = make(1, 50, 90, 2, 2, 64, torch.float32, seed=5)
    check(q * 10, k * 10, v, do)
    check(q, k, v, do, scale=0.01)
    q, k, v, do = make(1, 50, 90, 2, 2, 64, torch.bfloat16, seed=6)
    check(q * 8, k * 4, v, do, grad=False)


@pytest.mark.parametrize("d", [4, 12, 20, 100])
def test_cross_attention_fp32_in_steps_of_four(d):
    check(*make(2, 70, 81, 2, 2, d, torch.float32, seed=d))


def test_more_sequences_than_lanes():
    g = torch.Generator(device="cuda").manual_seed(13)
    q, k, v, do = make(70, 9, 40, 2, 1, 64, torch.bfloat16, seed=13)
    n = lambda top: torch.randint(0, top + 1, (70,), generator=g, device="cuda", dtype=torch.int32)
    check(q, k, v, do, n(9), n(40))


def test_many_keys_in_fp16():
    """Probabilities of 2^-13 and far less: below 2^-14 fp16 has fewer bits for them, dv does not suffer from it."""
    q, k, v, do = make(1, 300, 8000, 1, 1, 64, torch.float16, seed=14)
    _, _, _, dv = check(q, k, v, do)
    p = torch.softmax(q[0, :, 0].double() @ k[0, :, 0].double().t() / 8, 1)
    want = p.t() @ do[0, :, 0].double()
    # one rounding of the probabilities and one of the result, each at most u = 2^-11, in the 2-norm: sums of 300 roundings of random sign
    assert ((dv[0, :, 0].double() - want).norm() / want.norm()).item() < 2 * 2.0 ** -11


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_cross_attention_of_views(dtype):
    t = T[dtype]
    g = torch.Generator(device="cuda").manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(t)
    kv = r(2, 50, 2, 3, 64)                                     # keys and values packed
    q = r(2, 3, 70, 64).transpose(1, 2)                         # heads outside
    do = r(2, 70, 3, 64)
    check(q, kv[:, :, 0], kv[:, :, 1], do)
    check(r(2, 70, 3, 72)[..., 8:72], kv[:, :, 0], kv[:, :, 1], do.transpose(1, 2).contiguous().transpose(1, 2))
    check(r(2, 70, 3, 67)[..., 1:65], r(2, 50, 3, 66)[..., :64], kv[:, :, 1], do)          # off 16 bytes: copied
    one = r(1, 50, 3, 64)
    k = one.expand(2, 50, 3, 64)                                # one prompt for the whole batch
    check(q, k, kv[:, :, 1], do)
    leaf = one.requires_grad_()
    o = ops.cross_attention(q, leaf.expand(2, 50, 3, 64), kv[:, :, 1])
    gk, = torch.autograd.grad(o, leaf, do)
    full = one.detach().expand(2, 50, 3, 64).contiguous().requires_grad_()
    gf, = torch.autograd.grad(ops.cross_attention(q, full, kv[:, :, 1]), full, do)
    assert torch.equal(gk, gf.sum(0, keepdim=True))
    mask = torch.rand(50, device="cuda") < 0.5
    assert torch.equal(ops.cross_attention(q, k, k, key_mask=mask.expand(2, 50)), ops.cross_attention(q, k, k, key_mask=mask.repeat(2, 1)))


@pytest.mark.parametrize("b,sq,skv", [(0, 3, 4), (2, 0, 4), (2, 3, 0)])
def test_cross_attention_of_nothing(b, sq, skv):
    leaves = [t.requires_grad_() for t in make(b, sq, skv, 4, 2, 64, torch.float16)[:3]]
    o = ops.cross_attention(*leaves)
    assert o.shape == (b, sq, 4, 64) and not o.any()
    for gr, x in zip(torch.autograd.grad(o, leaves, torch.ones_like(o)), leaves):
        assert gr.shape == x.shape and not gr.any()


def test_wanted_gradients_alone():
    q, k, v, do = make(2, 70, 90, 4, 2, 64, torch.bfloat16, seed=8)
    full = [t.detach().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(ops.cross_attention(*full), full, do)
    for i in range(3):
        args = [t.detach().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        got, = torch.autograd.grad(ops.cross_attention(*args), args[i], do)
        assert torch.equal(got, want[i])


def test_offsets_past_32_bits():
    """Keys of a cache whose sequences lie 3 GB apart, and heads outside of 1.2 GB of positions each."""
    n = 3 << 29
    cache = torch.empty(2 * n, dtype=torch.float16, device="cuda")
    k = cache.as_strided((2, 100, 2, 64), (n, 128, 64, 1))
    q, kk, v, _ = make(2, 9, 100, 4, 2, 64, torch.float16, seed=9)
    k.copy_(kk)
    assert torch.equal(ops.cross_attention(q, k, v), ops.cross_attention(q, kk, v))
    far = cache.as_strided((1, 700, 1, 64), (0, 1 << 21, 64, 1))          # 4 MB from key to key: the last is 2.8 GB away
    q, kk, v, _ = make(1, 40, 700, 1, 1, 64, torch.float16, seed=10)
    far.copy_(kk)
    assert torch.equal(ops.cross_attention(q, far, v), ops.cross_attention(q, kk, v))


def test_cross_attention_gradient_against_differences():
    q, k, v, do = make(1, 6, 9, 2, 1, 16, torch.float32, seed=11)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.cross_attention(*leaves), leaves, do)
    g = torch.Generator(device="cuda").manual_seed(12)
    steps = [torch.randn(t.shape, generator=g, device="cuda") for t in (q, k, v)]
    h = 2.0 ** -7
    up, down = ([t + sign * h * s for t, s in zip((q, k, v), steps)] for sign in (1, -1))
    num = ((ops.cross_attention(*up) - ops.cross_attention(*down)).double() * do.double()).sum().item() / (2 * h)
    want = sum((a.double() * s.double()).sum().item() for a, s in zip(grads, steps))
    # h^2 / 6 of the third derivative (192 values, each of order 50 along this step) and rounding of 192 values of order 1, divided by h
    assert abs(num - want) < h * h / 6 * 192 * 50 + 192 * 2.0 ** -20 / h


def test_cross_attention_refuses():
    q, k, v, _ = make(2, 4, 6, 4, 2, 64, torch.float16)
    for bad in ((q[0], k, v), (q, k[:1], v[:1]), (q, k, v[:, :5]), (q[..., :32], k, v), (q[:, :, :3], k, v), (q[..., :60], k[..., :60], v[..., :60])):
        with pytest.raises(ValueError):
            ops.cross_attention(*bad)
    for kw in ({"kv_lens": lens(1)}, {"kv_lens": lens(1, 2).float()}, {"q_lens": lens(1, 2).cpu()}, {"key_mask": torch.ones(2, 5, dtype=torch.bool, device="cuda")},
               {"key_mask": torch.zeros(2, 6, device="cuda")}, {"scale": 0.0}, {"scale": -1.0}, {"scale": float("nan")}):
        with pytest.raises(ValueError):
            ops.cross_attention(q, k, v, **kw)
    with pytest.raises(TypeError):
        ops.cross_attention(q, k.float(), v)
