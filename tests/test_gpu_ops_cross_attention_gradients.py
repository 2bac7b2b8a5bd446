"""GPU: the score gradients of ops.cross_attention in fp16 keep their precision whatever the size of the upstream gradient.

A score gradient ds = p (dp - delta) is p ~ 1 / Skv times smaller than the upstream gradient do, and fp16 has few bits below 2^-14 and none below 2^-24.
Bound, in the 2-norm, u = 2^-11 (half a step of fp16, relative): ds is rounded once as an operand and the result once, each at most u and of random sign; o's rounding
inside delta is smaller (with thousands of keys o is a mean).  2 u in all, and half a step of fp16's smallest values, 2^-25, for each element of the result."""
import pytest
import torch

from diffusers_amd import ops

pytestmark = pytest.mark.gpu
U, HALF_STEP = 2.0 ** -11, 2.0 ** -25


def gradients(q, k, v, do, scale):
    """dq, dk, dv in 64 bits; q, do [R, D], k, v [S, D]: one head."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    p = torch.softmax(scale * (q @ k.t()), 1)
    dp = do @ v.t()
    ds = p * (dp - (p * dp).sum(1, keepdim=True))
    return scale * (ds @ k), scale * (ds.t() @ q), p.t() @ do


def run(q, k, v, do, scale):
    leaves = [t[None, :, None].clone().requires_grad_() for t in (q, k, v)]
    return [g[0, :, 0] for g in torch.autograd.grad(ops.cross_attention(*leaves, scale=scale), leaves, do[None, :, None].clone())]


def near(got, want, what):
    assert torch.isfinite(got).all(), what
    off = (got.double() - want).norm().item()
    bar = 2 * U * want.norm().item() + HALF_STEP * want.numel() ** 0.5
    assert off <= bar, f"{what}: {off / want.norm().item():.3g} relative, {bar / want.norm().item():.3g} allowed"


def make(rows, keys, d, by, seed, qk=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda n, s: (torch.randn(n, d, generator=g, device="cuda") * s).half()
    return r(rows, qk), r(keys, qk), r(keys, 1.0), r(rows, by)


@pytest.mark.parametrize("d", [40, 64, 128, 160])
@pytest.mark.parametrize("keys", [100, 1000, 8000])
@pytest.mark.parametrize("by", [1.0, 1e-2, 1e-3, 1e-4])
def test_small_upstream_gradients(by, keys, d):
    # q and k are 2^-4 of their usual size and the scale 2^8 of it: the same scores, and dq and dk 16 times larger, so that their own rounding hides less
    q, k, v, do = make(300, keys, d, by, seed=keys + d, qk=2.0 ** -4)
    scale = 256 * d ** -0.5
    for name, a, b in zip(("dq", "dk", "dv"), run(q, k, v, do, scale), gradients(q, k, v, do, scale)):
        near(a, b, name)


@pytest.mark.parametrize("rows", [1, 16, 300])
@pytest.mark.parametrize("keys", [2, 60, 90])
def test_large_upstream_gradients(rows, keys):
    """Score gradients past fp16's largest value, with results that fp16 holds."""
    q, k, v, do = make(rows, keys, 64, 1.5e4, seed=rows + keys, qk=2.0 ** -5)
    scale = 0.125
    want = gradients(q, k, v, do, scale)
    assert all(w.abs().max() < 60000 for w in want[:2])
    for name, a, b in zip(("dq", "dk"), run(q, k, v, do, scale), want):
        near(a, b, name)


@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("keys", [60, 100, 2000])
@pytest.mark.parametrize("by", [1e-3, 30.0, 1000.0])
def test_small_and_large_values(by, keys, rows):
    q, k, v, do = make(rows, keys, 64, 1e-2, seed=rows + keys, qk=2.0 ** -4)
    v = (v * by).half()
    want = gradients(q, k, v, do, 2.0)
    for name, a, b in zip(("dq", "dk"), run(q, k, v, do, 2.0), want):
        near(a, b, name)


def test_values_that_grow_from_key_to_key():
    """Every tile of keys brings larger score gradients than the one before."""
    q, k, v, do = make(100, 1000, 64, 1e-2, seed=9, qk=2.0 ** -4)
    v = (v * 2.0 ** torch.linspace(-12, 12, 1000, device="cuda")[:, None]).half()
    dq, dk, _ = run(q, k, v, do, 2.0)
    wq, wk, _ = gradients(q, k, v, do, 2.0)
    near(dq, wq, "dq")
    near(dk, wk, "dk")


def test_rows_of_very_different_size():
    """Upstream gradients from 2^-14 to 2^10 in one call, small ones first, large ones first and mixed: dq row by row, dk as a whole."""
    for turn in range(3):
        q, k, v, do = make(256, 2000, 64, 1.0, seed=turn, qk=2.0 ** -4)
        by = 2.0 ** torch.linspace(-14, 10, 256, device="cuda")
        by = (by, by.flip(0), by[torch.randperm(256, generator=torch.Generator().manual_seed(1)).cuda()])[turn]
        do = (do * by[:, None]).half()
        dq, dk, _ = run(q, k, v, do, 32.0)
        wq, wk, _ = gradients(q, k, v, do, 32.0)
        for i in range(256):
            near(dq[i], wq[i], f"dq, row {i}, order {turn}")
        near(dk, wk, f"dk, order {turn}")


def test_a_row_with_infinities_spoils_itself_alone():
    q, k, v, do = make(200, 300, 64, 1e-3, seed=5)
    good = run(q, k, v, do, 0.125)[0]
    do[7, 3] = float("inf")
    do[90, 0] = float("nan")
    bad = run(q, k, v, do, 0.125)[0]
    keep = [i for i in range(200) if i not in (7, 90)]
    assert torch.equal(good[keep], bad[keep]) and not torch.isfinite(bad[[7, 90]]).any()


def test_upstream_gradients_of_zero():
    q, k, v, do = make(70, 200, 64, 1.0, seed=6)
    for g in run(q, k, v, torch.zeros_like(do), 0.125):
        assert not g.any()
    do[10:] = 0
    dq = run(q, k, v, do, 0.125)[0]
    assert dq[:10].any() and not dq[10:].any()


def test_shared_heads_and_lengths():
    """The 2-norm of each sequence, with shared heads, padded queries and keys and a small upstream gradient."""
    g = torch.Generator(device="cuda").manual_seed(8)
    r = lambda *s, by=1.0: (torch.randn(*s, generator=g, device="cuda") * by).half()
    q, k, v, do = r(3, 150, 6, 64, by=2.0 ** -4), r(3, 900, 2, 64, by=2.0 ** -4), r(3, 900, 2, 64), r(3, 150, 6, 64, by=1e-3)
    ql, kl = [150, 33, 100], [900, 500, 64]
    leaves = [t.requires_grad_() for t in (q, k, v)]
    lens = lambda n: torch.tensor(n, dtype=torch.int32, device="cuda")
    dq, dk, _ = torch.autograd.grad(ops.cross_attention(*leaves, q_lens=lens(ql), kv_lens=lens(kl), scale=32.0), leaves, do)
    for b in range(3):
        for h in range(2):
            sum_k = 0
            for i in range(3):
                wq, wk, _ = gradients(q[b, :ql[b], 3 * h + i].detach(), k[b, :kl[b], h].detach(), v[b, :kl[b], h].detach(), do[b, :ql[b], 3 * h + i], 32.0)
                near(dq[b, :ql[b], 3 * h + i], wq, f"dq {b} {h} {i}")
                sum_k = sum_k + wk
            near(dk[b, :kl[b], h], sum_k, f"dk {b} {h}")


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("keys", [2, 100])
def test_the_largest_gradients_that_can_be(keys, d):
    """do and v at fp16's largest values, their signs alike in half of the keys: dp is up to D 65504^2.  The scale brings the results back into range."""
    g = torch.Generator(device="cuda").manual_seed(keys + d)
    q, k = (torch.randn(n, d, generator=g, device="cuda").half() for n in (70, keys))
    sign = torch.where(torch.rand(d, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    v = (65504 * sign * torch.where(torch.arange(keys, device="cuda") % 2 == 0, 1.0, -1.0)[:, None]).half()
    do = (65504 * sign).expand(70, d).half()
    scale = 2.0 ** -28
    want = gradients(q, k, v, do, scale)
    assert all(1 < w.abs().max() < 60000 for w in want[:2])
    for name, a, b in zip(("dq", "dk"), run(q, k, v, do, scale), want):
        near(a, b, name)
