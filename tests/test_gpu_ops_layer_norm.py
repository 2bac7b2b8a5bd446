"""GPU: ops.layer_norm and its gradient against the formulas in 64 bits.

Bounds, elementwise.  u = half a step of the result's type; v = 2^-24.  A sum over C values runs in at most n = 90 + C / 256 dependent additions (64
in a lane, then a tree; rows past the register limit: C / 256 in a lane), so its error is at most n v times the sum of magnitudes."""
import pytest
import torch

from diffusers_amd import ops

pytestmark = pytest.mark.gpu
V = 2.0 ** -24
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}
T = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def within(got, want, bound, what):
    u, tiny = U[got.dtype], TINY[got.dtype]
    off = (got.double() - want).abs() - (u * want.abs() + tiny + (1 + u) * bound)
    assert torch.isfinite(got.double()).all(), what
    assert off.max().item() <= 0, f"{what}: {off.max().item():.3g} past its bound at {off.argmax().item()}, value {want.flatten()[off.argmax()].item():.3g}"


def check(x, w, b, dy, eps=1e-5):
    c = x.shape[-1]
    xs, ws, bs = x.detach().requires_grad_(), w.detach().requires_grad_() if w is not None else None, b.detach().requires_grad_() if b is not None else None
    y = ops.layer_norm(xs, ws, bs, eps)
    plain = ops.layer_norm(x.detach(), w, b, eps)
    assert torch.equal(y, plain)                                       # with and without statistics kept: the same bits
    X, D = x.detach().double().reshape(-1, c), dy.double().reshape(-1, c)
    W = w.double() if w is not None else torch.ones(c, dtype=torch.float64, device=x.device)
    B = b.double() if b is not None else torch.zeros(c, dtype=torch.float64, device=x.device)
    n = (90 + c / 256) * V
    mean, var = X.mean(1, keepdim=True), X.var(1, correction=0, keepdim=True)
    rstd = (var + eps) ** -0.5
    xh = (X - mean) * rstd
    e_mean = n * X.abs().mean(1, keepdim=True) + V * mean.abs()
    e_xc = e_mean + V * (X - mean).abs()                                # error of x - mean
    # variance: its own sum, twice the deviation's error in each square (the mean's error enters squared, but count it once)
    e_var = n * var + 2 * (e_xc * (X - mean).abs()).mean(1, keepdim=True)
    e_xh = rstd * e_xc + xh.abs() * (0.5 * e_var * rstd ** 2 + 4 * V)
    within(y.reshape(-1, c), xh * W + B, W.abs() * e_xh + 4 * V * ((xh * W).abs() + B.abs()), "y")
    grads = torch.autograd.grad(y, [t for t in (xs, ws, bs) if t is not None], dy)
    G = D * W
    s1, s2 = G.mean(1, keepdim=True), (G * xh).mean(1, keepdim=True)
    e1 = (n + 2 * V) * G.abs().mean(1, keepdim=True)
    e2 = (n + 2 * V) * (G * xh).abs().mean(1, keepdim=True) + (G.abs() * e_xh).mean(1, keepdim=True)
    want = rstd * (G - s1 - xh * s2)
    inner = G.abs() * 4 * V + e1 + xh.abs() * e2 + s2.abs() * e_xh + 4 * V * (s1.abs() + (xh * s2).abs())
    within(grads[0].reshape(-1, c), want, rstd * inner + want.abs() * (0.5 * e_var * rstd ** 2 + 4 * V), "dx")
    rows = X.shape[0]
    nr = (rows / 64 + 600) * V        # rows of a block in turn, shuffles and waves, then the blocks' sums four ways
    if ws is not None:
        within(grads[1], (D * xh).sum(0), nr * (D * xh).abs().sum(0) + (D.abs() * e_xh).sum(0), "dweight")
    if bs is not None:
        within(grads[-1], D.sum(0), nr * D.abs().sum(0), "dbias")


def make(rows, c, t, pt=None, seed=0, spread=1.5, shift=0.25):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return ((r(rows, c) * spread + shift).to(t), (r(c) * 0.3 + 1).to(pt or t), (r(c) * 0.2).to(pt or t), r(rows, c).to(t))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,c", [(1, 1), (1, 1280), (2, 1280), (3, 7), (5, 47), (700, 320), (1500, 640), (517, 1280), (33, 2560), (9, 4096), (1025, 5120),
                                    (1, 16384), (3, 10007), (2, 20000), (600, 8)])
def test_layer_norm(rows, c, dtype):
    check(*make(rows, c, T[dtype], seed=rows + c))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_layer_norm_with_fp32_parameters(dtype):
    x, w, b, dy = make(129, 320, T[dtype], torch.float32, seed=5)
    check(x, w, b, dy)


def test_layer_norm_without_parameters():
    x, w, b, dy = make(40, 192, torch.float32, seed=6)
    check(x, None, None, dy)
    check(x, w, None, dy)
    check(x, None, b, dy)


def test_layer_norm_of_far_values_and_of_constant_rows():
    x, w, b, dy = make(64, 320, torch.float32, seed=7, spread=0.01, shift=100.0)
    check(x, w, b, dy)
    flat = torch.full((3, 64), 2.0, device="cuda")
    assert torch.equal(ops.layer_norm(flat, None, b[:64].contiguous()), b[:64].expand(3, 64))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_layer_norm_of_views(dtype):
    t = T[dtype]
    x, w, b, dy = make(50, 330, t, seed=8)
    check(x[:, :320], w[:320].contiguous(), b[:320].contiguous(), dy[:, 5:325])          # rows apart, one of them off 16 bytes
    check(x[::2, 1:8], w[1:8].contiguous(), b[1:8].contiguous(), dy[::2, 1:8])
    y = ops.layer_norm(x.t()[:48], None, None)                                             # transposed: copied first
    assert torch.equal(y, ops.layer_norm(x.t()[:48].contiguous(), None, None))
    x3 = x[:48].view(2, 24, 330)
    assert torch.equal(ops.layer_norm(x3, w, b), ops.layer_norm(x[:48], w, b).view(2, 24, 330))
    one = x[:1].expand(5, 330)                                                             # rows that share memory
    assert torch.equal(ops.layer_norm(one, w, b), ops.layer_norm(one.contiguous(), w, b))


def test_layer_norm_of_nothing_and_of_rows_with_nan():
    x = torch.empty(0, 320, device="cuda", requires_grad=True)
    w = torch.ones(320, device="cuda", requires_grad=True)
    y = ops.layer_norm(x, w)
    gx, gw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == gx.shape == (0, 320) and torch.equal(gw, torch.zeros_like(gw))
    z, w2, b2, _ = make(6, 320, torch.float16, seed=9)
    good = ops.layer_norm(z, w2, b2)
    z[2, 5] = float("nan")
    z[4, 0] = float("inf")
    y = ops.layer_norm(z, w2, b2)
    assert y[2].isnan().all() and y[4].isnan().all() and torch.equal(y[[0, 1, 3, 5]], good[[0, 1, 3, 5]])


def test_layer_norm_rows_behind_the_last_are_left_as_they_were():
    from diffusers_amd import _lib
    x, w, b, _ = make(8, 64, torch.float32, seed=10)
    y = torch.full((12, 70), 7.0, device="cuda")
    a = _lib.LayerNormArgs(2, 2, 8, 64, 64, 70, 0, 0, 1e-5, x.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr())
    _lib.check(_lib.lib().sde_layer_norm_forward(a, _lib.OpExec(0, torch.cuda.current_stream().cuda_stream, None, 0)))
    # rows 70 apart are not on 16 bytes: the sums run in another order than those of rows 64 apart, so the same bound holds and not the same bits
    X, W = x.double(), w.double()
    mean, var = X.mean(1, keepdim=True), X.var(1, correction=0, keepdim=True)
    xh = (X - mean) * (var + 1e-5) ** -0.5
    e_xh = (var + 1e-5) ** -0.5 * 91 * V * X.abs().mean(1, keepdim=True) + 190 * V * xh.abs() + 2 * V * xh.abs()
    within(y[:8, :64], xh * W + b.double(), W.abs() * e_xh + 4 * V * ((xh * W).abs() + b.double().abs()), "y")
    assert (y[8:] == 7).all() and (y[:, 64:] == 7).all()
    good = ops.layer_norm(x, w, b)
    _lib.check(_lib.lib().sde_layer_norm_forward(_lib.LayerNormArgs(2, 2, 8, 64, 64, 64, 0, 0, 1e-5, x.data_ptr(), w.data_ptr(), b.data_ptr(), x.data_ptr()),
                                                 _lib.OpExec(0, torch.cuda.current_stream().cuda_stream, None, 0)))
    assert torch.equal(x, good)                                                              # in place


def test_layer_norm_gradient_against_differences():
    g = torch.Generator(device="cuda").manual_seed(11)
    x = torch.randn(3, 24, generator=g, device="cuda", requires_grad=True)
    dy = torch.randn(3, 24, generator=g, device="cuda")
    step = torch.randn(3, 24, generator=g, device="cuda")
    gx, = torch.autograd.grad(ops.layer_norm(x), x, dy)
    h = 2.0 ** -6
    with torch.no_grad():
        num = ((ops.layer_norm(x + h * step) - ops.layer_norm(x - h * step)).double() * dy.double()).sum() / (2 * h)
    # a central difference is off by h^2 / 6 times the third derivative along the step (of order |step|^3 / sigma^3 ~ 1e2) and by rounding: 24 x 3 x 2^-22 / h
    assert abs(num - (gx.double() * step.double()).sum()).item() < h * h / 6 * 400 + 72 * 2.0 ** -22 / h


def test_layer_norm_refuses():
    x, w, b, _ = make(4, 64, torch.float16)
    with pytest.raises(ValueError, match="shape"):
        ops.layer_norm(x, w[:32])
    with pytest.raises(TypeError):
        ops.layer_norm(x, w.bfloat16())
    with pytest.raises(TypeError):
        ops.layer_norm(x, w, b.float())
    with pytest.raises(TypeError):
        ops.layer_norm(x.double())
    with pytest.raises(ValueError, match="on"):
        ops.layer_norm(x, w.cpu())
