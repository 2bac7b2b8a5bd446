"""GPU: ops.gated_ff and its gradient against the formulas in 64 bits.

Bounds, elementwise.  u = half a step of the tensors' type, v = 2^-24.  A product of contraction length n is off by at most (n + 8) v times the
product of magnitudes; the projections' errors go through the activation (slope at most 1.13, curvature at most 1.2 for all three); exp and 1 / x of the
hardware and erf are good to a few v: 16 v (1 + |g|) for the activation, its slope likewise.  The gradients of the projections are rounded to the tensors' type once, as
operands of the next products: u of their magnitude; the bias gradient takes them unrounded."""
import math

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
    assert off.numel() == 0 or off.max().item() <= 0, f"{what}: {off.max().item():.3g} past its bound at {off.argmax().item()}, value {want.flatten()[off.argmax()].item():.3g}"


def activation(g, act):
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if act == "gelu":
        c = torch.special.ndtr(g)
        return g * c, c + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (g + 0.044715 * g ** 3))
    return g * (1 + t) / 2, (1 + t) / 2 + g * (1 - t * t) / 2 * k * (1 + 3 * 0.044715 * g * g)


def check(x, w, b, dh, act):
    xs, ws, bs = (t.detach().requires_grad_() if t is not None else None for t in (x, w, b))
    h = ops.gated_ff(xs, ws, bs, activation=act)
    assert torch.equal(h, ops.gated_ff(x, w, b, activation=act))
    f, k = w.shape[0] // 2, w.shape[1]
    X, W, D = x.double().reshape(-1, k), w.double(), dh.double().reshape(-1, f)
    B = b.double() if b is not None else torch.zeros(2 * f, dtype=torch.float64, device=x.device)
    ag = X @ W.t() + B
    e = (k + 8) * V * (X.abs() @ W.abs().t() + B.abs())
    a, g, ea, eg = ag[:, :f], ag[:, f:], e[:, :f], e[:, f:]
    y, slope = activation(g, act)
    e_act = 1.13 * eg + 16 * V * (1 + g.abs())
    e_slope = 1.2 * eg + 16 * V * (1 + g.abs())
    within(h.reshape(-1, f), a * y, ea * y.abs() + a.abs() * e_act + ea * e_act + 4 * V * (a * y).abs(), "h")
    grads = torch.autograd.grad(h, [t for t in (xs, ws, bs) if t is not None], dh)
    dag = torch.cat([D * y, D * a * slope], 1)
    e_dag = torch.cat([D.abs() * e_act, D.abs() * (ea * slope.abs() + a.abs() * e_slope + ea * e_slope)], 1) + 4 * V * dag.abs()
    u, tiny = U[x.dtype], TINY[x.dtype]
    r = e_dag + u * (dag.abs() + e_dag) + tiny                       # as operands
    m = X.shape[0]
    within(grads[0].reshape(-1, k), dag @ W, r @ W.abs() + (2 * f + 8) * V * (dag.abs() @ W.abs()), "dx")
    within(grads[1], dag.t() @ X, r.t() @ X.abs() + (m + 8) * V * (dag.abs().t() @ X.abs()), "dweight")
    if bs is not None:
        within(grads[2], dag.sum(0), e_dag.sum(0) + (m + 8) * V * dag.abs().sum(0), "dbias")


def make(m, k, f, t, seed=0, bt=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return r(m, k).to(t), (r(2 * f, k) * k ** -0.5).to(t), (r(2 * f) * 0.3).to(bt or t), r(m, f).to(t)


SIZES = [(1, 64, 64), (2, 1280, 640), (7, 8, 8), (16, 72, 136), (33, 320, 1280), (64, 200, 264), (65, 256, 128), (257, 136, 392), (1000, 320, 1280), (300, 2048, 256),
         (2049, 64, 520)]


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("m,k,f", SIZES)
def test_gated_ff(m, k, f, dtype, act):
    check(*make(m, k, f, T[dtype], seed=m + k + f), act)


def test_gated_ff_in_steps_of_four_fp32():
    check(*make(37, 68, 44, torch.float32, seed=1), "gelu")


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_gated_ff_small_gates(dtype, act):
    """A gate of 0 gives exactly 0, and small gates keep their relative precision.  x is 0, so a = 1 and g are the bias, exactly.  act(g) = g c with c
    near 1 / 2: the tail of the erf form is off by 7.5e-8 < 2 v, the other steps by a few v, so 32 v |g| covers each form, beside the one rounding of h."""
    t = T[dtype]
    g = torch.zeros(64, device="cuda", dtype=torch.float64)
    g[2::2] = 2.0 ** -torch.linspace(4, 14, 31, device="cuda", dtype=torch.float64)
    g[3::2] = -g[2::2]
    b = torch.cat([torch.ones_like(g), g]).to(t)
    x = torch.zeros(40, 64, device="cuda", dtype=t)
    h = ops.gated_ff(x, make(40, 64, 64, t, seed=5)[1], b, activation=act)
    g = b[64:].double()
    want = activation(g, act)[0]
    assert (h[:, :2] == 0).all()
    within(h, want.expand(40, 64), (32 * V * g.abs()).expand(40, 64), "h")


def test_gated_ff_large_gates():
    """Gates far out on both sides: the activation is the gate itself or nothing, its slope 1 or 0."""
    for act in ("gelu", "gelu_tanh", "silu"):
        x, w, b, dh = make(40, 64, 64, torch.float32, seed=2)
        check(x, w * 20, b, dh, act)
        b2 = torch.full_like(b, 100.0)
        b2[96:] = -100.0
        check(x, w, b2, dh, act)


def test_gated_ff_bias_forms():
    x, w, b, dh = make(100, 320, 256, torch.bfloat16, seed=3, bt=torch.float32)
    check(x, w, b, dh, "gelu")
    check(x, w, None, dh, "silu")


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_gated_ff_of_views(dtype):
    t = T[dtype]
    x, w, b, dh = make(60, 144, 128, t, seed=4)
    check(x[:, 8:136], w[:, 16:144], b, dh, "gelu")                         # rows apart
    check(x[:, 1:129], w[:, 3:131], b, dh, "gelu")                          # off 16 bytes: copied
    check(x[:1, :128].expand(60, 128), w[:, :128], b, dh[:, :1].expand(60, 128), "silu")
    check(x.view(3, 20, 144), w, b, dh.view(3, 20, 128), "silu")


def test_gated_ff_of_nothing():
    x, w, b, dh = make(0, 64, 64, torch.float16)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    h = ops.gated_ff(*leaves)
    gx, gw, gb = torch.autograd.grad(h, leaves, dh)
    assert h.shape == (0, 64) and gx.shape == (0, 64) and not gw.any() and not gb.any()


def test_gated_ff_wanted_gradients_alone():
    x, w, b, dh = make(300, 64, 64, torch.float32, seed=5)
    full = [t.detach().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(ops.gated_ff(*full), full, dh)
    for i in range(3):
        args = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        got, = torch.autograd.grad(ops.gated_ff(*args), args[i], dh)
        assert torch.equal(got, want[i])


def test_gated_ff_spreads_nan_to_its_row_and_column_alone():
    x, w, b, _ = make(70, 64, 64, torch.float16, seed=6)
    good = ops.gated_ff(x, w, b)
    x[3, 7] = float("nan")
    bad = ops.gated_ff(x, w, b)
    assert bad[3].isnan().all() and torch.equal(bad[:3], good[:3]) and torch.equal(bad[4:], good[4:])
    x[3, 7] = 0
    w[5, 1] = float("inf")
    bad = ops.gated_ff(x, w, b)
    keep = [i for i in range(64) if i != 5]
    assert not torch.isfinite(bad[:, 5]).any() and torch.isfinite(bad[:, keep]).all()


def test_gated_ff_rows_behind_the_last_are_left_as_they_were():
    from diffusers_amd import _lib
    x, w, b, _ = make(70, 64, 96, torch.bfloat16, seed=7)
    h = torch.full((300, 104), 7.0, device="cuda", dtype=torch.bfloat16)
    a = _lib.GatedFfArgs(1, 1, 2, 70, 64, 96, 64, 64, 104, 0, 0, 0, x.data_ptr(), w.data_ptr(), b.data_ptr(), h.data_ptr())
    L = _lib.lib()
    import ctypes as C
    n = C.c_size_t()
    _lib.check(L.sde_gated_ff_workspace(a, 0, n))
    ws = torch.empty(max(1, n.value), dtype=torch.uint8, device="cuda")
    _lib.check(L.sde_gated_ff_forward(a, _lib.OpExec(0, torch.cuda.current_stream().cuda_stream, ws.data_ptr(), ws.numel())))
    assert torch.equal(h[:70, :96], ops.gated_ff(x, w, b, activation="silu")) and (h[70:] == 7).all() and (h[:, 96:] == 7).all()


def test_gated_ff_gradient_against_differences():
    x, w, b, dh = make(5, 32, 16, torch.float32, seed=8)
    for act in ("gelu", "gelu_tanh", "silu"):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        grads = torch.autograd.grad(ops.gated_ff(*leaves, activation=act), leaves, dh)
        g = torch.Generator(device="cuda").manual_seed(9)
        steps = [torch.randn(t.shape, generator=g, device="cuda") * s for t, s in ((x, 1.0), (w, 0.1), (b, 0.3))]
        h = 2.0 ** -7
        up, down = ([t + sign * h * s for t, s in zip((x, w, b), steps)] for sign in (1, -1))
        num = ((ops.gated_ff(*up, activation=act) - ops.gated_ff(*down, activation=act)).double() * dh.double()).sum().item() / (2 * h)
        want = sum((a.double() * s.double()).sum().item() for a, s in zip(grads, steps))
        # h^2 / 6 of the third derivative (80 terms, each of order 20 along this step) and rounding of 80 values of order 4 divided by h
        assert abs(num - want) < h * h / 6 * 80 * 20 + 80 * 4 * 2.0 ** -20 / h


def test_gated_ff_refuses():
    x, w, b, _ = make(4, 64, 32, torch.float16)
    with pytest.raises(ValueError, match="activation"):
        ops.gated_ff(x, w, b, activation="relu")
    with pytest.raises(ValueError):
        ops.gated_ff(x[:, :60], w[:, :60], b)
    with pytest.raises(ValueError):
        ops.gated_ff(x, w[:62], b[:62])
    with pytest.raises(ValueError):
        ops.gated_ff(x, w[:, :32], b)
    with pytest.raises(ValueError, match="shape"):
        ops.gated_ff(x, w, b[:32])
    with pytest.raises(TypeError):
        ops.gated_ff(x, w.float(), b)
    with pytest.raises(ValueError, match="on"):
        ops.gated_ff(x, w, b.cpu())
