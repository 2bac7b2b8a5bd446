"""GPU: the erf gate of ops.gated_ff far out on the negative side, where the activation is g w(g) with w = Phi(g) and nothing is subtracted.

v = 2^-24.  fp32: w = E(|g|) exp(-g^2 / 2).  E is good to a few v (a fit off by 1e-8, nine terms, one reciprocal); the exponential's argument is rounded twice, 2 v g^2 / 2 of the
value; the product with the value, its bias and the rounding of h add a few: (g^2 + 32) v, relative.  16-bit types: w is good to 7.5e-8, absolutely."""
import pytest
import torch

from diffusers_amd import ops

pytestmark = pytest.mark.gpu
V = 2.0 ** -24


def gate(g):
    """g Phi(g) in 64 bits, for g < 0 too without a difference."""
    w = torch.special.erfcx(g.abs() / 2 ** 0.5) / 2 * torch.exp(-g * g / 2)
    return torch.where(g < 0, g * w, g - g * w)


def h_of(g, t):
    n = g.numel()
    b = torch.cat([torch.ones_like(g), g]).to(t)
    x, w = torch.zeros(3, 64, device="cuda", dtype=t), torch.zeros(2 * n, 64, device="cuda", dtype=t)
    return ops.gated_ff(x, w, b, activation="gelu"), b[n:].double()


def test_fp32_keeps_its_relative_precision():
    h, g = h_of(-torch.linspace(0.01, 12.5, 2048, device="cuda"), torch.float32)
    want = gate(g)
    off = ((h.double() - want) / want).abs() / ((g * g + 32) * V)
    assert off.max().item() <= 1, (off.max().item(), g[off.max(0).values.argmax()].item())


def test_fp32_positive_side_and_slope():
    """g > 0: g - g w.  The slope, Phi + g phi, absolutely: terms of order 1."""
    g0 = torch.linspace(-9, 9, 2048, device="cuda")
    h, g = h_of(g0.abs() + 1e-3, torch.float32)
    want = gate(g)
    assert (((h.double() - want) / want).abs() <= 32 * V).all()
    b = torch.cat([torch.ones_like(g0), g0]).requires_grad_()
    x, w = torch.zeros(1, 64, device="cuda"), torch.zeros(4096, 64, device="cuda")
    db, = torch.autograd.grad(ops.gated_ff(x, w, b).sum(), b)
    g = g0.double()
    slope = torch.special.ndtr(g) + g * torch.exp(-g * g / 2) * 0.3989422804014327
    assert ((db[2048:].double() - slope).abs() <= 32 * V).all()
    assert ((db[:2048].double() - gate(g)).abs() <= (32 * V * g.abs()).clamp_min(V)).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_16_bit_types_are_good_to_the_stated_bound(dtype):
    h, g = h_of(-torch.linspace(0.01, 12.5, 2048, device="cuda"), dtype)
    want = gate(g)
    bound = 7.5e-8 * g.abs() + 32 * V * want.abs()
    u, tiny = {torch.float16: (2.0 ** -11, 2.0 ** -25), torch.bfloat16: (2.0 ** -8, 0.0)}[dtype]
    off = (h.double() - want).abs() - (u * want.abs() + tiny + (1 + u) * bound)
    assert off.max().item() <= 0
