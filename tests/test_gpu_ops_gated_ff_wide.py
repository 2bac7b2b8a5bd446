"""GPU: ops.gated_ff with rows of [da dg] so long that 256 of them span more than 2 GB."""
import pytest
import torch

from diffusers_amd import ops

pytestmark = pytest.mark.gpu
V = 2.0 ** -24


def test_dx_of_fp32_rows_of_8_megabytes():
    """F = 1.1 million.  All but 512 columns of dh are zero, from both ends of F, so that the contraction has 1024 terms that are not zero and its bound, (1024 + 8) v of the
    magnitudes, is sharp; the pre-activations are x times those 512 rows of the weight, 512 long."""
    m, k, f = 1024, 512, 1_100_000
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    at = torch.cat([torch.arange(256), torch.arange(f - 256, f)]).cuda()
    x, wv, wg, d = r(m, k), r(512, k) * k ** -0.5, r(512, k) * k ** -0.5, r(m, 512)
    w = torch.zeros(2 * f, k, device="cuda")
    w[at], w[f + at] = wv, wg
    dh = torch.zeros(m, f, device="cuda")
    dh[:, at] = d
    x.requires_grad_()
    h = ops.gated_ff(x, w, activation="silu")
    dx, = torch.autograd.grad(h, x, dh)
    X, WV, WG, D = x.detach().double(), wv.double(), wg.double(), d.double()
    a, gate = X @ WV.t(), X @ WG.t()
    s = torch.sigmoid(gate)
    act, slope = gate * s, s * (1 + gate * (1 - s))
    e = (k + 8) * V * (X.abs() @ WV.abs().t()).maximum(X.abs() @ WG.abs().t())      # of both pre-activations
    e_act = 1.13 * e + 16 * V * (1 + gate.abs())
    assert ((h.detach()[:, at].double() - a * act).abs() <= e * act.abs() + (a.abs() + e) * e_act + 5 * V * (a * act).abs()).all()
    da, dg = D * act, D * a * slope
    e_da = D.abs() * e_act + 5 * V * da.abs()
    e_dg = D.abs() * (e * slope.abs() + (a.abs() + e) * (1.2 * e + 16 * V * (1 + gate.abs()))) + 5 * V * dg.abs()
    want = da @ WV + dg @ WG
    bound = e_da @ WV.abs() + e_dg @ WG.abs() + 1032 * V * (da.abs() @ WV.abs() + dg.abs() @ WG.abs()) + V * want.abs()
    off = (dx.double() - want).abs() - bound
    assert off.max().item() <= 0, (off.max().item(), divmod(off.argmax().item(), k))
