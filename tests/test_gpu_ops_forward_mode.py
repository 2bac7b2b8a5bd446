"""GPU: the operators have no forward-mode derivatives: a tensor that carries a tangent is refused, never taken without it."""
import pytest
import torch
from torch.autograd import forward_ad

from diffusers_amd import ops

pytestmark = pytest.mark.gpu


def r(*s, seed=0, dtype=torch.float16):
    return torch.randn(*s, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def calls():
    """name -> (function of one tensor, that tensor, another one of its shape); strided and ND inputs among them"""
    w, b, wf, bf, k, v = r(64, seed=1), r(64, seed=2), r(96, 64, seed=3), r(96, seed=4), r(2, 9, 2, 64, seed=5), r(2, 9, 2, 64, seed=6)
    lens, mask = torch.tensor([9, 4], dtype=torch.int32, device="cuda"), torch.tensor([[True] * 8 + [False]] * 2, device="cuda")
    return {
        "layer_norm": (lambda x: ops.layer_norm(x, w, b), r(3, 5, 64, seed=7), r(3, 5, 64, seed=8)),
        "layer_norm of a view": (lambda x: ops.layer_norm(x[:, 1:65], None, b), r(6, 70, seed=9), r(6, 70, seed=10)),
        "gated_ff": (lambda x: ops.gated_ff(x, wf, bf, activation="silu"), r(3, 5, 64, seed=11), r(3, 5, 64, seed=12)),
        "gated_ff of a view": (lambda x: ops.gated_ff(x[:, 1:65], wf), r(6, 70, seed=13), r(6, 70, seed=14)),
        "cross_attention": (lambda q: ops.cross_attention(q, k, v, kv_lens=lens, key_mask=mask), r(2, 7, 4, 64, seed=15), r(2, 7, 4, 64, seed=16)),
        "cross_attention, long lengths": (lambda q: ops.cross_attention(q, k, v, q_lens=lens.long(), scale=0.2), r(2, 9, 4, 64, seed=17), r(2, 9, 4, 64, seed=18)),
    }


NAMES = ["layer_norm", "layer_norm of a view", "gated_ff", "gated_ff of a view", "cross_attention", "cross_attention, long lengths"]


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(name, grad):
    f, x, tangent = calls()[name]
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward"):
            f(forward_ad.make_dual(x.requires_grad_(grad), tangent))
    assert torch.isfinite(f(x)).all()


def test_forward_mode_is_refused_for_every_argument():
    x, w, b = r(4, 64), r(64, seed=1), r(64, seed=2)
    wf, bf, q, k = r(96, 64, seed=3), r(96, seed=4), r(1, 4, 2, 64, seed=5), r(1, 6, 2, 64, seed=6)
    with forward_ad.dual_level():
        d = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: ops.layer_norm(x, d(w), b), lambda: ops.layer_norm(x, w, d(b)), lambda: ops.gated_ff(x, d(wf), bf), lambda: ops.gated_ff(x, wf, d(bf)),
                     lambda: ops.cross_attention(q, d(k), k), lambda: ops.cross_attention(q, k, d(k))):
            with pytest.raises(RuntimeError, match="forward"):
                call()


def test_forward_over_reverse_is_refused():
    x, w = r(4, 64).requires_grad_(), r(96, 64, seed=1)
    y = ops.gated_ff(x, w)
    with forward_ad.dual_level():
        dy = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(RuntimeError, match="forward"):
            torch.autograd.grad(y, x, dy)
