"""CPU: the operators are nodes of their own to torch's tracers; shapes, types and refusals come from their Meta entries, without a device."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from diffusers_amd import ops


def fake(*shape, dtype=torch.float16):
    return torch.empty(*shape, dtype=dtype, device="cuda")


@pytest.fixture(autouse=True)
def mode():
    with FakeTensorMode():
        yield


def targets(g):
    return [str(n.target) for n in g.graph.nodes if n.op == "call_function" and "diffusers_amd" in str(n.target)]


def test_shapes_and_types():
    y = ops.layer_norm(fake(3, 5, 64, dtype=torch.bfloat16), fake(64, dtype=torch.float32))
    assert y.shape == (3, 5, 64) and y.dtype == torch.bfloat16 and y.device.type == "cuda" and y.is_contiguous()
    assert ops.gated_ff(fake(3, 5, 64), fake(96, 64), fake(96)).shape == (3, 5, 48)
    assert ops.cross_attention(fake(2, 7, 4, 64), fake(2, 9, 2, 64), fake(2, 9, 2, 64), kv_lens=fake(2, dtype=torch.int64)).shape == (2, 7, 4, 64)
    x = fake(6, 70)[:, 1:65]
    assert ops.layer_norm(x).shape == (6, 64) and ops.gated_ff(x, fake(96, 64)).shape == (6, 48)
    assert ops.layer_norm(fake(0, 64)).shape == (0, 64)


CALLS = [(lambda x, w, b: ops.layer_norm(x, w, b), [(4, 64), (64,), (64,)], "layer_norm"),
         (lambda x, w, b: ops.gated_ff(x, w, b, activation="silu"), [(2, 4, 64), (96, 64), (96,)], "gated_ff"),
         (lambda q, k, v: ops.cross_attention(q, k, v), [(2, 7, 4, 64), (2, 9, 2, 64), (2, 9, 2, 64)], "cross_attention")]


@pytest.mark.parametrize("f,shapes,name", CALLS)
def test_a_call_is_recorded_as_one_node(f, shapes, name):
    assert targets(make_fx(f)(*[fake(*s) for s in shapes])) == [f"diffusers_amd.{name}.default"]


# autograd of "cuda" tensors asks for a device, that of meta tensors does not: they go to the registered operators themselves
META = [(lambda x, w, b: torch.ops.diffusers_amd.layer_norm(x, w, b), [(4, 64), (64,), (64,)], "layer_norm"),
        (lambda x, w, b: torch.ops.diffusers_amd.gated_ff(x, w, b, 2), [(2, 4, 64), (96, 64), (96,)], "gated_ff"),
        (lambda q, k, v: torch.ops.diffusers_amd.cross_attention(q, k, v), [(2, 7, 4, 64), (2, 9, 2, 64), (2, 9, 2, 64)], "cross_attention")]


@pytest.mark.parametrize("f,shapes,name", META)
@pytest.mark.parametrize("alone", [None, 0, 1, 2])
def test_a_backward_pass_is_recorded(f, shapes, name, alone):
    ops._native()
    leaves = [torch.empty(s, dtype=torch.float16, device="meta", requires_grad=alone in (None, i)) for i, s in enumerate(shapes)]
    dy = torch.empty_like(f(*leaves)).detach()

    def step(dy, *leaves):
        y = f(*leaves)
        return y.detach(), *torch.autograd.grad(y, [t for t in leaves if t.requires_grad], dy)

    out = step(dy, *leaves)
    assert [g.shape for g in out[1:]] == [t.shape for t in leaves if t.requires_grad]
    kept = "gated_ff" if name == "gated_ff" else f"_{name}_kept"
    assert targets(make_fx(step)(dy, *leaves)) == [f"diffusers_amd.{kept}.default", f"diffusers_amd._{name}_backward.default"]


def test_refusals_without_a_device():
    for bad, error in ((lambda: ops.layer_norm(fake(4, 64), fake(32)), ValueError), (lambda: ops.layer_norm(fake(4, 64, dtype=torch.float64)), TypeError),
                       (lambda: ops.gated_ff(fake(4, 60), fake(96, 60)), ValueError), (lambda: ops.gated_ff(fake(4, 64), fake(96, 64, dtype=torch.float32)), TypeError),
                       (lambda: ops.cross_attention(fake(2, 7, 3, 64), fake(2, 9, 2, 64), fake(2, 9, 2, 64)), ValueError),
                       (lambda: ops.layer_norm(torch.empty(4, 64)), ValueError)):
        with pytest.raises(error):
            bad()


def test_second_derivatives_and_tangents_are_refused_without_a_device():
    ops._native()
    x = torch.empty(4, 64, device="meta", requires_grad=True)
    with pytest.raises(RuntimeError, match="first derivatives"):
        torch.autograd.grad(torch.ops.diffusers_amd.layer_norm(x).sum(), x, create_graph=True)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x.detach(), torch.empty_like(x).detach())
        with pytest.raises(RuntimeError, match="forward"):
            torch.ops.diffusers_amd.layer_norm(d)
