"""GPU: a captured call whose backward pass would reach another stream's nodes is refused, in order, however the leaves are reached."""
import pytest
import torch

from diffusers_amd import ops

pytestmark = pytest.mark.gpu


def r(*s, seed=0):
    return torch.randn(*s, generator=torch.Generator().manual_seed(seed)).half().cuda()


# name -> (leaf, call of it): leaves behind views, casts, products and copies of arguments
def reached():
    x, wf, k = r(4, 64, seed=1), r(96, 64, seed=2), r(2, 9, 2, 64, seed=3)
    return {
        "a view": (r(8, 8, 64, seed=4), lambda t: ops.layer_norm(t.view(64, 64))),
        "columns": (r(64, 96, seed=5), lambda t: ops.gated_ff(x, t.t())),
        "a weight out of a larger one": (r(128, seed=6), lambda t: ops.layer_norm(x, t[::2])),
        "one row for all": (r(1, 64, seed=7), lambda t: ops.gated_ff(t.expand(4, 64), wf)),
        "a cast": (r(64, seed=8), lambda t: ops.layer_norm(x.float(), t.float())),
        "a product before": (r(64, 64, seed=9), lambda t: ops.gated_ff(x @ t, wf)),
        "packed keys": (r(2, 9, 2, 2, 64, seed=10), lambda t: ops.cross_attention(k, t[:, :, 0], t[:, :, 1])),
        "the operators in a row": (r(64, seed=11), lambda t: ops.gated_ff(ops.layer_norm(x, t), wf)),
    }


NAMES = ["a view", "columns", "a weight out of a larger one", "one row for all", "a cast", "a product before", "packed keys", "the operators in a row"]


@pytest.mark.parametrize("name", NAMES)
def test_refused_while_another_graph_lives_and_captured_after(name):
    leaf, call = reached()[name]
    leaf.requires_grad_()
    alive = call(leaf)                                                   # on the default stream, kept
    dy = torch.ones_like(alive)
    want, = torch.autograd.grad(alive, leaf, dy, retain_graph=True)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="alive"):
            call(leaf)
        with torch.no_grad():
            y = call(leaf)
    g.replay()
    assert torch.equal(y, alive)
    del alive
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got, = torch.autograd.grad(call(leaf), leaf, dy)
    for _ in range(3):
        got.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_a_step_from_outside_of_the_capture():
    """Its gradient is refused in the captured backward pass; the call, and the gradients of the leaves beside it, are not."""
    x, w = r(4, 64, seed=1).requires_grad_(), r(64, seed=2).requires_grad_()
    h = x * 2                                                            # outside
    dy = torch.ones(4, 64, device="cuda", dtype=torch.half)
    want, = torch.autograd.grad(ops.layer_norm(h.detach(), w), w, dy)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.layer_norm(h, w)
        with pytest.raises(RuntimeError, match="another stream"):
            torch.autograd.grad(y, (h, w), dy, retain_graph=True)
        gw, = torch.autograd.grad(y, w, dy)
    for _ in range(2):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(gw, want)


def test_refused_under_a_dispatch_mode_too():
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    x, w = r(4, 64, seed=1), r(64, seed=2).requires_grad_()
    alive = ops.layer_norm(x, w)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with Watch(), pytest.raises(RuntimeError, match="alive"):
            ops.layer_norm(x, w)
        with torch.no_grad():
            y = ops.layer_norm(x, w)
    g.replay()
    assert torch.equal(y, alive)
