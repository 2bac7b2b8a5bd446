"""GPU: what torch's tracers record of the operators runs the kernels, forward and backward, on other inputs than those it was recorded with."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from diffusers_amd import _lib, ops

pytestmark = pytest.mark.gpu


def r(*s, seed=0, dtype=torch.float16):
    return torch.randn(*s, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def lens(*n, dtype=torch.int32):
    return torch.tensor(n, dtype=dtype, device="cuda")


def case(name, seed=0):
    """A function of tensors alone, and its tensors; those of floating point take gradients."""
    mask = torch.tensor([[True] * 8 + [False]] * 2, device="cuda")
    q, k, v = r(2, 9, 4, 64, seed=seed), r(2, 9, 2, 64, seed=seed + 1), r(2, 9, 2, 64, seed=seed + 2)
    return {
        "layer_norm": (lambda x, w, b: ops.layer_norm(x, w, b), [r(3, 5, 64, seed=seed), r(64, seed=seed + 1), r(64, seed=seed + 2)]),
        "layer_norm of a view": (lambda x, b: ops.layer_norm(x[:, 1:65], None, b), [r(6, 70, seed=seed), r(64, seed=seed + 1, dtype=torch.float32)]),
        "layer_norm of columns": (lambda x: ops.layer_norm(x.t()), [r(64, 6, seed=seed)]),
        "gated_ff": (lambda x, w, b: ops.gated_ff(x, w, b, activation="silu"), [r(3, 5, 64, seed=seed), r(96, 64, seed=seed + 1), r(96, seed=seed + 2)]),
        "gated_ff of a view": (lambda x, w: ops.gated_ff(x[:, 1:65], w[:, 3:67]), [r(6, 70, seed=seed), r(96, 70, seed=seed + 1)]),
        "cross_attention": (lambda q, k, v, n, m: ops.cross_attention(q, k, v, kv_lens=n, key_mask=m), [q, k, v, lens(9, 4), mask]),
        "cross_attention, long lengths": (lambda q, k, v, n: ops.cross_attention(q, k, v, q_lens=n, scale=0.2), [q, k, v, lens(9, 4, dtype=torch.int64)]),
        "cross_attention of a view": (lambda q, k, v: ops.cross_attention(q[..., 1:41], k[..., 2:42], v[..., 3:43]), [q, k, v]),
    }[name]


NAMES = ["layer_norm", "layer_norm of a view", "layer_norm of columns", "gated_ff", "gated_ff of a view", "cross_attention", "cross_attention, long lengths", "cross_attention of a view"]


def leaves_of(tensors):
    return [t.requires_grad_() for t in tensors if t.is_floating_point()]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("grad", [False, True])
def test_a_jit_trace_runs_the_kernels(name, grad):
    f, args = case(name)
    traced = torch.jit.trace(f, tuple(args), check_trace=False)
    assert "diffusers_amd::" in str(traced.graph)
    for seed in (0, 10):
        args = case(name, seed)[1]
        leaves = leaves_of(args) if grad else []
        got, want = traced(*args), f(*args)
        assert torch.equal(got, want)
        if grad:
            dy = torch.ones_like(want)
            assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, leaves, dy), torch.autograd.grad(want, leaves, dy)))


@pytest.mark.parametrize("mode", ["real", "fake"])
@pytest.mark.parametrize("name", NAMES)
def test_a_recorded_graph_runs_the_kernels(name, mode):
    f, args = case(name)
    g = make_fx(f, tracing_mode=mode)(*args)
    assert any("diffusers_amd" in str(n.target) for n in g.graph.nodes)
    for seed in (0, 10):
        args = case(name, seed)[1]
        assert torch.equal(g(*args), f(*args))


@pytest.mark.parametrize("mode", ["real", "fake"])
@pytest.mark.parametrize("name", NAMES)
def test_a_recorded_backward_pass_runs_the_kernels(name, mode):
    f, args = case(name)
    dy = r(*f(*args).shape, seed=30)

    def step(dy, *args):
        y = f(*args)
        return y.detach(), *torch.autograd.grad(y, [t for t in args if t.requires_grad], dy)

    leaves_of(args)
    g = make_fx(step, tracing_mode=mode)(dy, *args)
    assert sum("diffusers_amd" in str(n.target) for n in g.graph.nodes) == 2
    for seed in (0, 10):
        args = case(name, seed)[1]
        plain = g(dy, *args)                                            # the graph holds the backward pass itself
        leaves_of(args)
        assert all(torch.equal(a, b) for a, b in zip(plain, step(dy, *args)))


def test_a_trace_survives_saving_and_loading(tmp_path):
    f, args = case("gated_ff")
    torch.jit.trace(f, tuple(args), check_trace=False).save(str(tmp_path / "t.pt"))
    assert torch.equal(torch.jit.load(str(tmp_path / "t.pt"))(*args), f(*args))


def test_batches_of_calls():
    """torch.func.vmap: call by call."""
    x, w = r(3, 5, 64), r(64, seed=1)
    try:
        y = torch.func.vmap(lambda t: ops.layer_norm(t, w))(x)
    except RuntimeError:                                                # refused: as good
        return
    assert torch.equal(y, ops.layer_norm(x, w))


def test_what_the_library_refuses_in_a_backward_pass_is_its_own_error():
    """F = 2^21: past the backward pass's limit, not the forward pass's."""
    x, w = r(1, 8), torch.zeros(1 << 22, 8, device="cuda", dtype=torch.float16, requires_grad=True)
    h = ops.gated_ff(x, w)
    with pytest.raises(_lib.SdeError, match="too large") as e:
        torch.autograd.grad(h, w, torch.ones_like(h))
    assert e.value.status == 1


@pytest.mark.parametrize("name", ["layer_norm", "gated_ff", "cross_attention"])
def test_several_upstream_gradients_at_once(name):
    """is_grads_batched: the backward pass for each of them."""
    f, args = case(name)
    leaves = leaves_of(args)
    y = f(*args)
    dy = r(3, *y.shape, seed=31)
    got = torch.autograd.grad(y, leaves, dy, is_grads_batched=True, retain_graph=True)
    for i in range(3):
        assert all(torch.equal(a[i], b) for a, b in zip(got, torch.autograd.grad(y, leaves, dy[i], retain_graph=True)))


@pytest.mark.parametrize("name", ["layer_norm", "gated_ff", "cross_attention"])
def test_functional_transforms_are_right_or_refused(name):
    f, args = case(name)
    g = lambda x: f(x, *args[1:])
    assert torch.equal(torch.func.vmap(g)(torch.stack([args[0], 2 * args[0]])), torch.stack([g(args[0]), g(2 * args[0])]))
    assert torch.equal(torch.func.functionalize(g)(args[0]), g(args[0]))
    for transform in (torch.func.grad(lambda x: g(x).float().sum()), torch.func.jacrev(g), lambda x: torch.func.jvp(g, (x,), (x,))):
        with pytest.raises(RuntimeError):
            transform(args[0])


@pytest.mark.parametrize("name", ["layer_norm", "gated_ff", "cross_attention"])
def test_torchs_own_checks_of_an_operator(name):
    args = {"layer_norm": case(name)[1], "gated_ff": [*case(name)[1], 2], "cross_attention": case(name)[1][:3]}[name]
    leaves_of([t for t in args if isinstance(t, torch.Tensor)])
    torch.library.opcheck(getattr(torch.ops.diffusers_amd, name).default, tuple(args), test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))
