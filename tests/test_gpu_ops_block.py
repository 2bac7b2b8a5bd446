"""GPU: the operators together, as a transformer block uses them -- forward, gradients, captured graphs, streams, threads."""
import threading

import pytest
import torch

from diffusers_amd import ops

pytestmark = pytest.mark.gpu


class Block(torch.nn.Module):
    """norm - cross attention to prompts of different lengths - norm - gated feed-forward, with the projections around them."""

    def __init__(self, c, heads, cross, dtype, seed=0):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.nn.Parameter((torch.randn(*s, generator=g) * s[-1] ** -0.5).to(dtype).cuda())
        v = lambda n, m: torch.nn.Parameter((torch.randn(n, generator=g) * 0.1 + m).to(dtype).cuda())
        self.heads = heads
        self.g1, self.b1, self.g2, self.b2 = v(c, 1), v(c, 0), v(c, 1), v(c, 0)
        self.wq, self.wk, self.wv, self.wo = r(c, c), r(c, cross), r(c, cross), r(c, c)
        self.wff, self.bff, self.wdown = r(8 * c, c), v(8 * c, 0), r(c, 4 * c)

    def forward(self, x, ehs, lens):
        b, s, c = x.shape
        split = lambda t: t.view(b, -1, self.heads, c // self.heads)
        h = ops.layer_norm(x, self.g1, self.b1)
        o = ops.cross_attention(split(h @ self.wq.t()), split(ehs @ self.wk.t()), split(ehs @ self.wv.t()), kv_lens=lens)
        x = x + o.reshape(b, s, c) @ self.wo.t()
        return x + ops.gated_ff(ops.layer_norm(x, self.g2, self.b2), self.wff, self.bff) @ self.wdown.t()

    def plain(self, p, x, ehs, lens):
        """The same in 64 bits; p: the parameters by name."""
        b, s, c = x.shape
        norm = lambda t, g, bb: (t - t.mean(-1, keepdim=True)) / (t.var(-1, correction=0, keepdim=True) + 1e-5).sqrt() * g + bb
        split = lambda t: t.view(b, -1, self.heads, c // self.heads).transpose(1, 2)
        q, k, v = split(norm(x, p["g1"], p["b1"]) @ p["wq"].t()), split(ehs @ p["wk"].t()), split(ehs @ p["wv"].t())
        sc = (q @ k.transpose(2, 3).contiguous()) * (c // self.heads) ** -0.5
        on = torch.arange(ehs.shape[1], device=x.device) < lens[:, None]
        w = torch.softmax(sc.masked_fill(~on[:, None, None], float("-inf")), -1)
        x = x + (w @ v).transpose(1, 2).reshape(b, s, c) @ p["wo"].t()
        a, g = (norm(x, p["g2"], p["b2"]) @ p["wff"].t() + p["bff"]).chunk(2, -1)
        return x + (a * g * torch.special.ndtr(g)) @ p["wdown"].t()


def inputs(dtype, c=320, cross=128, b=3, s=300, skv=77, seed=1):
    g = torch.Generator().manual_seed(seed)
    r = lambda *sh: torch.randn(*sh, generator=g).to(dtype).cuda()
    return r(b, s, c), r(b, skv, cross), torch.tensor([skv, 20, 1], dtype=torch.int32, device="cuda"), r(b, s, c)


# relative 2-norm errors.  fp32: ten stages, each a product or sum of up to 1280 terms whose rounding errors add up as their square root at the least and in full at the
# most (400 v between the two), and each passed on with a factor of at most 4 (the norms divide by sigma ~ 1): 10 x 400 x 4 x 2^-24 = 9.6e-4.  16-bit types: the
# stages' results are rounded, ten roundings of u / sqrt(3) (uniform) that add in squares, times the same factor 4, and two for the operands rounded inside:
# 12^0.5 x 4 x u / 3^0.5 = 8 u.
BARS = {torch.float32: 9.6e-4, torch.float16: 8 * 2.0 ** -11, torch.bfloat16: 8 * 2.0 ** -8}


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_block_and_all_its_gradients(dtype):
    m = Block(320, 8, 128, dtype)
    x, ehs, lens, dy = inputs(dtype)
    x.requires_grad_()
    ehs.requires_grad_()
    names = [n for n, _ in m.named_parameters()]
    params = [t for _, t in m.named_parameters()]
    y = m(x, ehs, lens)
    grads = torch.autograd.grad(y, [x, ehs, *params], dy)
    wide = [t.detach().double().requires_grad_() for t in (x, ehs, *params)]
    want_y = m.plain(dict(zip(names, wide[2:])), wide[0], wide[1], lens)
    want = torch.autograd.grad(want_y, wide, dy.double())
    for name, a, b in zip(["y", "x", "ehs", *names], (y, *grads), (want_y, *want)):
        rel = ((a.double() - b).norm() / b.norm()).item()
        assert rel < BARS[dtype], (name, rel)
    past = torch.arange(77, device="cuda") >= lens[:, None]
    assert not grads[1][past].any()                                     # encoder states past a prompt's length get no gradient


def step(m, x, ehs, lens, dy):
    y = m(x, ehs, lens)
    return (y.detach(), *torch.autograd.grad(y, [x, ehs, *m.parameters()], dy))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_same_call_gives_the_same_bits(dtype):
    m = Block(320, 8, 128, dtype)
    x, ehs, lens, dy = inputs(dtype)
    x.requires_grad_()
    ehs.requires_grad_()
    first = step(m, x, ehs, lens, dy)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, step(m, x, ehs, lens, dy)))


def test_captured_forward_and_backward_replay_as_eager():
    m = Block(64, 2, 64, torch.float16)
    static = inputs(torch.float16, c=64, cross=64, s=130)
    for t in static[:2]:
        t.requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(m, *static)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                                  # two graphs, each with scratch of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(m, *static)
        graphs.append((g, out))
    for seed in range(3):
        fresh = inputs(torch.float16, c=64, cross=64, s=130, seed=10 + seed)
        with torch.no_grad():
            for a, b in zip(static, fresh):
                a.copy_(b)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        eager = [t.clone().requires_grad_(t.requires_grad) for t in static]
        want = step(m, *eager)
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), seed
        streams = [torch.cuda.Stream() for _ in graphs]                  # and both at once
        for (g, _), s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), seed


def test_a_capture_is_refused_while_a_graph_of_the_same_leaves_lives():
    w = torch.ones(64, device="cuda", requires_grad=True)
    x = torch.randn(4, 64, device="cuda")
    alive = ops.layer_norm(x, w)                                        # built on the default stream, kept
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="alive"):
            ops.layer_norm(x, w)
        with torch.no_grad():
            y = ops.layer_norm(x, w)                                     # without gradients it is fine
    g.replay()
    assert torch.equal(y, alive)
    del alive
    g2 = torch.cuda.CUDAGraph()
    dy = torch.ones(4, 64, device="cuda")
    with torch.cuda.graph(g2):
        gw, = torch.autograd.grad(ops.layer_norm(x, w), w, dy)
    g2.replay()
    again, = torch.autograd.grad(ops.layer_norm(x, w), w, dy)
    assert torch.equal(gw, again)


def test_on_two_streams_and_from_two_threads_at_once():
    m = Block(320, 8, 128, torch.float16)
    data = [inputs(torch.float16, seed=20 + i) for i in range(2)]
    want = []
    for d in data:
        for t in d[:2]:
            t.requires_grad_()
        want.append(step(m, *d))
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(5):
                    got[i] = step(m, *data[i])
            s.synchronize()
        except Exception as e:                                            # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_first_derivatives_only_and_saved_tensors_are_watched():
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    w = torch.randn(32, 64, device="cuda", requires_grad=True)
    q = torch.randn(1, 4, 2, 64, device="cuda", requires_grad=True)
    for y in (ops.layer_norm(x), ops.gated_ff(x, w), ops.cross_attention(q, q, q)):
        leaf = q if y.dim() == 4 else x
        with pytest.raises(RuntimeError, match="first derivatives"):
            torch.autograd.grad(y.sum(), leaf, create_graph=True)
    y = ops.gated_ff(x, w)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_backward_adds_into_grad_and_skips_what_is_frozen():
    m = Block(320, 8, 128, torch.bfloat16)
    m.wff.requires_grad_(False)
    m.g1.requires_grad_(False)
    x, ehs, lens, dy = inputs(torch.bfloat16)
    m(x, ehs, lens).backward(dy)
    first = {n: p.grad.clone() for n, p in m.named_parameters() if p.requires_grad}
    m(x, ehs, lens).backward(dy)
    assert m.wff.grad is None and m.g1.grad is None
    for n, p in m.named_parameters():
        if p.requires_grad:
            assert torch.equal(p.grad, first[n] + first[n]), n
