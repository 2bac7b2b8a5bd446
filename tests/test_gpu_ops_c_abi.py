"""GPU: what include/sdengine.h says of the operators' tensors and the torch binding never does: outputs with strides of their own, outputs in place of inputs, one workspace for
call after call.  What a call does not own keeps its values.  The torch binding runs the same kernels on packed tensors, so the bits are the same."""
import ctypes as C

import pytest
import torch

from diffusers_amd import _lib, ops

pytestmark = pytest.mark.gpu
T = {"f16": (0, torch.float16), "bf16": (1, torch.bfloat16), "f32": (2, torch.float32)}
L = _lib.lib()


def r(*s, seed=0, dtype=torch.float16):
    return torch.randn(*s, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def execute(fn, query, args, extra=(), ws=None):
    n = C.c_size_t()
    _lib.check(query(args, *extra, n))
    if ws is None:
        ws = torch.full((n.value + 256,), 0xFF, dtype=torch.uint8, device="cuda")           # NaN, were it read before it is written
    assert ws.numel() >= n.value
    _lib.check(fn(args, _lib.OpExec(0, torch.cuda.current_stream().cuda_stream, ws.data_ptr(), ws.numel())))
    return ws


def p(t):
    return t.data_ptr() if t is not None else None


ROWS = [(5, 47), (700, 320), (40, 1280), (9, 4099), (3, 20001), (600, 8), (2, 1)]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,c", ROWS)
def test_layer_norm_in_place_and_with_rows_apart(rows, c, dtype):
    code, t = T[dtype]
    x, w, b, dy = r(rows, c, dtype=t), r(c, seed=1, dtype=t), r(c, seed=2, dtype=t), r(rows, c, seed=3, dtype=t)
    xs, ws_, bs = (v.clone().requires_grad_() for v in (x, w, b))
    y = ops.layer_norm(xs, ws_, bs)
    dx, dw, db = torch.autograd.grad(y, (xs, ws_, bs), dy)
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    out = x.clone()                                                                            # y in place of x
    fwd = lambda X, Y, ldx, ldy: _lib.LayerNormArgs(code, code, rows, c, ldx, ldy, 0, 0, 1e-5, p(X), p(w), p(b), p(Y), p(mean), p(rstd))
    execute(L.sde_layer_norm_forward, L.sde_layer_norm_workspace, fwd(out, out, c, c))
    assert torch.equal(out, y)
    wide = torch.full((rows + 1, c + 3), 7.0, device="cuda", dtype=t)                          # rows apart
    execute(L.sde_layer_norm_forward, L.sde_layer_norm_workspace, fwd(x, wide, c, c + 3))
    assert torch.equal(wide[:rows, :c], y) and (wide[rows:] == 7).all() and (wide[:, c:] == 7).all()
    gw, gb = torch.empty_like(w), torch.empty_like(b)

    def bwd(D, DX, ld_dy, ld_dx):
        a = fwd(x, None, c, c)
        a.ld_dy, a.ld_dx, a.dy, a.dx, a.dgamma, a.dbeta = ld_dy, ld_dx, p(D), p(DX), p(gw), p(gb)
        execute(L.sde_layer_norm_backward, L.sde_layer_norm_workspace, a)
        assert torch.equal(gw, dw) and torch.equal(gb, db)

    d = dy.clone()                                                                             # dx in place of dy
    bwd(d, d, c, c)
    assert torch.equal(d, dx)
    wide.fill_(7.0)
    bwd(dy, wide, c, c + 3)
    assert torch.equal(wide[:rows, :c], dx) and (wide[rows:] == 7).all() and (wide[:, c:] == 7).all()
    wide[:rows, :c] = dy                                                                       # in place and rows apart
    bwd(wide, wide, c + 3, c + 3)
    assert torch.equal(wide[:rows, :c], dx) and (wide[rows:] == 7).all() and (wide[:, c:] == 7).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("m,k,f", [(70, 64, 96), (1, 72, 136), (300, 200, 264), (2059, 80, 2856), (1507, 48, 1032)])
def test_gated_ff_with_rows_apart(m, k, f, dtype):
    code, t = T[dtype]
    x, w, b, dh = r(m, k, dtype=t), r(2 * f, k, seed=1, dtype=t) * k ** -0.5, r(2 * f, seed=2, dtype=t), r(m, f, seed=3, dtype=t)
    leaves = [v.clone().requires_grad_() for v in (x, w, b)]
    h = ops.gated_ff(*leaves)
    dx, dw, db = torch.autograd.grad(h, leaves, dh)
    X, W, H, D, DX, DW = (torch.full((n + 2, c + 24), 7.0, device="cuda", dtype=t) for n, c in ((m, k), (2 * f, k), (m, f), (m, f), (m, k), (2 * f, k)))
    DB = torch.full((2 * f + 8,), 7.0, device="cuda", dtype=t)
    X[:m, :k], W[:2 * f, :k], D[:m, :f] = x, w, dh
    a = _lib.GatedFfArgs(code, code, 0, m, k, f, k + 24, k + 24, f + 24, f + 24, k + 24, k + 24, p(X), p(W), p(b), p(H), p(D), p(DX), p(DW), p(DB))
    execute(L.sde_gated_ff_forward, L.sde_gated_ff_workspace, a, (0,))
    execute(L.sde_gated_ff_backward, L.sde_gated_ff_workspace, a, (1,))
    for got, want in ((H, h), (DX, dx), (DW, dw)):
        n, c = want.shape
        assert torch.equal(got[:n, :c], want) and (got[n:] == 7).all() and (got[:, c:] == 7).all()
    assert torch.equal(DB[:2 * f], db) and (DB[2 * f:] == 7).all()


def laid_out(shape, order, pad, t):
    """A [B, S, H, D] view of a larger tensor whose axes lie in the given order, D padded."""
    sizes = [shape[i] + (pad if i < 3 else 8) for i in order]
    base = torch.full(sizes, 7.0, device="cuda", dtype=t)
    view = base.permute(*[order.index(i) for i in range(4)])
    return base, view[tuple(slice(0, n) for n in shape)]


@pytest.mark.parametrize("order", [(0, 1, 2, 3), (0, 2, 1, 3), (2, 0, 1, 3), (1, 2, 0, 3)])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("b,sq,skv,h,hkv,d", [(2, 70, 90, 4, 2, 64), (3, 1, 700, 4, 2, 128), (2, 300, 33, 3, 3, 40), (1, 40, 2000, 2, 1, 96)])
def test_cross_attention_with_outputs_laid_out_otherwise(b, sq, skv, h, hkv, d, dtype, order):
    code, t = T[dtype]
    q, k, v, do = r(b, sq, h, d, dtype=t), r(b, skv, hkv, d, seed=1, dtype=t), r(b, skv, hkv, d, seed=2, dtype=t), r(b, sq, h, d, seed=3, dtype=t)
    lens = torch.tensor([skv, skv // 2, 1][:b], dtype=torch.int32, device="cuda")
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    o = ops.cross_attention(*leaves, kv_lens=lens)
    want = (o.detach(), *torch.autograd.grad(o, leaves, do))
    pairs = [laid_out(x.shape, order, 1, t) for x in want]
    lse = torch.full((b, sq, h), 7.0, device="cuda")
    a = _lib.CrossAttentionArgs(code, b, sq, skv, h, hkv, d, d ** -0.5, p(q), p(k), p(v), p(pairs[0][1]), p(lse), p(do), *(p(x[1]) for x in pairs[1:]), None, p(lens), None, 0)
    for name, x in zip(("q", "k", "v", "o", "do", "dq", "dk", "dv"), (q, k, v, pairs[0][1], do, *(x[1] for x in pairs[1:]))):
        setattr(a, name + "_stride", (C.c_int64 * 3)(*x.stride()[:3]))
    execute(L.sde_cross_attention_forward, L.sde_cross_attention_workspace, a, (0,))
    execute(L.sde_cross_attention_backward, L.sde_cross_attention_workspace, a, (1,))
    for (base, view), w, name in zip(pairs, want, ("o", "dq", "dk", "dv")):
        assert torch.equal(view, w), name
        view.fill_(7.0)
        assert (base == 7).all(), name


def test_one_workspace_for_call_after_call():
    """The operators' backward passes on one stream with the same scratch, without a wait between them, twice."""
    x, w, b, dy = r(700, 320), r(320, seed=1), r(320, seed=2), r(700, 320, seed=3)
    wf, bf, dh = r(2 * 520, 320, seed=4) * 320 ** -0.5, r(2 * 520, seed=5), r(700, 520, seed=6)
    q, k, v, do = r(2, 40, 4, 64, seed=7), r(2, 900, 2, 64, seed=8), r(2, 900, 2, 64, seed=9), r(2, 40, 4, 64, seed=10)

    def grads(f, *args, d):
        leaves = [t.clone().requires_grad_() for t in args]
        return torch.autograd.grad(f(*leaves), leaves, d)

    want = [*grads(ops.layer_norm, x, w, b, d=dy), *grads(ops.gated_ff, x, wf, bf, d=dh), *grads(ops.cross_attention, q, k, v, d=do)]
    mean, rstd, y, h, o, lse = torch.empty(700, device="cuda"), torch.empty(700, device="cuda"), torch.empty_like(x), torch.empty_like(dh), torch.empty_like(q), torch.empty(2, 40, 4, device="cuda")
    ln = _lib.LayerNormArgs(0, 0, 700, 320, 320, 320, 320, 320, 1e-5, p(x), p(w), p(b), p(y), p(mean), p(rstd), p(dy))
    ff = _lib.GatedFfArgs(0, 0, 0, 700, 320, 520, 320, 320, 520, 520, 320, 320, p(x), p(wf), p(bf), p(h), p(dh))
    xa = _lib.CrossAttentionArgs(0, 2, 40, 900, 4, 2, 64, 0.125, p(q), p(k), p(v), p(o), p(lse), p(do))
    for name, t in zip(("q", "k", "v", "o", "do", "dq", "dk", "dv"), (q, k, v, o, do, q, k, v)):
        setattr(xa, name + "_stride", (C.c_int64 * 3)(*t.stride()[:3]))
    ws = torch.full((64 << 20,), 0xFF, dtype=torch.uint8, device="cuda")
    for fn, query, a, extra in ((L.sde_layer_norm_forward, L.sde_layer_norm_workspace, ln, ()), (L.sde_gated_ff_forward, L.sde_gated_ff_workspace, ff, (0,)),
                                (L.sde_cross_attention_forward, L.sde_cross_attention_workspace, xa, (0,))):
        execute(fn, query, a, extra, ws)
    for _ in range(2):
        got = [torch.full_like(t, 7.0) for t in want]
        ln.dx, ln.dgamma, ln.dbeta = map(p, got[:3])
        ff.dx, ff.dweight, ff.dbias = map(p, got[3:6])
        xa.dq, xa.dk, xa.dv = map(p, got[6:])
        execute(L.sde_layer_norm_backward, L.sde_layer_norm_workspace, ln, (), ws)
        execute(L.sde_gated_ff_backward, L.sde_gated_ff_workspace, ff, (1,), ws)
        execute(L.sde_cross_attention_backward, L.sde_cross_attention_workspace, xa, (1,), ws)
        for i, (g, t) in enumerate(zip(got, want)):
            assert torch.equal(g, t), i
