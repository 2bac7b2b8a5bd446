"""The transformer block's operators on torch tensors: layer norm, gated feed-forward and cross attention, with their gradients.

Each call runs the library's own kernels (``sde_layer_norm_*``, ``sde_gated_ff_*``, ``sde_cross_attention_*`` of include/sdengine.h) on the
current stream of the tensors' device and returns without waiting.  fp16, bf16 and fp32 tensors on a GPU; there is no CPU form.  The
functions take part in autograd (first derivatives).  Tensors may be strided views: one whose last axis is not contiguous, or whose rows do
not start on 16 bytes where the operator needs that, is copied first.

    y = layer_norm(x, weight, bias)
    o = cross_attention(q, k, v, kv_lens=lens)           # prompts of different lengths
    h = gated_ff(x, weight, bias, activation="gelu")     # GEGLU; "silu": SwiGLU

Calls can be captured into a graph.  A backward pass that is to be captured is taken with ``torch.autograd.grad`` of a forward pass in
the same capture: ``.backward()`` adds into ``.grad`` through nodes that belong to the stream on which the leaves were first used.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["layer_norm", "gated_ff", "cross_attention"]

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_ACTIVATIONS = {"gelu": 0, "gelu_tanh": 1, "silu": 2}
_checked = None


def _library():
    """The library, once it is known to share torch's HIP runtime (streams and tensors of one are unknown to another)."""
    global _checked
    if _checked is None:
        handle = _lib.lib()
        try:
            with open("/proc/self/maps") as f:
                runtimes = {line.split()[-1] for line in f if "libamdhip64" in line}
        except OSError:
            runtimes = set()
        if len(runtimes) > 1:
            raise RuntimeError("two HIP runtimes are loaded (" + ", ".join(sorted(runtimes)) + "): import torch before diffusers_amd's library is loaded")
        _checked = handle
    return _checked


def _same(x, **others):
    """Every tensor that is given is on x's device."""
    if not isinstance(x, torch.Tensor) or x.device.type != "cuda":
        raise ValueError("the operators take tensors on a GPU")
    if x.dtype not in _DTYPES:
        raise TypeError(f"fp16, bf16 or fp32 tensors, not {x.dtype}")
    for name, t in others.items():
        if t is not None and t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, the first tensor on {x.device}")


def _exec(device, workspace=None):
    return _lib.OpExec(device.index, torch.cuda.current_stream(device).cuda_stream, workspace.data_ptr() if workspace is not None else None,
                       workspace.numel() if workspace is not None else 0)


def _workspace(query, args, device, *direction):
    n = C.c_size_t()
    _lib.check(query(args, *direction, n))
    return torch.empty(n.value, dtype=torch.uint8, device=device) if n.value else None


def _ptr(t):
    return None if t is None else t.data_ptr()


def _rows(x, cols, align):
    """x as [rows, cols] with contiguous rows that do not overlap, every row on `align` bytes; copied where it has to be."""
    if x.dim() != 2:
        x = x.reshape(-1, cols) if cols else x
    e = x.element_size()
    if x.stride(1) != 1 and cols > 1 or (x.shape[0] > 1 and x.stride(0) < cols):
        x = x.contiguous()
    if x.data_ptr() % align or (x.stride(0) * e % align and x.shape[0] > 1) or (align > 1 and x.stride(0) * e >= 1 << 23):
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _ld(x, cols):
    return x.stride(0) if x.shape[0] > 1 else cols


def _param(p, like, shape, name):
    if p is None:
        return None
    if tuple(p.shape) != shape:
        raise ValueError(f"{name} has shape {tuple(p.shape)}, not {shape}")
    if p.dtype not in (like.dtype, torch.float32):
        raise TypeError(f"{name} is {p.dtype}: {like.dtype} or torch.float32")
    return p.contiguous()


# ---------------------------------------------------------------------------------------------- layer norm

def _ln_forward(x2, weight, bias, eps, stats):
    rows, cols = x2.shape
    y = torch.empty((rows, cols), dtype=x2.dtype, device=x2.device)
    mean, rstd = (torch.empty(rows, dtype=torch.float32, device=x2.device) for _ in range(2)) if stats else (None, None)
    param = weight if weight is not None else bias
    a = _lib.LayerNormArgs(_DTYPES[x2.dtype], _DTYPES[param.dtype if param is not None else x2.dtype], rows, cols, _ld(x2, cols), cols, 0, 0, eps,
                           x2.data_ptr(), _ptr(weight), _ptr(bias), y.data_ptr(), _ptr(mean), _ptr(rstd))
    _lib.check(_library().sde_layer_norm_forward(a, _exec(x2.device)))
    return y, mean, rstd


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        cols = x.shape[-1]
        x2 = _rows(x, cols, 1)
        y, mean, rstd = _ln_forward(x2, weight, bias, eps, True)
        ctx.save_for_backward(x2, weight, bias, mean, rstd)
        ctx.eps = eps
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x2, weight, bias, mean, rstd = ctx.saved_tensors
        rows, cols = x2.shape
        d2 = _rows(dy, cols, 1)
        dev = x2.device
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        dx = torch.empty((rows, cols), dtype=x2.dtype, device=dev) if want_x else None
        dw = torch.empty_like(weight) if want_w else None
        db = torch.empty_like(bias) if want_b else None
        param = weight if weight is not None else bias
        a = _lib.LayerNormArgs(_DTYPES[x2.dtype], _DTYPES[param.dtype if param is not None else x2.dtype], rows, cols, _ld(x2, cols), cols, _ld(d2, cols),
                               cols, ctx.eps, x2.data_ptr(), _ptr(weight), _ptr(bias), None, mean.data_ptr(), rstd.data_ptr(), d2.data_ptr(), _ptr(dx),
                               _ptr(dw), _ptr(db))
        L = _library()
        ws = _workspace(L.sde_layer_norm_workspace, a, dev)
        _lib.check(L.sde_layer_norm_backward(a, _exec(dev, ws)))
        return dx.view(dy.shape) if want_x else None, dw, db, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis.  weight and bias: [C], both of x's type or both fp32, either may be left
    out.  Statistics and sums are fp32.  Gradients for x, weight and bias."""
    _same(x, weight=weight, bias=bias)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("layer_norm needs a last axis that is not empty")
    cols = x.shape[-1]
    weight, bias = _param(weight, x, (cols,), "weight"), _param(bias, x, (cols,), "bias")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias have one type")
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _ln_forward(_rows(x, cols, 1), weight, bias, float(eps), False)[0].view(x.shape)


# ---------------------------------------------------------------------------------------------- gated feed-forward

def _ff_forward(x2, weight, bias, act):
    (m, k), f = x2.shape, weight.shape[0] // 2
    h = torch.empty((m, f), dtype=x2.dtype, device=x2.device)
    t = _DTYPES[x2.dtype]
    a = _lib.GatedFfArgs(t, t if bias is None else _DTYPES[bias.dtype], act, m, k, f, _ld(x2, k), _ld(weight, k), f, 0, 0, 0, x2.data_ptr(),
                         weight.data_ptr(), _ptr(bias), h.data_ptr())
    L = _library()
    ws = _workspace(L.sde_gated_ff_workspace, a, x2.device, 0)
    _lib.check(L.sde_gated_ff_forward(a, _exec(x2.device, ws)))
    return h


class _GatedFf(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, act):
        x2, w2 = _rows(x, x.shape[-1], 16), _rows(weight, weight.shape[1], 16)
        ctx.save_for_backward(x2, w2, bias)
        ctx.act, ctx.x_shape = act, x.shape
        return _ff_forward(x2, w2, bias, act).view(*x.shape[:-1], weight.shape[0] // 2)

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x2, w2, bias = ctx.saved_tensors
        (m, k), f = x2.shape, w2.shape[0] // 2
        d2 = _rows(dh, f, 16)
        dev = x2.device
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        dx = torch.empty((m, k), dtype=x2.dtype, device=dev) if want_x else None
        dw = torch.empty((2 * f, k), dtype=w2.dtype, device=dev) if want_w else None
        db = torch.empty_like(bias) if want_b else None
        t = _DTYPES[x2.dtype]
        a = _lib.GatedFfArgs(t, t if bias is None else _DTYPES[bias.dtype], ctx.act, m, k, f, _ld(x2, k), _ld(w2, k), f, _ld(d2, f), k, k,
                             x2.data_ptr(), w2.data_ptr(), _ptr(bias), None, d2.data_ptr(), _ptr(dx), _ptr(dw), _ptr(db))
        L = _library()
        ws = _workspace(L.sde_gated_ff_workspace, a, dev, 1)
        _lib.check(L.sde_gated_ff_backward(a, _exec(dev, ws)))
        return dx.view(ctx.x_shape) if want_x else None, dw, db, None


def gated_ff(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "gelu") -> torch.Tensor:
    """(x Wv^T + bv) * act(x Wg^T + bg): both projections, the activation and the product in one kernel.  x [..., K]; weight [2F, K], the F value
    rows first, then the F gate rows; bias [2F] of x's type or fp32, or None; result [..., F].  activation: "gelu" (erf), "gelu_tanh" or
    "silu".  K and F are multiples of 8 (fp32: of 4).  Gradients for x, weight and bias; the backward pass forms the projections again."""
    _same(x, weight=weight, bias=bias)
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation is one of {', '.join(_ACTIVATIONS)}, not {activation!r}")
    step = 16 // x.element_size()
    if x.dim() == 0 or weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.shape[0] % 2:
        raise ValueError(f"x [..., K] and weight [2F, K], not {tuple(x.shape)} and {tuple(weight.shape)}")
    if weight.dtype != x.dtype:
        raise TypeError(f"weight is {weight.dtype}, x is {x.dtype}")
    if x.shape[-1] == 0 or weight.shape[0] == 0 or x.shape[-1] % step or weight.shape[0] // 2 % step:
        raise ValueError(f"K and F are positive multiples of {step} for {x.dtype}")
    bias = _param(bias, x, (weight.shape[0],), "bias")
    act = _ACTIVATIONS[activation]
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        return _GatedFf.apply(x, weight, bias, act)
    x2 = _rows(x, x.shape[-1], 16)
    return _ff_forward(x2, _rows(weight, weight.shape[1], 16), bias, act).view(*x.shape[:-1], weight.shape[0] // 2)


# ---------------------------------------------------------------------------------------------- cross attention

def _heads(x):
    """x [B, S, H, D] as the kernels take it: last axis contiguous, every (b, s, h) on 16 bytes, offsets inside a tile within 2 GB."""
    step, (b, s, h, d) = 16 // x.element_size(), x.stride()
    if d != 1 or b % step or s % step or h % step or x.data_ptr() % 16 or (65 * s + x.shape[2] * h + x.shape[3]) * x.element_size() >= 1 << 31:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


_NONE3 = (0, 0, 0)


def _xa_args(q, k, v, o, lse, lens, scale, do=None, dq=None, dk=None, dv=None):
    b, sq, h, d = q.shape
    q_lens, kv_lens, mask = lens

    def strides(t):
        return _NONE3 if t is None else t.stride()[:3]

    return _lib.CrossAttentionArgs(_DTYPES[q.dtype], b, sq, k.shape[1], h, k.shape[2], d, scale, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                                   _ptr(lse), _ptr(do), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(q_lens), _ptr(kv_lens), _ptr(mask),
                                   mask.stride(0) if mask is not None else 0, q.stride()[:3], k.stride()[:3], v.stride()[:3], o.stride()[:3], strides(do),
                                   strides(dq), strides(dk), strides(dv))


def _xa_forward(q, k, v, lens, scale, want_lse):
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device) if want_lse else None
    a = _xa_args(q, k, v, o, lse, lens, scale)
    L = _library()
    ws = _workspace(L.sde_cross_attention_workspace, a, q.device, 0)
    _lib.check(L.sde_cross_attention_forward(a, _exec(q.device, ws)))
    return o, lse


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_lens, kv_lens, mask, scale):
        q, k, v = _heads(q), _heads(k), _heads(v)
        o, lse = _xa_forward(q, k, v, (q_lens, kv_lens, mask), scale, True)
        ctx.save_for_backward(q, k, v, o, lse, q_lens, kv_lens, mask)
        ctx.scale = scale
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse, *lens = ctx.saved_tensors
        do = _heads(do)
        want_q, want_k, want_v = ctx.needs_input_grad[:3]
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) if want else None for t, want in ((q, want_q), (k, want_k), (v, want_v)))
        a = _xa_args(q, k, v, o, lse, lens, ctx.scale, do, dq, dk, dv)
        L = _library()
        ws = _workspace(L.sde_cross_attention_workspace, a, q.device, 1)
        _lib.check(L.sde_cross_attention_backward(a, _exec(q.device, ws)))
        return dq, dk, dv, None, None, None, None


def _lens(t, b, name):
    if t is None:
        return None
    if t.dtype not in (torch.int32, torch.int64) or tuple(t.shape) != (b,):
        raise ValueError(f"{name} is an int32 (or int64) tensor of shape ({b},)")
    return t.to(torch.int32).contiguous()


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, q_lens: Optional[torch.Tensor] = None, kv_lens: Optional[torch.Tensor] = None,
                    key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """softmax(scale q k^T) v with keys and values of another length than the queries.  q [B, Sq, H, D]; k, v [B, Skv, Hkv, D], H a multiple of Hkv (shared
    heads); D at most 256 and a multiple of 8 (fp32: of 4); scale defaults to D ** -0.5.  q_lens, kv_lens: int32 [B] on the device, how many of the padded
    queries and keys count; key_mask: bool [B, Skv], true where a key counts.  What does not count is not read; a query that does not count, or that
    no key counts for, gives zeros.  Gradients for q, k and v."""
    _same(q, k=k, v=v, q_lens=q_lens, kv_lens=kv_lens, key_mask=key_mask)
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"q [B, Sq, H, D] and k, v [B, Skv, Hkv, D], not {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("q, k and v have one type")
    b, _, h, d = q.shape
    step = 16 // q.element_size()
    if k.shape[2] == 0 or h == 0 or h % k.shape[2] or not 0 < d <= 256 or d % step:
        raise ValueError(f"H is a multiple of Hkv, and D at most 256 and a multiple of {step} for {q.dtype}")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0 < scale < float("inf"):
        raise ValueError("scale is positive and finite")
    q_lens, kv_lens = _lens(q_lens, b, "q_lens"), _lens(kv_lens, b, "kv_lens")
    if key_mask is not None:
        if key_mask.dtype not in (torch.bool, torch.uint8) or tuple(key_mask.shape) != (b, k.shape[1]):
            raise ValueError(f"key_mask is a bool tensor of shape {(b, k.shape[1])}")
        if (key_mask.stride(1) != 1 and k.shape[1] > 1) or (b > 1 and key_mask.stride(0) < k.shape[1]):
            key_mask = key_mask.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _CrossAttention.apply(q, k, v, q_lens, kv_lens, key_mask, scale)
    return _xa_forward(_heads(q), _heads(k), _heads(v), (q_lens, kv_lens, key_mask), scale, False)[0]
