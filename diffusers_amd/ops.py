"""The transformer block's operators on torch tensors: layer norm, gated feed-forward and cross attention, with their gradients.

Each call runs the library's own kernels (``sde_layer_norm_*``, ``sde_gated_ff_*``, ``sde_cross_attention_*`` of include/sdengine.h) on the
current stream of the tensors' device and returns without waiting.  fp16, bf16 and fp32 tensors on a GPU; there is no CPU form.  The
functions take part in autograd (first derivatives, backward; a tensor that carries a forward-mode tangent is refused).  Tensors may be strided views: one whose last axis is not contiguous, or whose rows do
not start on 16 bytes where the operator needs that, is copied first.  The same call gives the same bits.

    y = layer_norm(x, weight, bias)
    o = cross_attention(q, k, v, kv_lens=lens)           # prompts of different lengths
    h = gated_ff(x, weight, bias, activation="gelu")     # GEGLU; "silu": SwiGLU

Calls can be captured into a graph.  A backward pass that is to be captured is taken with ``torch.autograd.grad`` of a forward pass in
the same capture: ``.backward()`` adds into ``.grad`` through nodes that belong to the stream on which the leaves were first used.  While a graph of
the same leaves that was built outside of the capture is alive, a call that would need their gradients, directly or through views and other steps of the capture, is
refused (RuntimeError); so is a captured backward pass that reaches a step taken outside of the capture.

They are registered with torch (``torch.ops.diffusers_amd``), so tracers record a call as one node; a saved trace is loaded in a process in
which one of them has been called.

A tensor of the wrong shape, device or value raises ValueError, of the wrong type TypeError; what the library itself refuses raises ``_lib.SdeError``.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib

__all__ = ["layer_norm", "gated_ff", "cross_attention"]

_ACTIVATIONS = {"gelu": 0, "gelu_tanh": 1, "silu": 2}
_bound = None


def _native():
    """The torch binding, bound to the library, once it is known that both use torch's HIP runtime (streams and tensors of one are unknown to another)."""
    global _bound
    if _bound is None:
        library = _lib.lib()
        try:
            from . import _torch_ops
        except ImportError as e:
            raise ImportError(f"{e}: build it with `python -c 'import __graft_entry__ as g; g.build()'` or `make -C diffusers_amd/csrc`") from e
        try:
            with open("/proc/self/maps") as f:
                runtimes = {line.split()[-1] for line in f if "libamdhip64" in line}
        except OSError:
            runtimes = set()
        if len(runtimes) > 1:
            raise RuntimeError("two HIP runtimes are loaded (" + ", ".join(sorted(runtimes)) + "): import torch before diffusers_amd's library is loaded")
        _torch_ops.bind({name: ctypes.cast(getattr(library, name), ctypes.c_void_p).value for name in _lib.SYMBOLS
                         if name.startswith(("sde_last_error", "sde_layer_norm", "sde_gated_ff", "sde_cross_attention"))}, _lib.SdeError)
        _bound = _torch_ops
    return _bound


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis.  weight and bias: [C], both of x's type or both fp32, either may be left
    out.  Statistics and sums are fp32.  Gradients for x, weight and bias."""
    return (_bound or _native()).layer_norm(x, weight, bias, eps)


def gated_ff(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "gelu") -> torch.Tensor:
    """(x Wv^T + bv) * act(x Wg^T + bg): both projections, the activation and the product in one kernel.  x [..., K]; weight [2F, K], the F value
    rows first, then the F gate rows; bias [2F] of x's type or fp32, or None; result [..., F].  activation: "gelu" (erf), "gelu_tanh" or
    "silu".  K and F are multiples of 8 (fp32: of 4).  Gradients for x, weight and bias; the backward pass forms the projections again."""
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation is one of {', '.join(_ACTIVATIONS)}, not {activation!r}")
    return (_bound or _native()).gated_ff(x, weight, bias, act)


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, q_lens: Optional[torch.Tensor] = None, kv_lens: Optional[torch.Tensor] = None,
                    key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """softmax(scale q k^T) v with keys and values of another length than the queries.  q [B, Sq, H, D]; k, v [B, Skv, Hkv, D], H a multiple of Hkv (shared
    heads); D at most 256 and a multiple of 8 (fp32: of 4); scale defaults to D ** -0.5.  q_lens, kv_lens: int32 [B] on the device, how many of the padded
    queries and keys count; key_mask: bool [B, Skv], true where a key counts.  What does not count is not read; a query that does not count, or that
    no key counts for, gives zeros.  Gradients for q, k and v."""
    return (_bound or _native()).cross_attention(q, k, v, q_lens, kv_lens, key_mask, scale)
