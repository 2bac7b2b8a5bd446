"""CPU: the operators' C entries refuse arguments that are not met, before anything touches a device, and say how much scratch they need."""
import ctypes as C

import pytest
import torch

from diffusers_amd import _lib, ops

P = 4096            # stands for a pointer: aligned, never read


def ln(**kw):
    a = dict(dtype=0, param_dtype=0, rows=4, C=64, ld_x=64, ld_y=64, ld_dy=64, ld_dx=64, eps=1e-5, x=P, gamma=P, beta=P, y=P, mean=P, rstd=P, dy=P, dx=P,
             dgamma=P, dbeta=P)
    return _lib.LayerNormArgs(**{**a, **kw})


def ff(**kw):
    a = dict(dtype=1, bias_dtype=1, activation=0, M=5, K=64, F=96, ld_x=64, ld_w=64, ld_h=96, ld_dh=96, ld_dx=64, ld_dw=64, x=P, weight=P, bias=P, h=P, dh=P,
             dx=P, dweight=P, dbias=P)
    return _lib.GatedFfArgs(**{**a, **kw})


def xa(**kw):
    a = dict(dtype=1, B=2, Sq=3, Skv=7, H=4, Hkv=2, D=64, scale=0.125, q=P, k=P, v=P, o=P, lse=P, d_o=P, dq=P, dk=P, dv=P, key_mask_stride=7)
    for n in ("q", "o", "do", "dq"):
        a[n + "_stride"] = (3 * 256, 256, 64)
    for n in ("k", "v", "dk", "dv"):
        a[n + "_stride"] = (7 * 128, 128, 64)
    return _lib.CrossAttentionArgs(**{**a, **kw})


def refused(fn, args, word, exec_=None):
    e = exec_ if exec_ is not None else _lib.OpExec(0, None, 1 << 20, 1 << 40)
    assert fn(args, e) == 1, "not refused"                # SDE_ERR_INVALID_ARGUMENT
    message = _lib.lib().sde_last_error().decode()
    assert word in message, message


L = _lib.lib()
LN_BOTH = [({"dtype": 3}, "dtype"), ({"param_dtype": 1}, "param_dtype"), ({"rows": -1}, "rows"), ({"C": 0}, "C must"), ({"C": 1 << 25}, "C must"),
           ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"), ({"ld_x": 63}, "ld_x"), ({"x": None}, "x")]


@pytest.mark.parametrize("change,word", LN_BOTH + [({"ld_y": 63}, "ld_y"), ({"y": None}, "null"), ({"mean": None}, "go together")])
def test_layer_norm_forward_refuses(change, word):
    refused(L.sde_layer_norm_forward, ln(**change), word)


@pytest.mark.parametrize("change,word", LN_BOTH + [({"ld_dy": 1}, "ld_dy"), ({"ld_dx": 0}, "ld_dx"), ({"dy": None}, "dy"), ({"rstd": None}, "rstd"),
                                                   ({"dx": None, "dgamma": None, "dbeta": None}, "no gradient")])
def test_layer_norm_backward_refuses(change, word):
    refused(L.sde_layer_norm_backward, ln(**change), word)


FF_BOTH = [({"dtype": -1}, "dtype"), ({"bias_dtype": 0}, "bias_dtype"), ({"activation": 3}, "activation"), ({"M": -1}, "M"), ({"K": 60}, "K must"), ({"K": 0}, "K must"),
           ({"F": 100}, "F must"), ({"x": None}, "x"), ({"x": P + 8}, "x"), ({"ld_x": 56}, "x"), ({"ld_x": 68}, "x"), ({"weight": None}, "weight"),
           ({"ld_w": 1 << 22}, "weight"), ({"M": (1 << 31) - 1, "F": 1 << 20}, "too large")]


@pytest.mark.parametrize("change,word", FF_BOTH + [({"h": None}, "h is"), ({"ld_h": 95}, "h is")])
def test_gated_ff_forward_refuses(change, word):
    refused(L.sde_gated_ff_forward, ff(**change), word)


@pytest.mark.parametrize("change,word", FF_BOTH + [({"dh": None}, "dh"), ({"ld_dh": 8}, "dh"), ({"ld_dx": 8}, "dx"), ({"ld_dw": 8}, "dweight"),
                                                   ({"dx": None, "dweight": None, "dbias": None}, "no gradient")])
def test_gated_ff_backward_refuses(change, word):
    refused(L.sde_gated_ff_backward, ff(**change), word)


XA_BOTH = [({"dtype": 7}, "dtype"), ({"H": 3}, "multiple of Hkv"), ({"Hkv": 0}, "multiple of Hkv"), ({"D": 60}, "D must"), ({"D": 264}, "D must"), ({"D": 0}, "D must"),
           ({"scale": 0.0}, "scale"), ({"scale": float("inf")}, "scale"), ({"B": -1}, "bad B"), ({"Skv": 1 << 31}, "bad B"), ({"q": None}, "q is"), ({"k": P + 2}, "k is"),
           ({"v_stride": (896, 130, 64)}, "v is"), ({"k_stride": (-8, 128, 64)}, "k is"), ({"q_stride": (8, 1 << 26, 8)}, "q is"),
           ({"key_mask": P, "key_mask_stride": 6}, "key_mask_stride"), ({"B": 1 << 24, "Hkv": 4}, "too large")]


@pytest.mark.parametrize("change,word", XA_BOTH + [({"o": None}, "o is"), ({"o_stride": (0, 256, 64)}, "overlap"), ({"o_stride": (768, 256, 32)}, "overlap")])
def test_cross_attention_forward_refuses(change, word):
    refused(L.sde_cross_attention_forward, xa(**change), word)


@pytest.mark.parametrize("change,word", XA_BOTH + [({"lse": None}, "lse"), ({"d_o": None}, "d_o"), ({"dk_stride": (0, 128, 64)}, "overlap"), ({"dv_stride": (896, 120, 64)}, "overlap"),
                                                   ({"dq": None, "dk": None, "dv": None}, "no gradient")])
def test_cross_attention_backward_refuses(change, word):
    refused(L.sde_cross_attention_backward, xa(**change), word)


@pytest.mark.parametrize("fn,args", [(L.sde_layer_norm_forward, ln), (L.sde_gated_ff_forward, ff), (L.sde_cross_attention_forward, xa)])
def test_null_arguments_are_refused(fn, args):
    assert fn(None, _lib.OpExec()) == 1 and b"null" in L.sde_last_error()
    assert fn(args(), None) == 1 and b"exec" in L.sde_last_error()
    refused(fn, args(), "device_id", _lib.OpExec(-1, None, None, 0))


@pytest.mark.parametrize("backward,query,args,extra", [(L.sde_layer_norm_backward, L.sde_layer_norm_workspace, ln, ()),
                                                       (L.sde_gated_ff_backward, L.sde_gated_ff_workspace, ff, (1,)),
                                                       (L.sde_cross_attention_backward, L.sde_cross_attention_workspace, xa, (1,))])
def test_scratch_has_to_be_there(backward, query, args, extra):
    n = C.c_size_t()
    assert query(args(), *extra, n) == 0 and n.value > 0
    refused(backward, args(), "workspace", _lib.OpExec(0, None, None, 0))
    refused(backward, args(), "workspace", _lib.OpExec(0, None, P, n.value - 1))
    refused(backward, args(), "aligned", _lib.OpExec(0, None, P + 128, n.value))
    assert query(args(), *extra, None) == 1
    assert query(None, *extra, n) == 1


def test_python_entries_refuse_tensors_that_are_not_on_a_gpu():
    x = torch.zeros(4, 64)
    for call in (lambda: ops.layer_norm(x), lambda: ops.gated_ff(x, torch.zeros(32, 64)), lambda: ops.cross_attention(x[None, None], x[None, None], x[None, None])):
        with pytest.raises(ValueError, match="GPU"):
            call()
