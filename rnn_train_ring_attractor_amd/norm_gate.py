"""What stands around a block: its output normalised, gated and added to the residual stream, and the next block's norm of that, in one pass."""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import Function

from . import _lib
from ._lib import SEQUENCE_TYPES, check_sequence_tensor, checked_parameter, empty_of, pointer

_Strides3, _Strides5 = ctypes.c_longlong * 3, ctypes.c_longlong * 5
_KINDS = {"rms": 0, "layer": 1}
_ACTIVATIONS = {None: 0, "silu": 1, "sigmoid": 2}


def _flat(t):
    """(t as rows at one stride, a row's values next to each other, copied where it is not; the stride)"""
    if t is None:
        return None, 0
    if not t.is_contiguous() or t.is_neg():
        t = _lib.rows_of(_lib.resolved(t).reshape(-1, t.shape[-1]))
        return t, t.stride(0)
    return t, t.shape[-1]


def _forward(x, weight, gate, residual, scale, next_weight, group, eps, kind, act):
    C, dev = x.shape[-1], x.device
    with _lib.on_device(dev):
        y = empty_of(x)
        n = empty_of(x) if next_weight is not None else None
        if x.numel() == 0:
            return y, n
        (fx, sx), (fg, sg), (fr, sr) = _flat(x), _flat(gate), _flat(residual)
        _lib.check(_lib.load().ringattr_norm_gate_fwd(
            fx.data_ptr(), pointer(fg), pointer(fr), _Strides3(sx, sg, sr), weight.data_ptr(), pointer(scale), pointer(next_weight), y.data_ptr(),
            pointer(n), eps, kind, act, SEQUENCE_TYPES[x.dtype], x.numel() // C, C, group, _lib.stream_handle(dev)))
    return y, n


class NormGateFunc(Function):
    @staticmethod
    def forward(ctx, x, weight, gate, residual, scale, next_weight, group, eps, kind, act):
        ctx.set_materialize_grads(False)
        # (the residual is read again for the next norm only: y is found from it unrounded)
        ctx.save_for_backward(x, weight, gate, residual if next_weight is not None else None, scale, next_weight)
        ctx.how = (group, eps, kind, act)
        return _forward(x, weight, gate, residual, scale, next_weight, group, eps, kind, act)

    @staticmethod
    def backward(ctx, grad_y, grad_n):
        if torch.is_grad_enabled():              # (create_graph: the result would pass for one that does not depend on x)
            raise RuntimeError("norm_gate_func is differentiable once: its backward takes no create_graph=True")
        if _lib.followed():
            _lib.refuse_followed("the backward of norm_gate_func", *(g for g in (grad_y, grad_n) if g is not None))
        x, weight, gate, residual, scale, next_weight = ctx.saved_tensors
        group, eps, kind, act = ctx.how
        C, dev, need = x.shape[-1], x.device, ctx.needs_input_grad
        lib, code = _lib.load(), SEQUENCE_TYPES[x.dtype]
        with _lib.on_device(dev):
            gx, gw, gg, gs, gn = (empty_of(t) if t is not None and n else None
                                  for t, n in zip((x, weight, gate, scale, next_weight), (*need[:3], *need[4:6])))
            gr = empty_of(x) if need[3] else None
            if grad_n is None and gn is not None:
                gn.zero_()
            if x.numel() == 0 or (grad_y is None and grad_n is None):
                for g in (gx, gw, gg, gr, gs, gn):
                    if g is not None:
                        g.zero_()
            elif any(need):
                rows, (fx, sx), (fg, sg), (fr, sr), (fy, sy), (fn, sn) = x.numel() // C, *(_flat(t) for t in (x, gate, residual, grad_y, grad_n))
                asked = gn if grad_n is not None else None
                nbytes = lib.ringattr_norm_gate_bwd_workspace_bytes(code, rows, C, group, any(g is not None for g in (gw, gs, asked)))
                ws = weight.new_empty((nbytes // 4,)) if nbytes else None
                _lib.check(lib.ringattr_norm_gate_bwd(
                    fx.data_ptr(), pointer(fg), pointer(fr), pointer(fy), pointer(fn),
                    _Strides5(sx, sg, sr, sy, sn), weight.data_ptr(), pointer(scale), pointer(next_weight), pointer(gx), pointer(gg), pointer(gr),
                    pointer(gw), pointer(gs), pointer(asked), eps, kind, act, code, rows, C, group, pointer(ws), nbytes, _lib.stream_handle(dev)))
        return gx, gw, gg, gr, gs, gn, None, None, None, None


def norm_gate_func(x, weight, gate=None, residual=None, scale=None, next_weight=None, group=None, eps=1e-5, kind="rms", activation="silu"):
    """y = residual + scale norm(x) weight act(gate), and with next_weight also norm(y) next_weight over whole rows: the norm behind a block, its
    gate, the scaled sum with the residual stream and the norm in front of the next block.

    x [..,C], C up to 8192; gate and residual (None: left out) of x's shape and type, float32, bfloat16 or float16, any strides.  weight, scale
    and next_weight [C] float32 (the last two may be None).  group: how many neighbouring channels the first norm spans, a divisor of C (a head's
    width; None: all).  kind "rms" divides by the root of the mean square plus eps, "layer" takes the mean away before.  activation of the
    gate: "silu", "sigmoid" or None.  The next norm is of y before its rounding.

    Returns y, with next_weight (y, norm of y).  Differentiable once with respect to all tensors."""
    check_sequence_tensor("x", x)
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    if kind not in _KINDS:
        raise ValueError(f"Invalid kind '{kind}'. Must be one of {list(_KINDS)}.")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"Invalid activation '{activation}'. Must be one of {list(_ACTIVATIONS)}.")
    C, dev, eps = x.shape[-1], x.device, float(eps)
    group = C if group is None else int(group)
    if not 1 <= C <= 8192 or group < 1 or C % group:
        raise ValueError(f"channels must be between 1 and 8192 and a multiple of group, got {C}, {group}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    for name, t in (("gate", gate), ("residual", residual)):
        if t is not None:
            check_sequence_tensor(name, t, x.shape, x.dtype, dev)
    args = (x, checked_parameter("weight", weight, (C,), dev), gate, residual, checked_parameter("scale", scale, (C,), dev),
            checked_parameter("next_weight", next_weight, (C,), dev), group, eps, _KINDS[kind], _ACTIVATIONS[activation])
    if weight is None:
        raise TypeError("weight must be a torch.Tensor, got NoneType")
    y, n = NormGateFunc.apply(*args) if _lib.followed() or _lib.wants_gradient(*args[:6]) else _forward(*args)
    return y if next_weight is None else (y, n)
