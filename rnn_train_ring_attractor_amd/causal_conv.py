"""Short causal convolution: every channel by itself over the last few tokens, what stands in front of a recurrence.

`causal_conv_func` takes whole sequences (training and prompts, differentiable with respect to its input, its parameters and the initial state),
`causal_conv_step` one token for each sequence of a batch (serving, the state moved on in place).  What the one leaves as its state the
other goes on from: the last K - 1 inputs, in their own type."""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import Function

from . import _lib
from ._lib import SEQUENCE_TYPES, check_sequence_sizes, check_sequence_tensor, checked_parameter, empty_of, pointer, resolved, rows_of

_Strides2, _Strides4 = ctypes.c_longlong * 2, ctypes.c_longlong * 4
_ACTIVATIONS = {None: 0, "silu": 1}


def _checked(x, weight, bias, activation, dims):
    check_sequence_tensor("x", x)
    if x.dim() != dims:
        raise ValueError(f"x must have {dims} dimensions, got {tuple(x.shape)}")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"Invalid activation '{activation}'. Must be one of {list(_ACTIVATIONS)}.")
    C, dev = x.shape[-1], x.device
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError(f"weight must be a tensor [channels, taps], got {tuple(weight.shape) if isinstance(weight, torch.Tensor) else type(weight).__name__}")
    K = weight.shape[1]
    if C == 0 or not 1 <= K <= 8:
        raise ValueError(f"channels must be positive and taps between 1 and 8, got {C}, {K}")
    check_sequence_sizes(x)
    return C, K, dev, checked_parameter("weight", weight, (C, K), dev), checked_parameter("bias", bias, (C,), dev)


def _forward(x, weight, bias, initial_state, lengths, act, want_state):
    B, T, C = x.shape
    K, dev = weight.shape[1], x.device
    with _lib.on_device(dev):
        y = empty_of(x)
        state = x.new_empty((B, K - 1, C)) if want_state else None
        if B == 0 or T == 0:
            if want_state:
                state.zero_() if initial_state is None else state.copy_(initial_state)
            return y, state
        _lib.check(_lib.load().ringattr_causal_conv_fwd(
            x.data_ptr(), _Strides2(*x.stride()[:2]), weight.data_ptr(), pointer(bias), pointer(initial_state), pointer(lengths), y.data_ptr(),
            pointer(state), act, SEQUENCE_TYPES[x.dtype], B, T, C, K, _lib.stream_handle(dev)))
    return y, state


class CausalConvFunc(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, initial_state, lengths, act, want_state):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, initial_state, lengths)
        ctx.act = act
        return _forward(x, weight, bias, initial_state, lengths, act, want_state)

    @staticmethod
    def backward(ctx, grad_y, grad_state):
        if torch.is_grad_enabled():              # (create_graph: the result would pass for one that does not depend on x and weight)
            raise RuntimeError("causal_conv_func is differentiable once: its backward takes no create_graph=True")
        if _lib.followed():
            _lib.refuse_followed("the backward of causal_conv_func", *(g for g in (grad_y, grad_state) if g is not None))
        x, weight, bias, initial_state, lengths = ctx.saved_tensors
        B, T, C = x.shape
        K, dev = weight.shape[1], x.device
        lib, kind = _lib.load(), SEQUENCE_TYPES[x.dtype]
        with _lib.on_device(dev):
            gx, gw, gb, g0 = (empty_of(t) if t is not None and needed else None
                              for t, needed in zip((x, weight, bias, initial_state), ctx.needs_input_grad))
            gs = None if grad_state is None else resolved(grad_state).contiguous()
            if B == 0 or T == 0:
                for g in (gw, gb):
                    if g is not None:
                        g.zero_()
                if g0 is not None:
                    g0.zero_() if gs is None else g0.copy_(gs)
            else:
                gy = x.new_zeros((1, 1, C)).expand(B, T, C) if grad_y is None else rows_of(grad_y)
                nbytes = lib.ringattr_causal_conv_bwd_workspace_bytes(kind, B, T, C, K, gw is not None or gb is not None)
                ws = weight.new_empty((nbytes // 4,)) if nbytes else None
                _lib.check(lib.ringattr_causal_conv_bwd(
                    x.data_ptr(), gy.data_ptr(), _Strides4(*x.stride()[:2], *gy.stride()[:2]), weight.data_ptr(), pointer(bias),
                    pointer(initial_state), pointer(lengths), pointer(gs), pointer(gx), pointer(gw), pointer(gb), pointer(g0), ctx.act, kind, B, T,
                    C, K, pointer(ws), nbytes, _lib.stream_handle(dev)))
        return gx, gw, gb, g0, None, None, None


def causal_conv_func(x, weight, bias=None, initial_state=None, lengths=None, activation=None, return_state=False):
    """y_t = act(bias + sum_k weight[:, k] x_(t - K + 1 + k)) over whole sequences, every channel by itself.

    x [B,T,C] float32, bfloat16 or float16; a token's channels lie next to each other, all other strides are free (a ring history's [T,B,..]
    order, a slice of one projection's output).  weight [C,K] with K up to 8 taps, bias [C] or None, both float32.  activation: None or
    "silu".  initial_state [B,K-1,C] in x's type or None (zeros): the inputs in front of the sequences.  lengths [B] int32 (int64
    is converted) or None: how many tokens of each sequence count, none among the possibilities; outputs and gradients behind them
    are zero, nothing there is read and the state is the one behind the last token that counts.

    Returns y [B,T,C], with return_state=True (y, the last K - 1 inputs that count).  Differentiable once with respect to x, weight, bias and
    initial_state."""
    C, K, dev, weight, bias = _checked(x, weight, bias, activation, 3)
    B, T = x.shape[:2]
    if initial_state is not None:
        check_sequence_tensor("initial_state", initial_state, (B, K - 1, C), x.dtype, dev)
        initial_state = resolved(initial_state).contiguous()
    lengths = _lib.checked_lengths(lengths, B, T, dev)
    args = (rows_of(x), weight, bias, initial_state, lengths, _ACTIVATIONS[activation], bool(return_state))
    y, state = CausalConvFunc.apply(*args) if _lib.followed() or _lib.wants_gradient(*args[:4]) else _forward(*args)
    return (y, state) if return_state else y


def causal_conv_step(x, weight, state, bias=None, active=None, activation=None):
    """One token for each sequence: x [B,C], weight, bias and activation as in `causal_conv_func`; state [B,K-1,C] in x's type, contiguous, is
    moved on in place.  active [B] (bool or uint8) or None: where it is zero the state stays as it is and the output is zero (a batch with
    places that wait).  Returns y [B,C].  It has no gradient."""
    C, K, dev, weight, bias = _checked(x, weight, bias, activation, 2)
    B = x.shape[0]
    check_sequence_tensor("state", state, (B, K - 1, C), x.dtype, dev)
    if not state.is_contiguous() or state.is_neg():
        raise RuntimeError("state must be contiguous and no negated view: it is updated in place")
    if _lib.wants_gradient(x, weight, bias, state):
        raise RuntimeError("causal_conv_step has no gradient: call it under torch.no_grad(), or causal_conv_func to train")
    if _lib.followed():
        _lib.refuse_followed("causal_conv_step", x, weight, state, *(() if bias is None else (bias,)))
    active = _lib.checked_active(active, B, dev)
    x = rows_of(x)
    with _lib.on_device(dev):
        y = x.new_empty((B, C))
        if B == 0:
            return y
        _lib.check(_lib.load().ringattr_causal_conv_step(
            x.data_ptr(), x.stride(0), weight.data_ptr(), pointer(bias), state.data_ptr(), pointer(active), y.data_ptr(),
            _ACTIVATIONS[activation], SEQUENCE_TYPES[x.dtype], B, C, K, _lib.stream_handle(dev)))
    torch.autograd.graph.increment_version(state)
    return y
