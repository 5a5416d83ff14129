"""Rotary positions: the pairs of a head's values turned by their position, for queries and keys in one launch.

A position is a token's number, however far, or an angle of its own: with whole frequencies 1, 2, 3, ... and a heading as position (the
angle that the ring integrates), two rows' product depends on the difference of their headings."""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd import Function

from . import _lib
from ._lib import SEQUENCE_TYPES, check_sequence_sizes, check_sequence_tensor, resolved

_POSITION_TYPES = {torch.int64: 0, torch.int32: 1, torch.float32: 2}
_LAYOUTS = {"half": 0, "interleaved": 1}


def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, original_length=None, fast=32.0, slow=1.0, device="cuda"):
    """(frequencies float64 [rotary_dim / 2] in radians per position, scale) for `rotary_func`: f_m = base ** (-2 m / rotary_dim).

    scaling, for contexts `factor` times as long as the one trained on:
      None      as they are
      "linear"  f_m / factor (positions are interpolated)
      "base"    the base grows to base * factor ** (d / (d - 2)): the fastest pair keeps its frequency, the slowest is divided by factor
      "ramp"    pairs that turn more than `fast` times within original_length keep their frequency, those that turn less than `slow`
                times are divided by factor, those between are mixed linearly over m; scale 0.1 ln(factor) + 1"""
    d = int(rotary_dim)
    if d < 2 or d % 2:
        raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
    if not base > 1.0 or not factor >= 1.0:
        raise ValueError(f"base must be greater than 1 and factor at least 1, got {base}, {factor}")
    m = torch.arange(d // 2, dtype=torch.float64)
    scale = 1.0
    if scaling == "base":
        if d == 2:
            raise ValueError("scaling the base needs at least two pairs (rotary_dim 4)")
        base = base * factor ** (d / (d - 2))
    f = float(base) ** (-2.0 * m / d)
    if scaling == "linear":
        f = f / factor
    elif scaling == "ramp":
        if original_length is None or original_length < 1 or not fast > slow > 0:
            raise ValueError("the ramp needs original_length >= 1 and fast > slow > 0")
        # the pair that turns x times within the original length
        pair = lambda x: d * math.log(original_length / (2 * math.pi * x)) / (2 * math.log(base))
        lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), d - 1)
        mix = ((m - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        f = f * (1.0 - mix) + f / factor * mix
        scale = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "base"):
        raise ValueError(f"Invalid scaling '{scaling}'. Must be None, 'linear', 'base' or 'ramp'.")
    return f.to(device), scale


def _turn(xs, positions, frequencies, layout, scale, inverse):
    B, T, _, D = xs[0].shape
    dev = xs[0].device
    xs = [resolved(x) for x in xs]
    xs = [x if x.shape[-1] == 1 or x.stride(-1) == 1 else x.contiguous() for x in xs]
    lib = _lib.load()
    with _lib.on_device(dev):
        ys = [x.new_empty(x.shape) for x in xs]
        if B == 0 or T == 0:
            return ys
        strides = [s for x in xs for s in x.stride()[:3]]
        two = len(xs) == 2
        per_b, per_t = positions.stride() if positions.dim() == 2 else (0, positions.stride(0))
        _lib.check(lib.ringattr_rotary(
            xs[0].data_ptr(), xs[1].data_ptr() if two else None, (ctypes.c_longlong * len(strides))(*strides), positions.data_ptr(), per_b,
            per_t, _POSITION_TYPES[positions.dtype], frequencies.data_ptr(), ys[0].data_ptr(), ys[1].data_ptr() if two else None, scale,
            layout, inverse, SEQUENCE_TYPES[xs[0].dtype], B, T, xs[0].shape[2], xs[1].shape[2] if two else 0, D, 2 * frequencies.numel(),
            _lib.stream_handle(dev)))
    return ys


def _turned(positions, frequencies, layout, scale, inverse, *xs):
    return tuple(_turn(xs, positions, frequencies, layout, scale, inverse))


class RotaryFunc(Function):
    @staticmethod
    def forward(ctx, positions, frequencies, layout, scale, inverse, *xs):
        ctx.save_for_backward(positions, frequencies)
        ctx.how = (layout, scale, inverse)
        return _turned(positions, frequencies, layout, scale, inverse, *xs)

    @staticmethod
    def backward(ctx, *grads):
        positions, frequencies = ctx.saved_tensors
        layout, scale, inverse = ctx.how
        # turned back: the transpose of a turn is the opposite turn, so a gradient of the gradient is this operator again
        back = RotaryFunc.apply if torch.is_grad_enabled() or _lib.followed() else _turned
        needed = ctx.needs_input_grad[5:]
        turned = iter(back(positions, frequencies, layout, scale, 1 - inverse, *(g for g, n in zip(grads, needed) if n)))
        return (None,) * 5 + tuple(next(turned) if n else None for n in needed)


def rotary_func(x, positions, frequencies, layout="half", scale=1.0):
    """x [B,T,H,D], or a pair (q, k) of such tensors with the same B, T, D and type and heads of their own, turned: pair m of the first
    2 * len(frequencies) values of each head, (m, m + len(frequencies)) in layout "half" or (2m, 2m + 1) in layout "interleaved", by the
    angle position * frequencies[m] and multiplied by `scale`; the rest of a head is copied.

    positions [T] or [B,T], int64, int32 or float32 (an angle); frequencies float64 (`rotary_frequencies`).  The angle, less whole turns, is
    that of the exact product for every int64 position (of frequencies up to 1000: to 2^-24 turns).  Differentiable with respect to x.
    Returns a tensor, or a tuple where x is a pair."""
    pair = isinstance(x, (tuple, list))
    xs = tuple(x) if pair else (x,)
    if len(xs) not in (1, 2):
        raise ValueError(f"x must be a tensor or a pair of tensors, got {len(xs)}")
    if layout not in _LAYOUTS:
        raise ValueError(f"Invalid layout '{layout}'. Must be one of {list(_LAYOUTS)}.")
    check_sequence_tensor("x", xs[0])
    if xs[0].dim() != 4:
        raise ValueError(f"x must be [B, T, H, D], got {tuple(xs[0].shape)}")
    B, T, H, D = xs[0].shape
    dev = xs[0].device
    if len(xs) == 2:
        check_sequence_tensor("x", xs[1], dtype=xs[0].dtype, device=dev)
        if xs[1].dim() != 4 or tuple(xs[1].shape[:2]) != (B, T) or xs[1].shape[3] != D:
            raise ValueError(f"x must be two tensors of [B, T, heads, D], got {tuple(xs[0].shape)} and {tuple(xs[1].shape)}")
    if any(t.shape[2] == 0 for t in xs):
        raise ValueError("x must have at least one head")
    check_sequence_sizes(*xs)
    if not isinstance(positions, torch.Tensor) or positions.dtype not in _POSITION_TYPES:
        raise TypeError("positions must be an int64, int32 or float32 tensor")
    if tuple(positions.shape) not in ((T,), (B, T)):
        raise ValueError(f"positions must have shape ({T},) or ({B}, {T}), got {tuple(positions.shape)}")
    if positions.device != dev:
        raise RuntimeError(f"positions must be on {dev} (got {positions.device})")
    if positions.requires_grad and torch.is_grad_enabled():
        raise ValueError("positions get no gradient (detach them)")
    check_sequence_tensor("frequencies", frequencies, dtype=torch.float64, device=dev)
    if frequencies.requires_grad and torch.is_grad_enabled():
        raise ValueError("frequencies get no gradient (detach them)")
    if frequencies.dim() != 1 or not 1 <= frequencies.numel() <= D // 2:
        raise ValueError(f"frequencies must be one-dimensional, between 1 and {D // 2} of them, got {tuple(frequencies.shape)}")
    positions, frequencies, scale = resolved(positions), resolved(frequencies).contiguous(), float(scale)
    if _lib.followed() or (torch.is_grad_enabled() and any(t.requires_grad for t in xs)):
        ys = RotaryFunc.apply(positions, frequencies, _LAYOUTS[layout], scale, 0, *xs)
    else:
        ys = _turned(positions, frequencies, _LAYOUTS[layout], scale, 0, *xs)
    return ys if pair else ys[0]
