"""Dropout whose mask is a function of a seed, an offset and an element's index, and is never stored: the backward forms it again."""
from __future__ import annotations

import torch
from torch.autograd import Function

from . import _lib
from ._lib import SEQUENCE_TYPES, check_sequence_tensor, resolved


def _drop(x, residual, p, seed, offset, counter):
    x = resolved(x).contiguous()
    residual = None if residual is None else resolved(residual).contiguous()
    y = torch.empty_like(x)
    if x.numel() == 0:
        return y
    with _lib.on_device(x.device):
        _lib.check(_lib.load().ringattr_dropout(
            x.data_ptr(), None if residual is None else residual.data_ptr(), y.data_ptr(), x.numel(), int(p * 2.0 ** 32), 1.0 / (1.0 - p),
            seed, offset, None if counter is None else counter.data_ptr(), SEQUENCE_TYPES[x.dtype], _lib.stream_handle(x.device)))
    return y


class DropoutFunc(Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset, counter):
        ctx.save_for_backward(counter)          # (a counter that was advanced in between is an error, not another mask)
        ctx.how = (p, seed, offset)
        return _drop(x, residual, p, seed, offset, counter)

    @staticmethod
    def backward(ctx, grad):
        counter, = ctx.saved_tensors
        p, seed, offset = ctx.how
        again = DropoutFunc.apply if torch.is_grad_enabled() or _lib.followed() else _drop          # (a gradient of the gradient is this operator again)
        gx = again(grad, None, p, seed, offset, counter) if ctx.needs_input_grad[0] else None
        return gx, grad if ctx.needs_input_grad[1] else None, None, None, None, None


def dropout_func(x, p, seed, offset=0, residual=None):
    """residual + dropout(x), or dropout(x) without one: an element is dropped with probability p (0 <= p < 1), otherwise multiplied by
    1 / (1 - p).  Which ones is a function of seed, offset and the element's index in row-major order: word i % 4 of block i // 4 of
    Philox (four words, seven rounds; counter: block and offset, key: seed) below floor(p 2^32) drops element i.

    x and residual: any shape, the same for both, float32, bfloat16 or float16.  seed and offset: whole numbers of 64 bits; a program
    gives every call of a step an offset of its own.  offset may be an int64 GPU tensor of one element, which is read when the kernel
    runs: a step recorded into a HIP graph advances it itself, behind its backward.  Differentiable with respect to x and residual."""
    check_sequence_tensor("x", x)
    if residual is not None:
        check_sequence_tensor("residual", residual, x.shape, x.dtype, x.device)
    p = float(p)
    if not 0.0 <= p < 1.0:
        raise ValueError(f"p must lie in [0, 1), got {p}")
    counter = None
    if isinstance(offset, torch.Tensor):
        if offset.dtype != torch.int64 or offset.numel() != 1 or offset.device != x.device:
            raise ValueError(f"an offset tensor must be one int64 element on {x.device}, got {offset.dtype} {tuple(offset.shape)} on {offset.device}")
        counter, offset = offset, 0
    seed, offset = int(seed), int(offset)
    if not (0 <= seed < 1 << 64 and 0 <= offset < 1 << 64):
        raise ValueError("seed and offset must be whole numbers from 0 to 2^64 - 1")
    if _lib.followed() or (torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad))):
        return DropoutFunc.apply(x, residual, p, seed, offset, counter)
    return _drop(x, residual, p, seed, offset, counter)
