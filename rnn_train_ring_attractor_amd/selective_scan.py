"""Selective state space scan: a leak on a few states of every channel whose rate, input and output the token itself decides.

    d_t = softplus(delta_t + delta_bias),  h_t[n] = exp(d_t A[n]) h_(t-1)[n] + d_t x_t B_t[n],  y_t = (sum_n C_t[n] h_t[n] + D x_t) silu(z_t)

`selective_scan_func` takes whole sequences (training and prompts, differentiable with respect to everything but the lengths), `selective_scan_step` one token
for each sequence of a batch (serving, the state updated in place).  What the one leaves as its state the other goes on from.

The rows are float32, bfloat16 or float16, parameters and states float32; all sums are float32, results are rounded once."""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import Function

from . import _lib
from ._lib import SEQUENCE_TYPES, check_sequence_sizes, check_sequence_tensor, checked_parameter, empty_of, pointer, resolved, rows_of

_Strides12, _Strides14, _Strides7 = ctypes.c_longlong * 12, ctypes.c_longlong * 14, ctypes.c_longlong * 7


def _checked(x, delta, A, B, C, D, z, delta_bias, dims):
    check_sequence_tensor("x", x)
    if x.dim() != dims:
        raise ValueError(f"x must have {dims} dimensions, got {tuple(x.shape)}")
    dev, lead, channels = x.device, tuple(x.shape[:-1]), x.shape[-1]
    check_sequence_tensor("delta", delta, x.shape, x.dtype, dev)
    if z is not None:
        check_sequence_tensor("z", z, x.shape, x.dtype, dev)
    if not isinstance(A, torch.Tensor) or A.dim() != 2:
        raise ValueError(f"A must be a tensor [channels, states], got {tuple(A.shape) if isinstance(A, torch.Tensor) else type(A).__name__}")
    N = A.shape[1]
    check_sequence_tensor("B", B, dtype=x.dtype, device=dev)
    if B.dim() != dims + 1 or tuple(B.shape[:-2]) != lead or B.shape[-1] != N:
        raise ValueError(f"B must have shape {lead + ('groups', N)}, got {tuple(B.shape)}")
    check_sequence_tensor("C", C, B.shape, x.dtype, dev)
    G = B.shape[-2]
    if channels == 0 or G == 0 or channels % G != 0 or not 1 <= N <= 64:
        raise ValueError(f"channels ({channels}) must be a positive multiple of groups ({G}), states between 1 and 64 ({N})")
    check_sequence_sizes(x, B)
    return N, G, dev, checked_parameter("A", A, (channels, N), dev), checked_parameter("D", D, (channels,), dev), checked_parameter(
        "delta_bias", delta_bias, (channels,), dev)


def _strides(x, delta, z, B, C):
    return (*x.stride()[:2], *delta.stride()[:2], *((0, 0) if z is None else z.stride()[:2]), *B.stride()[:3], *C.stride()[:3])


def _forward(x, delta, A, B, C, D, z, delta_bias, initial_state, lengths, softplus, want_state, keep):
    batch, T, channels = x.shape
    N, G, dev = A.shape[1], B.shape[2], x.device
    lib, sizes = _lib.load(), (SEQUENCE_TYPES[x.dtype], batch, T, channels, N, G)
    with _lib.on_device(dev):
        y = empty_of(x)
        state = A.new_empty((batch, channels, N)) if want_state else None
        if batch == 0 or T == 0:
            if want_state:
                state.zero_() if initial_state is None else state.copy_(initial_state)
            return y, state, None
        nbytes = lib.ringattr_selective_scan_fwd_workspace_bytes(*sizes)
        ws = A.new_empty((nbytes // 4,)) if nbytes else None
        along = A.new_empty((lib.ringattr_selective_scan_states_bytes(*sizes) // 4,)) if keep else None
        _lib.check(lib.ringattr_selective_scan_fwd(
            x.data_ptr(), delta.data_ptr(), pointer(z), B.data_ptr(), C.data_ptr(), _Strides12(*_strides(x, delta, z, B, C)), A.data_ptr(), pointer(D),
            pointer(delta_bias), pointer(initial_state), pointer(lengths), y.data_ptr(), pointer(state), pointer(along), softplus, *sizes,
            pointer(ws), nbytes, _lib.stream_handle(dev)))
    return y, state, along


class SelectiveScanFunc(Function):
    @staticmethod
    def forward(ctx, x, delta, A, B, C, D, z, delta_bias, initial_state, lengths, softplus, want_state):
        ctx.set_materialize_grads(False)
        y, state, along = _forward(x, delta, A, B, C, D, z, delta_bias, initial_state, lengths, softplus, want_state, True)
        ctx.save_for_backward(x, delta, A, B, C, D, z, delta_bias, lengths, along)
        ctx.softplus, ctx.start = softplus, None if initial_state is None else initial_state.shape
        return y, state

    @staticmethod
    def backward(ctx, grad_y, grad_state):
        if torch.is_grad_enabled():              # (create_graph: the result would pass for one that does not depend on the inputs)
            raise RuntimeError("selective_scan_func is differentiable once: its backward takes no create_graph=True")
        if _lib.followed():
            _lib.refuse_followed("the backward of selective_scan_func", *(g for g in (grad_y, grad_state) if g is not None))
        x, delta, A, B, C, D, z, delta_bias, lengths, along = ctx.saved_tensors
        batch, T, channels = x.shape
        lib, dev, sizes = _lib.load(), x.device, (SEQUENCE_TYPES[x.dtype], batch, T, channels, A.shape[1], B.shape[2])
        need = ctx.needs_input_grad
        with _lib.on_device(dev):
            gx, gd, gA, gB, gC, gD, gz, gb = (empty_of(t) if t is not None and n else None
                                              for t, n in zip((x, delta, A, B, C, D, z, delta_bias), need))
            g0 = A.new_empty(ctx.start) if ctx.start is not None and need[8] else None
            gs = None if grad_state is None else resolved(grad_state).contiguous()
            if batch == 0 or T == 0:
                for g in (gA, gD, gb):
                    if g is not None:
                        g.zero_()
                if g0 is not None:
                    g0.zero_() if gs is None else g0.copy_(gs)
            else:
                gy = x.new_zeros((1, 1, channels)).expand(batch, T, channels) if grad_y is None else rows_of(grad_y)
                nbytes = lib.ringattr_selective_scan_bwd_workspace_bytes(*sizes, gB is not None or gC is not None,
                                                                         any(g is not None for g in (gA, gD, gb)))
                ws = A.new_empty((nbytes // 4,)) if nbytes else None
                _lib.check(lib.ringattr_selective_scan_bwd(
                    x.data_ptr(), delta.data_ptr(), pointer(z), B.data_ptr(), C.data_ptr(), gy.data_ptr(),
                    _Strides14(*_strides(x, delta, z, B, C), *gy.stride()[:2]), A.data_ptr(), pointer(D), pointer(delta_bias), pointer(lengths),
                    along.data_ptr(), pointer(gs), pointer(gx), pointer(gd), pointer(gz), pointer(gB), pointer(gC), pointer(gA), pointer(gD),
                    pointer(gb), pointer(g0), ctx.softplus, *sizes, pointer(ws), nbytes, _lib.stream_handle(dev)))
        return gx, gd, gA, gB, gC, gD, gz, gb, g0, None, None, None


def selective_scan_func(x, delta, A, B, C, D=None, z=None, delta_bias=None, initial_state=None, lengths=None, softplus=False, return_state=False):
    """Selective state space scan over whole sequences (the formula is at the head of this module).

    x, delta and z (None: no gate) [B,T,channels], B and C [B,T,groups,states], of one type, float32, bfloat16 or float16; groups divide the channels
    (channel c uses group c // (channels // groups)), up to 64 states; a token's channels, and a group's states, lie next to each other, all other
    strides are free.  A [channels,states], D and delta_bias [channels] (or None) float32; A is finite, negative for states that fade.
    softplus=False takes delta + delta_bias as the step itself.  initial_state [B,channels,states] float32 or None (zeros).  lengths [B] int32
    (int64 is converted) or None: how many tokens of each sequence count, none among the possibilities; outputs and gradients behind
    them are zero, nothing there is read and the state is the one behind the last token that counts.

    Returns y [B,T,channels], with return_state=True (y, the state behind the sequences).  Differentiable once with respect to all tensors but the
    lengths; a forward that will be differentiated keeps the state in front of every sixteenth token (states rounded up to 4, 8, 16, 32 or 64)."""
    N, _, dev, A, D, delta_bias = _checked(x, delta, A, B, C, D, z, delta_bias, 3)
    batch, T, channels = x.shape
    if initial_state is not None:
        check_sequence_tensor("initial_state", initial_state, (batch, channels, N), torch.float32, dev)
        initial_state = resolved(initial_state).contiguous()
    lengths = _lib.checked_lengths(lengths, batch, T, dev)
    args = (rows_of(x), rows_of(delta), A, rows_of(B), rows_of(C), D, None if z is None else rows_of(z), delta_bias, initial_state, lengths,
            int(bool(softplus)), bool(return_state))
    if _lib.followed() or _lib.wants_gradient(*args[:9]):
        y, state = SelectiveScanFunc.apply(*args)
    else:
        y, state, _ = _forward(*args, False)
    return (y, state) if return_state else y


def selective_scan_step(x, delta, A, B, C, state, D=None, z=None, delta_bias=None, active=None, softplus=False):
    """One token for each sequence: x, delta, z [B,channels], B and C [B,groups,states] and the parameters as in `selective_scan_func`; state
    [B,channels,states] float32, contiguous, is updated in place.  active [B] (bool or uint8) or None: where it is zero the state stays as it is
    and the output is zero (a batch with places that wait).  Returns y [B,channels].  It has no gradient."""
    N, G, dev, A, D, delta_bias = _checked(x, delta, A, B, C, D, z, delta_bias, 2)
    batch, channels = x.shape
    check_sequence_tensor("state", state, (batch, channels, N), torch.float32, dev)
    if not state.is_contiguous() or state.is_neg():
        raise RuntimeError("state must be contiguous and no negated view: it is updated in place")
    if _lib.wants_gradient(x, delta, A, B, C, D, z, delta_bias, state):
        raise RuntimeError("selective_scan_step has no gradient: call it under torch.no_grad(), or selective_scan_func to train")
    if _lib.followed():
        _lib.refuse_followed("selective_scan_step", *(t for t in (x, delta, A, B, C, D, z, delta_bias, state) if t is not None))
    active = _lib.checked_active(active, batch, dev)
    x, delta, B, C, z = rows_of(x), rows_of(delta), rows_of(B), rows_of(C), None if z is None else rows_of(z)
    with _lib.on_device(dev):
        y = x.new_empty((batch, channels))
        if batch == 0:
            return y
        strides = _Strides7(x.stride(0), delta.stride(0), 0 if z is None else z.stride(0), *B.stride()[:2], *C.stride()[:2])
        _lib.check(_lib.load().ringattr_selective_scan_step(
            x.data_ptr(), delta.data_ptr(), pointer(z), B.data_ptr(), C.data_ptr(), strides, A.data_ptr(), pointer(D), pointer(delta_bias),
            state.data_ptr(), pointer(active), y.data_ptr(), int(bool(softplus)), SEQUENCE_TYPES[x.dtype], batch, channels, N, G,
            _lib.stream_handle(dev)))
    torch.autograd.graph.increment_version(state)
    return y
