"""Linear attention with a decay for each head: the leak of the ring's time loop on a matrix of associations.

    S_t = exp(log_decay[h]) S_(t-1) + k_t v_t^T,   o_t = scale q_t S_t

`linear_attention_func` takes whole sequences (training and prompts: the chunked form, differentiable with respect to q, k, v and the
initial state, by the same kernels run over other operands), `linear_attention_step` one token for each sequence of a batch (serving:
the recurrent form, the state updated in place).  What the one leaves as its state the other goes on from.

The operands are float32, bfloat16 or float16; states are float32.  With bfloat16 what is computed on the way, weights and states, enters
products as sums of two bfloat16 numbers (2^-15), so that a result's error is its own rounding; states that are results are as exact as
float32 sums."""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import Function

from . import _lib
from ._lib import SEQUENCE_TYPES, check_sequence_sizes, check_sequence_tensor, resolved

_Strides9, _Strides12, _Strides6 = ctypes.c_longlong * 9, ctypes.c_longlong * 12, ctypes.c_longlong * 6


def _rows(t):
    """t with a head's values as neighbours (any other strides are taken as they are)."""
    if t.is_neg():
        t = resolved(t)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _checked(q, k, v, log_decay, dims):
    check_sequence_tensor("q", q)
    if q.dim() != dims:
        raise ValueError(f"q must have {dims} dimensions, got {tuple(q.shape)}")
    lead, (H, Dk), dev = tuple(q.shape[:-2]), q.shape[-2:], q.device
    check_sequence_tensor("k", k, dtype=q.dtype, device=dev)
    check_sequence_tensor("v", v, dtype=q.dtype, device=dev)
    if k.dim() != dims or tuple(k.shape[:-2]) != lead or k.shape[-1] != Dk:
        raise ValueError(f"k must have shape {lead + ('kv_heads', Dk)}, got {tuple(k.shape)}")
    G = k.shape[-2]
    if v.dim() != dims or tuple(v.shape[:-1]) != lead + (G,):
        raise ValueError(f"v must have shape {lead + (G, 'dv')}, got {tuple(v.shape)}")
    Dv = v.shape[-1]
    if H == 0 or G == 0 or Dk == 0 or Dv == 0 or H % G != 0:
        raise ValueError(f"heads ({H}) must be a positive multiple of kv_heads ({G}), dk and dv positive ({Dk}, {Dv})")
    check_sequence_sizes(q, v)
    check_sequence_tensor("log_decay", log_decay, (H,), torch.float32, dev)
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError("log_decay is a setting, as the time loop's alpha: it gets no gradient (detach it)")
    return H, G, Dk, Dv, dev


def _ptr(t):
    return None if t is None else t.data_ptr()


def _forward(q, k, v, log_decay, initial_state, lengths, scale, want_state):
    B, T, H, Dk = q.shape
    G, Dv, dev = k.shape[2], v.shape[3], q.device
    lib, kind = _lib.load(), SEQUENCE_TYPES[q.dtype]
    with _lib.on_device(dev):
        o = q.new_empty((B, T, H, Dv))
        state = log_decay.new_empty((B, H, Dk, Dv)) if want_state else None
        if B == 0 or T == 0:
            if want_state:
                state.zero_() if initial_state is None else state.copy_(initial_state)
            return o, state, None
        nbytes = lib.ringattr_linear_attention_fwd_workspace_bytes(kind, B, T, H, G, Dk, Dv)
        ws = log_decay.new_empty((nbytes // 4,)) if nbytes else None
        strides = _Strides9(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3])
        _lib.check(lib.ringattr_linear_attention_fwd(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), strides, log_decay.data_ptr(), _ptr(initial_state), _ptr(lengths), o.data_ptr(),
            _ptr(state), scale, kind, B, T, H, G, Dk, Dv, _ptr(ws), nbytes, _lib.stream_handle(dev)))
    return o, state, ws


class LinearAttentionFunc(Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, initial_state, lengths, scale, want_state):
        ctx.set_materialize_grads(False)
        o, state, along = _forward(q, k, v, log_decay, initial_state, lengths, scale, want_state)
        ctx.save_for_backward(q, k, v, log_decay, initial_state, lengths, along)
        ctx.scale = scale
        return o, state

    @staticmethod
    def backward(ctx, grad_o, grad_state):
        if torch.is_grad_enabled():              # (create_graph: the result would pass for one that does not depend on q, k and v)
            raise RuntimeError("linear_attention_func is differentiable once: its backward takes no create_graph=True")
        if _lib.followed():
            _lib.refuse_followed("the backward of linear_attention_func", *(g for g in (grad_o, grad_state) if g is not None))
        q, k, v, log_decay, initial_state, lengths, along = ctx.saved_tensors
        B, T, H, Dk = q.shape
        G, Dv, dev = k.shape[2], v.shape[3], q.device
        lib, kind = _lib.load(), SEQUENCE_TYPES[q.dtype]
        with _lib.on_device(dev):
            want = initial_state is not None and ctx.needs_input_grad[4]
            # (what is frozen costs no pass; the initial state's gradient is found along with v's)
            gq, gk, gv = (x.new_empty(x.shape) if needed else None
                          for x, needed in zip((q, k, v), (*ctx.needs_input_grad[:2], ctx.needs_input_grad[2] or want)))
            g0 = log_decay.new_empty((B, H, Dk, Dv)) if want else None
            gs = None if grad_state is None else resolved(grad_state).contiguous()
            if B == 0 or T == 0:
                if want:
                    g0.zero_() if gs is None else g0.copy_(gs)
            else:
                go = q.new_zeros((B, T, H, Dv)) if grad_o is None else _rows(grad_o)
                nbytes = lib.ringattr_linear_attention_bwd_workspace_bytes(kind, B, T, H, G, Dk, Dv, along is not None)
                ws = log_decay.new_empty((nbytes // 4,)) if nbytes else None
                strides = _Strides12(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *go.stride()[:3])
                _lib.check(lib.ringattr_linear_attention_bwd(
                    q.data_ptr(), k.data_ptr(), v.data_ptr(), go.data_ptr(), strides, log_decay.data_ptr(), _ptr(initial_state),
                    _ptr(lengths), _ptr(along), _ptr(gs), _ptr(gq), _ptr(gk), _ptr(gv), _ptr(g0), ctx.scale, kind, B, T, H, G, Dk, Dv,
                    _ptr(ws), nbytes, _lib.stream_handle(dev)))
        return gq, gk, gv if ctx.needs_input_grad[2] else None, None, g0, None, None, None


def linear_attention_func(q, k, v, log_decay, initial_state=None, lengths=None, scale=None, return_state=False):
    """Linear attention over whole sequences.

    q [B,T,H,dk], k [B,T,G,dk], v [B,T,G,dv], G a divisor of H (head h uses head h // (H // G) of k and v), dk and dv up to 256, of one
    type; a head's values lie next to each other, all other strides are free (a ring history's [T,B,..] order, a slice of one
    projection's output).  log_decay [H] float32, at most zero for a memory that fades (-inf: one that holds the last token only).
    initial_state [B,H,dk,dv] float32 or None (zeros).  lengths [B] int32 (int64 is converted) or None: how many tokens of each sequence
    count, none among the possibilities; outputs and gradients behind them are zero, nothing there is read and the state is the one
    behind the last token that counts.  scale: dk ** -0.5 if None.

    Returns o [B,T,H,dv], with return_state=True (o, the state behind the sequences).  Differentiable once with respect to q, k, v and
    initial_state.  A value that is infinite or NaN reaches the rows that see it (as an infinity or as NaN) and no other."""
    H, G, Dk, Dv, dev = _checked(q, k, v, log_decay, 4)
    B, T = q.shape[:2]
    if initial_state is not None:
        check_sequence_tensor("initial_state", initial_state, (B, H, Dk, Dv), torch.float32, dev)
        initial_state = resolved(initial_state).contiguous()
    if lengths is not None:
        if isinstance(lengths, torch.Tensor) and lengths.dtype == torch.int64:
            lengths = lengths.clamp(0, T).to(torch.int32)
        check_sequence_tensor("lengths", lengths, (B,), torch.int32, dev)
        lengths = resolved(lengths).contiguous()
    q, k, v, log_decay = _rows(q), _rows(k), _rows(v), resolved(log_decay).contiguous()
    scale = Dk ** -0.5 if scale is None else float(scale)
    if _lib.followed() or (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or
                                                       (initial_state is not None and initial_state.requires_grad))):
        o, state = LinearAttentionFunc.apply(q, k, v, log_decay, initial_state, lengths, scale, bool(return_state))
    else:
        o, state, _ = _forward(q, k, v, log_decay, initial_state, lengths, scale, bool(return_state))
    return (o, state) if return_state else o


def linear_attention_step(q, k, v, log_decay, state, active=None, scale=None):
    """One token for each sequence: q [B,H,dk], k [B,G,dk], v [B,G,dv] as in `linear_attention_func`; state [B,H,dk,dv] float32,
    contiguous, is updated in place.  active [B] (bool or uint8) or None: where it is zero the state stays as it is and the output is
    zero (a batch with places that wait).  Returns o [B,H,dv].  It has no gradient."""
    H, G, Dk, Dv, dev = _checked(q, k, v, log_decay, 3)
    B = q.shape[0]
    check_sequence_tensor("state", state, (B, H, Dk, Dv), torch.float32, dev)
    if not state.is_contiguous() or state.is_neg():
        raise RuntimeError("state must be contiguous and no negated view: it is updated in place")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad):
        raise RuntimeError("linear_attention_step has no gradient: call it under torch.no_grad(), or linear_attention_func to train")
    if _lib.followed():
        _lib.refuse_followed("linear_attention_step", q, k, v, log_decay, state)
    if active is not None:
        check_sequence_tensor("active", active, (B,), torch.uint8 if getattr(active, "dtype", None) == torch.uint8 else torch.bool, dev)
        active = active.contiguous()
    q, k, v, log_decay = _rows(q), _rows(k), _rows(v), resolved(log_decay).contiguous()
    lib = _lib.load()
    with _lib.on_device(dev):
        o = q.new_empty((B, H, Dv))
        if B == 0:
            return o
        strides = _Strides6(*q.stride()[:2], *k.stride()[:2], *v.stride()[:2])
        _lib.check(lib.ringattr_linear_attention_step(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), strides, log_decay.data_ptr(), state.data_ptr(), _ptr(active), o.data_ptr(),
            Dk ** -0.5 if scale is None else float(scale), SEQUENCE_TYPES[q.dtype], B, H, G, Dk, Dv, _lib.stream_handle(dev)))
    torch.autograd.graph.increment_version(state)
    return o
