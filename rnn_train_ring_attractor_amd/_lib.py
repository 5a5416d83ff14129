"""ctypes binding of libringattr.so (the C ABI declared in include/ringattr.h).

The library is looked up next to this file (prebuilt, in-tree); if it is absent it is built once
with hipcc (same prebuilt-then-build order as the reference's cpp/ring_rnn_cuda.py:6-16).  There is
no CPU fallback: a missing or unloadable library raises.
"""
from __future__ import annotations

import ctypes
import os
import threading

import torch  # noqa: F401  (loads torch's libamdhip64 first so the library binds to the same HIP runtime)

from . import build as _build

_lock = threading.Lock()
_lib = None

c_void_p, c_int, c_float, c_size_t, c_char_p = (ctypes.c_void_p, ctypes.c_int, ctypes.c_float,
                                                ctypes.c_size_t, ctypes.c_char_p)

# name -> (restype, argtypes): one entry per prototype in include/ringattr.h
PROTOTYPES = {
    "ringattr_version": (c_int, []),
    "ringattr_last_error": (c_char_p, []),
    "ringattr_saved_bytes": (c_size_t, [c_int] * 4),
    "ringattr_fwd_workspace_bytes": (c_size_t, [c_int] * 4),
    "ringattr_bwd_workspace_bytes": (c_size_t, [c_int] * 5),
    "ringattr_bwd_workspace_bytes_for": (c_size_t, [c_int] * 6),
    "ringattr_fwd": (c_int, [c_void_p, c_void_p, c_float, c_float, c_void_p, c_void_p, c_void_p, c_float,
                             c_int, c_int, c_int, c_int, c_int, c_void_p, c_void_p, c_size_t, c_void_p]),
    "ringattr_fwd_loss": (c_int, [c_void_p, c_void_p, c_float, c_float, c_void_p, c_void_p, c_void_p, c_float,
                                  c_int, c_int, c_int, c_int, c_int, c_void_p, c_void_p, c_size_t,
                                  c_void_p, c_void_p, c_float, c_void_p, c_void_p, c_size_t, c_void_p]),
    "ringattr_fwd_loss_total": (c_int, [c_void_p, c_void_p, c_float, c_float, c_void_p, c_void_p, c_void_p, c_float,
                                  c_int, c_int, c_int, c_int, c_int, c_void_p, c_void_p, c_size_t,
                                  c_void_p, c_void_p, c_float, c_void_p, c_void_p, c_void_p, c_size_t, c_void_p]),
    "ringattr_fwd_noalloc": (c_int, [c_void_p, c_void_p, c_float, c_float, c_void_p, c_void_p, c_void_p, c_float,
                                     c_int, c_int, c_int, c_int, c_int, c_void_p, c_void_p]),
    "ringattr_bwd": (c_int, [c_void_p, c_void_p, c_void_p, c_float, c_float, c_void_p, c_void_p, c_void_p,
                             c_void_p, c_void_p, c_float, c_int, c_int, c_int, c_int, c_int, c_int,
                             c_void_p, c_void_p, c_void_p, c_void_p, c_size_t, c_void_p]),
    "ringattr_loss_workspace_bytes": (c_size_t, [c_int] * 3),
    "ringattr_loss_fwd": (c_int, [c_void_p, c_void_p, c_void_p, c_float, c_void_p, c_int, c_int, c_int,
                                  c_void_p, c_size_t, c_void_p]),
    "ringattr_loss_bwd": (c_int, [c_void_p, c_void_p, c_void_p, c_float, c_void_p, c_void_p, c_int, c_int, c_int,
                                  c_void_p, c_size_t, c_void_p]),
    "ringattr_bwd_loss_available": (c_int, [c_int] * 4),
    "ringattr_bwd_loss": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_float, c_float, c_void_p, c_void_p, c_void_p,
                                  c_void_p, c_void_p, c_float, c_int, c_int, c_int, c_int, c_int, c_int,
                                  c_void_p, c_void_p, c_void_p, c_void_p, c_size_t, c_void_p]),
    "ringattr_gain_workspace_bytes": (c_size_t, [c_int] * 4),
    "ringattr_gain_fwd": (c_int, [c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p]),
    "ringattr_gain_bwd": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int,
                                  c_void_p, c_size_t, c_void_p]),
    "ringattr_generator_initial_zeros": (c_int, [c_int, ctypes.c_double]),
    "ringattr_generate_inputs": (c_int, [ctypes.c_ulonglong, c_int, c_int, c_int, c_int, ctypes.c_double,
                                         ctypes.POINTER(c_float), c_int, c_float, c_int, c_int, c_float,
                                         c_void_p, c_void_p, c_void_p, c_void_p, c_void_p]),
    "ringattr_gain_nets_fwd": (c_int, [c_void_p, c_int, ctypes.POINTER(c_void_p), c_void_p, c_int, c_int, c_int, c_int, c_void_p]),
    "ringattr_gain_nets_fwd_kept": (c_int, [c_void_p, c_int, ctypes.POINTER(c_void_p), c_void_p, c_void_p, c_int, c_int, c_int, c_int,
                                            c_void_p]),
    "ringattr_gain_nets_bwd": (c_int, [c_void_p, c_int, ctypes.POINTER(c_void_p), c_void_p, c_void_p, c_int, c_int, c_int, c_int,
                                       c_void_p, c_size_t, c_void_p]),
    "ringattr_action_signal": (c_int, [c_void_p, c_void_p, c_int, c_int, c_int, c_void_p]),
    "ringattr_bump": (c_int, [c_void_p, c_size_t, c_void_p, c_int, c_int, c_float, c_void_p]),
    "ringattr_compact_workspace_bytes": (c_size_t, []),
    "ringattr_compact_channels": (c_int, [c_void_p] * 4 + [c_int] * 6 + [c_void_p, c_size_t, c_void_p]),
    "ringattr_clip_adam_workspace_bytes": (c_size_t, [c_int, ctypes.POINTER(c_size_t)]),
    "ringattr_clip_adam": (c_int, [c_int, ctypes.POINTER(c_void_p), ctypes.POINTER(c_void_p), ctypes.POINTER(c_void_p),
                                   ctypes.POINTER(c_void_p), ctypes.POINTER(c_size_t), c_float, c_float, c_float,
                                   c_float, c_float, c_int, c_void_p, c_size_t, c_void_p]),
    "ringattr_clip_adam_counted": (c_int, [c_int, ctypes.POINTER(c_void_p), ctypes.POINTER(c_void_p),
                                           ctypes.POINTER(c_void_p), ctypes.POINTER(c_void_p), ctypes.POINTER(c_size_t),
                                           c_float, c_float, c_float, c_float, c_float, c_void_p, c_void_p, c_size_t,
                                           c_void_p]),
    "ringattr_linear_attention_fwd_workspace_bytes": (c_size_t, [c_int] * 7),
    "ringattr_linear_attention_fwd": (c_int, [c_void_p] * 3 + [ctypes.POINTER(ctypes.c_longlong)] + [c_void_p] * 5 + [c_float] +
                                      [c_int] * 7 + [c_void_p, c_size_t, c_void_p]),
    "ringattr_linear_attention_bwd_workspace_bytes": (c_size_t, [c_int] * 8),
    "ringattr_linear_attention_bwd": (c_int, [c_void_p] * 4 + [ctypes.POINTER(ctypes.c_longlong)] + [c_void_p] * 9 + [c_float] +
                                      [c_int] * 7 + [c_void_p, c_size_t, c_void_p]),
    "ringattr_linear_attention_step": (c_int, [c_void_p] * 3 + [ctypes.POINTER(ctypes.c_longlong)] + [c_void_p] * 4 + [c_float] +
                                       [c_int] * 6 + [c_void_p]),
    "ringattr_rotary": (c_int, [c_void_p] * 2 + [ctypes.POINTER(ctypes.c_longlong), c_void_p, ctypes.c_longlong, ctypes.c_longlong, c_int] +
                        [c_void_p] * 3 + [c_float] + [c_int] * 9 + [c_void_p]),
    "ringattr_dropout": (c_int, [c_void_p] * 3 + [c_size_t, ctypes.c_uint, c_float, ctypes.c_ulonglong, ctypes.c_ulonglong, c_void_p, c_int,
                                 c_void_p]),
    "ringattr_causal_conv_fwd": (c_int, [c_void_p, ctypes.POINTER(ctypes.c_longlong)] + [c_void_p] * 6 + [c_int] * 6 + [c_void_p]),
    "ringattr_causal_conv_bwd_workspace_bytes": (c_size_t, [c_int] * 6),
    "ringattr_causal_conv_bwd": (c_int, [c_void_p] * 2 + [ctypes.POINTER(ctypes.c_longlong)] + [c_void_p] * 9 + [c_int] * 6 +
                                 [c_void_p, c_size_t, c_void_p]),
    "ringattr_causal_conv_step": (c_int, [c_void_p, ctypes.c_longlong] + [c_void_p] * 5 + [c_int] * 5 + [c_void_p]),
    "ringattr_selective_scan_states_bytes": (c_size_t, [c_int] * 6),
    "ringattr_selective_scan_fwd_workspace_bytes": (c_size_t, [c_int] * 6),
    "ringattr_selective_scan_fwd": (c_int, [c_void_p] * 5 + [ctypes.POINTER(ctypes.c_longlong)] + [c_void_p] * 8 + [c_int] * 7 +
                                    [c_void_p, c_size_t, c_void_p]),
    "ringattr_selective_scan_bwd_workspace_bytes": (c_size_t, [c_int] * 8),
    "ringattr_selective_scan_bwd": (c_int, [c_void_p] * 6 + [ctypes.POINTER(ctypes.c_longlong)] + [c_void_p] * 15 + [c_int] * 7 +
                                    [c_void_p, c_size_t, c_void_p]),
    "ringattr_selective_scan_step": (c_int, [c_void_p] * 5 + [ctypes.POINTER(ctypes.c_longlong)] + [c_void_p] * 6 + [c_int] * 6 + [c_void_p]),
    "ringattr_norm_gate_fwd": (c_int, [c_void_p] * 3 + [ctypes.POINTER(ctypes.c_longlong)] + [c_void_p] * 5 + [c_float] + [c_int] * 3 +
                               [c_size_t, c_int, c_int, c_void_p]),
    "ringattr_norm_gate_bwd_workspace_bytes": (c_size_t, [c_int, c_size_t] + [c_int] * 3),
    "ringattr_norm_gate_bwd": (c_int, [c_void_p] * 5 + [ctypes.POINTER(ctypes.c_longlong)] + [c_void_p] * 9 + [c_float] + [c_int] * 3 +
                               [c_size_t, c_int, c_int, c_void_p, c_size_t, c_void_p]),
    "ringattr_profile_enable": (c_int, [c_int]),
    "ringattr_profile_read": (c_int, [ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_longlong)]),
    "ringattr_last_kernel_name": (c_int, [c_int, ctypes.c_char_p, ctypes.c_size_t]),
    "ringattr_dw_segments": (c_int, [c_int] * 4),
    "fwd_cuda": (None, [c_void_p, c_void_p, c_float, c_float, c_void_p, c_void_p, c_void_p, c_float,
                        c_int, c_int, c_int, c_int, c_int]),
    "bwd_cuda": (None, [c_void_p, c_void_p, c_void_p, c_float, c_float, c_void_p, c_void_p, c_void_p, c_void_p,
                        c_void_p, c_void_p, c_float, c_int, c_int, c_int, c_int, c_int,
                        c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p]),
}


def library_path() -> str:
    """In-tree library, or the file named by RINGATTR_LIB (to try an experimental build)."""
    return os.environ.get("RINGATTR_LIB") or _build.LIB_PATH


def load():
    """Return the loaded library, building it first if no prebuilt file exists."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        path = library_path()
        if not os.path.exists(path):
            _build.build_library()
        lib = ctypes.CDLL(path)
        for name, (res, args) in PROTOTYPES.items():
            fn = getattr(lib, name)          # AttributeError if the library lacks a declared symbol
            fn.restype = res
            fn.argtypes = args
        _lib = lib
        return lib


def last_error() -> str:
    return load().ringattr_last_error().decode("utf-8", "replace")


def check(rc: int) -> None:
    """Turn a status code into a Python exception (the reference exits the process instead,
    cpp/cuda_common.cuh:30-39)."""
    if rc == 0:
        return
    msg = last_error()
    if rc == 1:
        raise ValueError(msg)
    raise RuntimeError(msg)


KERNEL_NAMES = ("pack_weights", "fwd", "rebuild_saved", "bptt", "dw", "dw_reduce")


def profile_enable(on) -> None:
    """False / 0: off.  True / 1: bracket every kernel launch with HIP events; n > 1: every n-th launch of each kernel
    (the two event records cost the stream 4-5 us per bracketed launch)."""
    check(load().ringattr_profile_enable(int(on)))


def last_kernel_names():
    """{kernel slot name: name of the kernel launched last in it} for the slots that have launched."""
    out = {}
    buf = ctypes.create_string_buffer(256)
    for i, key in enumerate(KERNEL_NAMES):
        check(load().ringattr_last_kernel_name(i, buf, len(buf)))
        if buf.value:
            out[key] = buf.value.decode()
    return out


def profile_read():
    """Returns {kernel name: (total ms, launches)} of the launches recorded since the last read."""
    n = len(KERNEL_NAMES)
    ms = (ctypes.c_double * n)()
    cnt = (ctypes.c_longlong * n)()
    check(load().ringattr_profile_read(ms, cnt))
    return {KERNEL_NAMES[i]: (ms[i], cnt[i]) for i in range(n)}


_C, _forward_ad = torch._C, torch.autograd.forward_ad
_SIZE_LIMIT = 1 << 31
SEQUENCE_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # RINGATTR_F32, _BF16, _F16


def check_sequence_sizes(*tensors) -> None:
    """Sizes go to the library in 32 bits with a sign, where larger ones would be others (a dimension that is expanded can be any size)."""
    for t in tensors:
        if t.numel() >= _SIZE_LIMIT and max(t.shape) >= _SIZE_LIMIT:
            raise ValueError(f"sizes must be below 2^31, got {tuple(t.shape)}")


def resolved(t):
    """t, written out if torch keeps it negated lazily (the imaginary part of a conjugate): kernels read memory as it lies."""
    return t.resolve_neg() if t is not None and t.is_neg() else t


def check_sequence_tensor(name, t, shape=None, dtype=None, device=None) -> None:
    """What the sequence operators ask of a tensor: one of their types (or the one given), on the GPU, and the shape."""
    # (in most cases these three; `device` is that of a tensor that has been looked at)
    if type(t) is torch.Tensor and t.dtype is dtype and device is not None and t.device == device and (shape is None or t.shape == shape):
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if dtype is None:
        if t.dtype not in SEQUENCE_TYPES:
            raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    elif t.dtype != dtype:
        raise TypeError(f"{name} must be {str(dtype)[6:]}, got {t.dtype}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if not t.is_cuda or (device is not None and t.device != device):
        raise RuntimeError(f"{name} must be on {device if device is not None else 'a GPU'} (got {t.device}); there is no CPU path")


def rows_of(t):
    """t, or a copy of it, with its last dimension's values as neighbours and as they are meant (any other strides are taken as they are)."""
    if t.is_neg():
        t = resolved(t)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def pointer(t):
    return None if t is None else t.data_ptr()


def empty_of(t):
    """Memory for a result of t's shape and type, contiguous (the first way costs the host a third less)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def checked_lengths(lengths, B, T, device):
    """The tokens that count of each sequence of a padded batch, as the library takes them."""
    if lengths is None:
        return None
    if isinstance(lengths, torch.Tensor) and lengths.dtype == torch.int64:
        lengths = lengths.clamp(0, T).to(torch.int32)
    check_sequence_tensor("lengths", lengths, (B,), torch.int32, device)
    return resolved(lengths).contiguous()


def checked_active(active, B, device):
    """Which places of a served batch take part in a step, as the library takes them."""
    if active is None:
        return None
    check_sequence_tensor("active", active, (B,), torch.uint8 if getattr(active, "dtype", None) == torch.uint8 else torch.bool, device)
    return active.contiguous()


def checked_parameter(name, t, shape, device):
    """A parameter, float32 and contiguous."""
    if t is None:
        return None
    check_sequence_tensor(name, t, shape, torch.float32, device)
    return resolved(t).contiguous()


def wants_gradient(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


class _Here:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def on_device(device):
    """`torch.cuda.device(device)` for a tensor's device; nothing to enter and leave where it is the current one.  (The question
    without the checks around it, where torch still has that private name: there is a tensor on the device.)"""
    try:
        here = torch._C._cuda_getDevice()
    except AttributeError:
        here = torch.cuda.current_device()
    return _HERE if here == device.index else torch.cuda.device(device)


def stream_handle(device) -> int:
    """The current stream of a tensor's device, as the library takes it.  (Without the Stream object around it, where torch
    still has that private name.)"""
    try:
        return torch._C._cuda_getCurrentRawStream(device.index)
    except AttributeError:
        return torch.cuda.current_stream(device).cuda_stream


def plain_gpu_tensor(t) -> bool:
    """Whether a helper may hand t's memory to a kernel in place of a chain of torch operations: an fp32 GPU tensor that no
    derivative is wanted of, and nothing that watches or transforms the operations (autograd, forward mode, functorch,
    tracing, compilation, a dispatch or function mode) to miss them."""
    if type(t) is not torch.Tensor or not t.is_cuda or t.dtype != torch.float32 or t.layout != torch.strided:
        return False
    if (t.requires_grad and torch.is_grad_enabled()) or torch.compiler.is_compiling() or torch.jit.is_tracing():
        return False
    return not _watched() and not t.is_neg() and t.numel() > 0


def _watched() -> bool:
    """functorch, forward mode, a dispatch or function mode.  These are torch's private names: where a version has them no
    longer, the helpers keep to the tensor operations."""
    try:
        return (torch._C._functorch.maybe_current_level() is not None or torch.autograd.forward_ad._current_level >= 0
                or torch._C._len_torch_dispatch_stack() != 0 or torch._C._len_torch_function_stack() != 0)
    except AttributeError:
        return True


def followed() -> bool:
    """Whether something beside autograd's backward follows the operations on tensors (tracing, functorch, forward mode; `_watched`'s private
    names).  An operator is called as an autograd Function then, which is recorded, or refused where it lacks a rule."""
    try:
        return _C._is_tracing() or _C._functorch.maybe_current_level() is not None or _forward_ad._current_level >= 0
    except AttributeError:
        return True


def refuse_followed(who, *tensors) -> None:
    """The same for an operator without any derivative, which is no Function: it raises."""
    if torch.jit.is_tracing():
        raise RuntimeError(f"{who} cannot be traced")
    # (a private name: without it a wrapped tensor is refused where its memory is asked for)
    wrapped = getattr(getattr(torch._C, "_functorch", None), "is_functorch_wrapped_tensor", lambda t: False)
    for t in tensors:
        if wrapped(t) or torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{who} has no gradient, in forward mode and function transforms neither")
