"""Host side of the recurrent layer's operators: what they refuse, workspace sizes and the oracle.  No kernel is launched."""
import ctypes

import pytest
import torch

from oracle import recurrent_oracle as O
from rnn_train_ring_attractor_amd import (_lib, causal_conv_func, causal_conv_step, norm_gate_func, selective_scan_func, selective_scan_step)


def _r(gen, *shape):
    return torch.randn(*shape, generator=gen, dtype=torch.float64)


def test_oracle_gradients_are_differences_and_sizes_bound_them():
    gen = torch.Generator().manual_seed(1)
    x, w, bias, start = _r(gen, 2, 6, 3), _r(gen, 3, 3), _r(gen, 3), _r(gen, 2, 2, 3)
    lengths = [6, 1]
    check = lambda f, *leaves: torch.autograd.gradcheck(f, [t.requires_grad_(True) for t in leaves], atol=1e-6)
    assert check(lambda *t: O.conv(*t, lengths, "silu"), x, w, bias, start)
    A, B, C, D, z = -torch.exp(_r(gen, 4, 2)), _r(gen, 2, 6, 2, 2), _r(gen, 2, 6, 2, 2), _r(gen, 4), _r(gen, 2, 6, 4)
    u, delta, b, s = _r(gen, 2, 6, 4), _r(gen, 2, 6, 4), _r(gen, 4), _r(gen, 2, 4, 2)
    leaves = (u, delta, A, B, C, D, z, b, s)
    assert check(lambda *t: O.scan(*t, lengths, True), *leaves)
    assert check(lambda *t: O.norm_gate(*t, 2, 1e-5, "layer", "sigmoid"), _r(gen, 3, 4), _r(gen, 4), _r(gen, 3, 4), _r(gen, 3, 4), _r(gen, 4), _r(gen, 4))
    dy, de = _r(gen, 2, 6, 4), _r(gen, 2, 4, 2)
    y, end = O.scan(*leaves, lengths, True)
    grads = torch.autograd.grad([y, end], leaves, [dy, de])
    size, _ = O.scan_sizes(*(t.detach() for t in leaves), lengths, True, dy, de)
    for n, t in zip(("y", "state", "dx", "ddelta", "dA", "dB", "dC", "dD", "dz", "dbias", "dstart"), (y, end, *grads)):
        assert (t.detach().abs() <= size[n] + 1e-12).all(), n


def test_oracle_pieces_go_on_from_each_other():
    gen = torch.Generator().manual_seed(2)
    x, w = _r(gen, 1, 9, 3), _r(gen, 3, 4)
    y, end = O.conv(x, w)
    a, mid = O.conv(x[:, :2], w)
    b, last = O.conv(x[:, 2:], w, start=mid)
    assert torch.allclose(torch.cat([a, b], 1), y) and torch.equal(last, end) and torch.equal(end, x[:, 6:])


def test_python_refusals():
    x, w = torch.zeros(2, 3, 4), torch.zeros(4, 3)
    with pytest.raises(RuntimeError, match="no CPU path"):
        causal_conv_func(x, w)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        causal_conv_func(x.double(), w)
    with pytest.raises(RuntimeError, match="no CPU path"):
        selective_scan_func(x, x, torch.zeros(4, 2), torch.zeros(2, 3, 1, 2), torch.zeros(2, 3, 1, 2))
    with pytest.raises(RuntimeError, match="no CPU path"):
        norm_gate_func(x, torch.zeros(4))
    with pytest.raises(RuntimeError, match="no CPU path"):
        causal_conv_step(x[:, 0], w, torch.zeros(2, 2, 4))
    with pytest.raises(RuntimeError, match="no CPU path"):
        selective_scan_step(x[:, 0], x[:, 0], torch.zeros(4, 2), torch.zeros(2, 1, 2), torch.zeros(2, 1, 2), torch.zeros(2, 4, 2))
    for call in (causal_conv_func, norm_gate_func):
        with pytest.raises(TypeError):
            call([1.0], w)


def test_c_abi_refusals():
    lib = _lib.load()
    buf = (ctypes.c_char * 8192)()
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    st = (ctypes.c_longlong * 16)(*[8] * 16)
    changed = lambda shape, i, v: shape[:i] + [v] + shape[i + 1:]
    # convolution: activation, type, B, T, C, taps
    shape = [1, 1, 2, 3, 8, 4]
    fwd = lambda s=shape, x=p, y=p: lib.ringattr_causal_conv_fwd(x, st, p, None, None, None, y, None, *s, None)
    bwd = lambda s=shape, gy=p, gx=p, gw=None, ws=None, n=0: lib.ringattr_causal_conv_bwd(p, gy, st, p, None, None, None, None, gx, gw, None, None, *s, ws, n, None)
    step = lambda s, x=p, state=p: lib.ringattr_causal_conv_step(x, 8, p, None, state, None, p, *s, None)
    for call in (fwd, bwd):
        assert call(changed(shape, 0, 2)) == 1 and "activation" in _lib.last_error()
        assert call(changed(shape, 1, 3)) == 1 and "type" in _lib.last_error()
        assert call(changed(shape, 2, 0)) == 1 and "positive" in _lib.last_error()
        assert call(changed(shape, 5, 9)) == 1 and call(changed(shape, 5, 0)) == 1 and "taps" in _lib.last_error()
        assert call(changed(shape, 2, 1 << 21)) == 1 and call(changed(changed(shape, 2, 1 << 16), 4, 1 << 16)) == 1 and "2^20" in _lib.last_error()
    assert fwd(x=None) == 1 and fwd(y=p + 8) == 1 and "aligned" in _lib.last_error()
    assert bwd(gy=None) == 1 and bwd(gx=p + 4) == 1
    need = lib.ringattr_causal_conv_bwd_workspace_bytes(*shape[1:], 1)
    assert need > 0 and lib.ringattr_causal_conv_bwd_workspace_bytes(*shape[1:], 0) == 0
    assert bwd(gw=p) == 2 and bwd(gw=p, ws=p, n=need - 1) == 2 and "workspace" in _lib.last_error()
    assert step([1, 1, 2, 8, 4], x=None) == 1 and step([1, 1, 2, 8, 4], state=None) == 1 and step([1, 1, 2, 8, 9]) == 1
    # scan: softplus, type, B, T, C, N, G
    shape = [1, 1, 2, 300, 64, 16, 2]
    fwd = lambda s=shape, x=p, y=p, ws=None, n=0: lib.ringattr_selective_scan_fwd(x, p, None, p, p, st, p, None, None, None, None, y, None, None, *s, ws, n, None)
    bwd = lambda s=shape, kept=p, gx=p, gz=None, gB=None, gA=None, ws=None, n=0: lib.ringattr_selective_scan_bwd(
        p, p, None, p, p, p, st, p, None, None, None, kept, None, gx, p, gz, gB, None, gA, None, None, None, *s, ws, n, None)
    for call in (fwd, bwd):
        assert call(changed(shape, 1, -1)) == 1 and "type" in _lib.last_error()
        assert call(changed(shape, 3, 0)) == 1 and "positive" in _lib.last_error()
        assert call(changed(shape, 5, 65)) == 1 and "states" in _lib.last_error()
        assert call(changed(shape, 6, 5)) == 1 and "multiple" in _lib.last_error()
        assert call(changed(shape, 3, (1 << 30) + 1)) == 1
        assert call([1, 1, 1 << 12, 3, 3000, 16, 3000]) == 1 and "groups" in _lib.last_error()
    sizes = shape[1:]
    assert fwd(x=None) == 1 and fwd(y=p + 4) == 1
    assert lib.ringattr_selective_scan_states_bytes(*sizes) == 2 * 19 * 64 * 16 * 4
    need = lib.ringattr_selective_scan_fwd_workspace_bytes(*sizes)
    assert need > 0 and need % 256 == 0 and fwd() == 2 and fwd(ws=p, n=need - 1) == 2 and "workspace" in _lib.last_error()
    assert bwd(kept=None) == 1 and bwd(gx=p + 8) == 1 and bwd(gz=p) == 1 and "grad_z" in _lib.last_error()
    queries = [lib.ringattr_selective_scan_bwd_workspace_bytes(*sizes, a, b) for a, b in ((0, 0), (1, 0), (0, 1), (1, 1))]
    assert queries[3] == queries[1] + queries[2] - queries[0] and queries[1] > queries[0] and queries[2] > queries[0]
    assert bwd(gB=p, ws=p, n=queries[1] - 1) == 2 and bwd(gA=p, ws=p, n=queries[2] - 1) == 2
    assert lib.ringattr_selective_scan_bwd_workspace_bytes(*changed(sizes, 4, 65), 0, 0) == 0
    step = lambda s, x=p, state=p: lib.ringattr_selective_scan_step(x, p, None, p, p, st, p, None, None, state, None, p, *s, None)
    assert step([1, 1, 2, 8, 4, 1], x=None) == 1 and step([1, 1, 2, 8, 4, 1], state=None) == 1 and step([1, 1, 2, 8, 4, 3]) == 1
    # norm: layer, activation, type, rows, channels, group
    shape = [0, 1, 1, 6, 8, 4]
    fwd = lambda s=shape, x=p, y=p, nxt=None, n=None: lib.ringattr_norm_gate_fwd(x, None, None, st, p, None, nxt, y, n, 1e-5, *s, None)
    bwd = lambda s=shape, gy=p, gn=None, gx=p, gg=None, gw=None, gs=None, gnw=None, ws=None, n=0: lib.ringattr_norm_gate_bwd(
        p, None, None, gy, gn, st, p, None, None, gx, gg, None, gw, gs, gnw, 1e-5, *s, ws, n, None)
    for call in (fwd, bwd):
        assert call(changed(shape, 1, 3)) == 1 and "activation" in _lib.last_error()
        assert call(changed(shape, 2, 7)) == 1 and "type" in _lib.last_error()
        assert call(changed(shape, 3, 0)) == 1 and call(changed(shape, 4, 8193)) == 1 and "8192" in _lib.last_error()
        assert call(changed(shape, 5, 3)) == 1 and "group" in _lib.last_error()
    assert fwd(x=None) == 1 and fwd(y=p + 8) == 1 and fwd(nxt=p) == 1 and "null" in _lib.last_error()
    assert bwd(gy=None) == 1 and bwd(gx=p + 8) == 1
    for bad in (dict(gn=p), dict(gg=p), dict(gs=p), dict(gnw=p)):
        assert bwd(**bad) == 1 and "gradient of" in _lib.last_error()
    need = lib.ringattr_norm_gate_bwd_workspace_bytes(*shape[2:], 1)
    assert need > 0 and lib.ringattr_norm_gate_bwd_workspace_bytes(*shape[2:], 0) == 0 and bwd(gw=p) == 2 and bwd(gw=p, ws=p, n=need - 1) == 2


def test_c_abi_refusals_of_single_tokens():
    """Sequences times channels times states (a power of two) end at 2^31, what a launch counts; sequences and channels at 2^20 each."""
    lib = _lib.load()
    buf = (ctypes.c_char * 512)()
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    st = (ctypes.c_longlong * 16)(*[8] * 16)
    conv = lambda B, C: lib.ringattr_causal_conv_step(p, 8, p, None, p, None, p, 1, 1, B, C, 4, None)
    scan = lambda B, C, N, G: lib.ringattr_selective_scan_step(p, p, None, p, p, st, p, None, None, p, None, p, 1, 1, B, C, N, G, None)
    for call in (lambda: conv(1 << 12, (1 << 19) + 8), lambda: conv((1 << 20) + 1, 8), lambda: conv(8, (1 << 20) + 8), lambda: scan(1 << 14, 1 << 12, 33, 1),
                 lambda: scan(1 << 16, (1 << 11) + 1, 16, 1), lambda: scan((1 << 20) + 1, 8, 1, 1)):
        assert call() == 1 and "2^20" in _lib.last_error()
    assert conv(0, 8) == 1 and scan(1, 0, 1, 1) == 1 and "positive" in _lib.last_error()
    assert scan(1 << 13, 1 << 11, 65, 1) == 1 and scan(1 << 13, 1 << 11, 16, 3) == 1 and "multiple" in _lib.last_error()
