"""Host side of the sequence operators: what they refuse, workspace sizes, frequencies and the oracle's two forms.  No kernel is launched."""
import ctypes
import math

import pytest
import torch

from oracle import sequence_oracle as O
from rnn_train_ring_attractor_amd import (_lib, dropout_func, linear_attention_func, linear_attention_step, rotary_frequencies,
                                          rotary_func)


def test_oracle_forms_agree_and_its_gradients_are_differences():
    gen = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)
    q, k, v, s0 = r(2, 9, 4, 3), r(2, 9, 2, 3), r(2, 9, 2, 5), r(2, 4, 3, 5)
    g = torch.tensor([0.0, -0.1, -2.0, -math.inf], dtype=torch.float64)
    for start in (None, s0):
        a, b = O.attention(q, k, v, g, start), O.attention_recurrent(q, k, v, g, start)
        assert all(torch.allclose(x, y, rtol=0, atol=1e-12) for x, y in zip(a, b))
    o, s = O.attention(q, k, v, g, s0, lengths=[4, 0])
    a = O.attention_recurrent(q[:1, :4], k[:1, :4], v[:1, :4], g, s0[:1])
    assert torch.allclose(o[:1, :4], a[0]) and (o[0, 4:] == 0).all() and (o[1] == 0).all()
    assert torch.allclose(s[:1], a[1]) and torch.equal(s[1], s0[1])
    leaves = [x.requires_grad_(True) for x in (q, k, v, s0)]
    assert torch.autograd.gradcheck(lambda *x: O.attention(*x[:3], g[:3].repeat(2)[:4], x[3]), leaves, atol=1e-6)


def test_philox():
    """One round by hand: zeros stay zeros but for the key, which the next round's key is added to."""
    assert O.philox_words(0, 0, 0, rounds=1) == [0, 0, 0, 0]
    assert O.philox_words(0, 0, 0, rounds=2) == [0x9E3779B9, 0, 0xBB67AE85, 0]
    assert O.philox_words(1, 0, 0, rounds=1) == [0, 0, 0, 0xD2511F53]
    assert O.philox_words(2 ** 32 + 4, 2 ** 32 * 7 + 2, 2 ** 32 * 9 + 8, rounds=1) == [
        (2 * 0xCD9E8D57 >> 32) ^ 1 ^ 8, 2 * 0xCD9E8D57 % 2 ** 32, (4 * 0xD2511F53 >> 32) ^ 7 ^ 9, 4 * 0xD2511F53 % 2 ** 32]
    keep = O.keep_mask(20000, 0.3, 5, 6)
    assert abs(keep.mean() - 0.7) < 5 * math.sqrt(0.21 / 20000)          # five standard deviations
    assert (O.keep_mask(100, 0.3, 5, 6, first=37) == keep[37:137]).all()
    assert (O.keep_mask(100, 0.3, 5, 7) != keep[:100]).any() and (O.keep_mask(100, 0.3, 4, 6) != keep[:100]).any()


def test_frequencies():
    f, scale = rotary_frequencies(8, base=100.0, device="cpu")
    assert f.dtype == torch.float64 and scale == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64))
    assert torch.allclose(rotary_frequencies(8, 100.0, "linear", 4.0, device="cpu")[0], f / 4)
    b, _ = rotary_frequencies(8, 100.0, "base", 4.0, device="cpu")
    assert b[0] == f[0] and math.isclose(float(b[-1]), float(f[-1]) / 4)
    r, scale = rotary_frequencies(64, 10000.0, "ramp", 8.0, original_length=2048, device="cpu")
    p = rotary_frequencies(64, device="cpu")[0]
    assert r[0] == p[0] and math.isclose(float(r[-1]), float(p[-1]) / 8) and math.isclose(scale, 0.1 * math.log(8) + 1)
    assert ((r <= p) & (r >= p / 8)).all() and (r[1:] < r[:-1]).all()
    for bad in (dict(rotary_dim=7), dict(rotary_dim=8, base=1.0), dict(rotary_dim=8, factor=0.5), dict(rotary_dim=8, scaling="other"),
                dict(rotary_dim=8, scaling="ramp", factor=2.0), dict(rotary_dim=2, scaling="base", factor=2.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad, device="cpu")


def _qkv():
    return torch.zeros(2, 3, 4, 8), torch.zeros(2, 3, 2, 8), torch.zeros(2, 3, 2, 6), torch.zeros(4)


def test_python_refusals():
    q, k, v, g = _qkv()
    with pytest.raises(RuntimeError, match="no CPU path"):
        linear_attention_func(q, k, v, g)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        linear_attention_func(q.double(), k, v, g)
    with pytest.raises(RuntimeError, match="no CPU path"):
        linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, torch.zeros(2, 4, 8, 6))
    f = torch.ones(4, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        rotary_func(q, torch.arange(3), f)
    with pytest.raises(ValueError, match="Invalid layout"):
        rotary_func(q, torch.arange(3), f, layout="quarter")
    with pytest.raises(RuntimeError, match="no CPU path"):
        dropout_func(q, 0.1, 1)
    with pytest.raises(TypeError):
        dropout_func([1.0], 0.1, 1)


def test_c_abi_refusals():
    lib = _lib.load()
    buf = (ctypes.c_char * 8192)()
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    st = (ctypes.c_longlong * 12)(*[8] * 12)
    shape = [1, 2, 3, 4, 2, 8, 6]                                        # type, B, T, heads, kv_heads, dk, dv
    fwd = lambda s=shape, q=p, o=p, ws=None, n=0: lib.ringattr_linear_attention_fwd(q, p, p, st, p, None, None, o, None, 1.0, *s, ws, n, None)
    bwd = lambda s=shape, go=p, gq=p, ws=None, n=0: lib.ringattr_linear_attention_bwd(p, p, p, go, st, p, None, None, None, None, gq, p, p, None, 1.0, *s,
                                                                                    ws, n, None)
    step = lambda s, q=p: lib.ringattr_linear_attention_step(q, p, p, st, p, p, None, p, 1.0, *s, None)
    changed = lambda i, x: shape[:i] + [x] + shape[i + 1:]
    for call in (fwd, bwd):
        assert call(changed(0, 3)) == 1 and "type" in _lib.last_error()
        assert call(changed(1, 0)) == 1 and "positive" in _lib.last_error()
        assert call(changed(4, 3)) == 1 and "multiple" in _lib.last_error()
        assert call(changed(5, 257)) == 1 and "256" in _lib.last_error()
        assert call(changed(1, 2000000)) == 1
    assert fwd(q=None) == 1 and "null" in _lib.last_error()
    assert fwd(o=p + 8) == 1 and "aligned" in _lib.last_error()
    assert bwd(go=None) == 1 and bwd(gq=p + 4) == 1
    assert bwd() == 2 and "workspace" in _lib.last_error()               # shared heads are summed in one
    long = [1, 1, 100000, 1, 1, 8, 6]
    assert lib.ringattr_linear_attention_fwd_workspace_bytes(*shape) == 0
    need = lib.ringattr_linear_attention_fwd_workspace_bytes(*long)
    assert need > 0 and need % 256 == 0
    states = [lib.ringattr_linear_attention_bwd_workspace_bytes(*long, have) for have in (0, 1)]
    assert states == [2 * need, need]                                    # the forward's own states, kept or formed again
    assert fwd(long) == 2 and fwd(long, ws=p, n=need - 1) == 2 and "workspace" in _lib.last_error()
    assert lib.ringattr_linear_attention_bwd_workspace_bytes(*changed(5, 300), 0) == 0 and "256" in _lib.last_error()
    one = [1, 2, 4, 2, 8, 6]
    assert step(one, q=None) == 1 and step([1, 2, 4, 3, 8, 6]) == 1 and step([9] + one[1:]) == 1
    rot = lambda kind=0, heads=(2, 0), dim=8, r=8, t=1, x1=None: lib.ringattr_rotary(p, x1, st, p, 0, 1, kind, p, p, None, 1.0, 0, 0, t, 2, 3, *heads, dim,
                                                                                 r, None)
    assert rot(kind=3) == 1 and "position_type" in _lib.last_error()
    assert rot(r=7) == 1 and rot(r=10) == 1 and rot(r=0) == 1 and rot(dim=4096, r=2050) == 1 and "rot" in _lib.last_error()
    assert rot(heads=(2, 1)) == 1 and "null" in _lib.last_error()
    assert rot(heads=(0, 0)) == 1 and rot(t=5) == 1 and rot(heads=(70000, 0), dim=64) == 1
    drop = lambda n=4, x=p, t=0: lib.ringattr_dropout(x, None, p, n, 5, 1.0, 0, 0, None, t, None)
    assert drop(n=0) == 1 and drop(x=None) == 1 and drop(t=-1) == 1
