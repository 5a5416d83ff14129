"""The recurrent layer's operators where their inner loops run: pieces of many tokens, workgroups that walk many rows, steps that are taken as they are,
and gradients against differences.  Bounds are counted as in test_gpu_recurrent.py; a parameter's sum has as many additions behind one another as a
thread has tokens (a workgroup rows), a workgroup threads, and the last sum parts."""
import math

import pytest
import torch

from oracle import recurrent_oracle as O
from tests.test_gpu_recurrent import CONV_IN, NORM_IN, TYPES, _reference, _within, check_scan, norm_problem, run_conv, run_norm, run_scan, scan_problem

pytestmark = pytest.mark.gpu


def _code(kind):
    from rnn_train_ring_attractor_amd import _lib
    return _lib.load(), _lib.SEQUENCE_TYPES[TYPES[kind]]


# ------------------------------------------------------------------------------------------------
# Convolution
# ------------------------------------------------------------------------------------------------
def conv_by_taps(x, weight, bias, start, lengths, silu):
    """fp64, all tokens at once: (pre-activation or its silu, zero behind the lengths; the last K - 1 inputs)"""
    B, T, _ = x.shape
    K = weight.shape[1]
    row = torch.cat([start, x], dim=1)
    p = bias + sum(weight[:, k] * row[:, k:k + T] for k in range(K))
    p = O.silu(p) if silu else p
    counts = (torch.arange(T, device=x.device)[None, :] < torch.tensor(lengths, device=x.device)[:, None])[..., None]
    return torch.where(counts, p, torch.zeros_like(p)), torch.stack([row[b, n:n + K - 1] for b, n in enumerate(lengths)])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("C", [4, 3])
@pytest.mark.parametrize("K", [2, 3, 4, 5, 8])
def test_conv_in_long_pieces(K, C, kind, gpu_device):
    """So many tokens that every thread's piece has at least 24: what is done without conditions in the middle of a piece needs three times eight.  x and the
    gradient are positive, so that a weight's gradient is near its terms' size and a token left out of every piece shows."""
    lib, code = _code(kind)
    B, T = 3, 1_450_001
    parts = lib.ringattr_causal_conv_bwd_workspace_bytes(code, B, T, C, K, 1) // (4 * C * (K + 1))
    piece = B * T / (parts * 256)                # (a workgroup takes at most 256 pieces)
    assert piece >= 24
    lengths = [T, T - 12345, 70_007]
    gen = torch.Generator(device=gpu_device).manual_seed(41)
    dtype = TYPES[kind]
    r = lambda *s: torch.randn(*s, generator=gen, device=gpu_device)
    rows = lambda *s: r(*s).abs().add(0.25).to(dtype)
    p = {"x": rows(B, T, C), "weight": r(C, K), "bias": r(C), "start": rows(B, K - 1, C), "dy": rows(B, T, C), "de": rows(B, K - 1, C)}
    for b, n in enumerate(lengths):
        p["x"][b, n:] = math.nan
        p["dy"][b, n:] = math.nan
    clean = {n: t.nan_to_num().double() for n, t in p.items()}
    for act in (None, "silu"):
        print(f"[case] long conv {K} {C} {kind} {act} {piece:.0f}", flush=True)
        got = run_conv(p, dtype, gpu_device, lengths, act)
        call = lambda *t: conv_by_taps(*t, lengths, act == "silu")
        outs, grads = _reference(call, [clean[n] for n in CONV_IN], [clean["dy"], clean["de"]])
        big = [clean[n].abs() for n in CONV_IN]
        pre = conv_by_taps(*big, lengths, False)[0]
        _, sizes = _reference(lambda *t: conv_by_taps(*t, lengths, False), big, [clean["dy"] * (1 + pre) if act else clean["dy"], clean["de"]])
        assert torch.equal(got["state"].double(), outs[1])
        adds = 256 + B * T / parts + parts       # (a piece's tokens are fewer than a workgroup's)
        for n, want, size in zip(("y", *("d" + n for n in CONV_IN)), (outs[0], *grads), (pre, *sizes)):
            _within(n, got[n], want.cpu(), size.cpu(), 2 * (K + 1 + 16) + (min(adds, 256 + 256 + parts) if n in ("dweight", "dbias") else 0))


# ------------------------------------------------------------------------------------------------
# Norm
# ------------------------------------------------------------------------------------------------
# (rows, values, group): a row of over 1024 values has a workgroup; one of 96 or 500 shares it with up to 31 others.  Rows that are read 16 bytes at a time and
# value by value, whose weights are kept and not, of 512 and 1024 threads
LONG = [(1541, 2048, None), (1541, 2048, 256), (1541, 2047, None), (1030, 8192, None), (1030, 8112, 1352), (1030, 8190, 65), (1030, 8191, None), (1030, 4100, 820), (40001, 96, 32),
        (40003, 500, 100)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,C,group", LONG, ids=[f"{a}x{b}-{c}" for a, b, c in LONG])
def test_norm_of_more_rows_than_workgroups(rows, C, group, kind, gpu_device):
    """Backwards each workgroup walks several rows, the last ones not all there."""
    lib, code = _code(kind)
    parts = lib.ringattr_norm_gate_bwd_workspace_bytes(code, rows, C, group or C, 1) // (4 * 3 * C)
    assert rows > 2 * parts * (1 if C > 1024 else 32) and rows % parts
    for form, act in (("rms", "silu"), ("layer", "sigmoid")):
        print(f"[case] long norm {rows} {C} {group} {kind} {form}", flush=True)
        p = norm_problem(43, (rows,), C, TYPES[kind])
        p["dy"], p["dn"] = p["dy"].abs(), p["dn"].abs()
        p = {n: t.to(gpu_device) for n, t in p.items()}
        got = run_norm(p, TYPES[kind], gpu_device, group=group, kind=form, activation=act)
        ins = [p[n] for n in NORM_IN]
        outs, grads = _reference(lambda *t: O.norm_gate(*t, group, 1e-5, form, act), ins, [p["dy"], p["dn"]])
        size = O.norm_sizes(*ins, group, 1e-5, form, act, p["dy"], p["dn"])
        K, adds = 2 * (group or C) + 2 * C + 64, math.ceil(rows / parts) + 32 + parts
        for n, want in zip(("y", "n", *("d" + n for n in NORM_IN)), (*outs, *grads)):
            _within(n, got[n], want.cpu(), size[n].cpu(), K + (adds if n in ("dweight", "dscale", "dnext_weight") else 0))


# ------------------------------------------------------------------------------------------------
# Scan
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("sizes", [(2, 31, 64, 16, 1), (1, 150, 24, 8, 3), (3, 95, 10, 5, 2), (1, 133, 40, 33, 1)], ids=lambda s: "x".join(map(str, s)))
def test_scan_of_steps_as_they_are(sizes, kind, gpu_device):
    """softplus=False with a decay, gate and bias: positive steps, and small ones of both signs."""
    for scale, sign in ((0.2, False), (0.03, True)):
        print(f"[case] steps {sizes} {kind} {scale}", flush=True)
        p = scan_problem(47, *sizes, TYPES[kind])
        p["delta"] = (scale * (p["delta"] if sign else p["delta"].abs())).to(TYPES[kind]).double()
        p["bias"] = (0.01 * (p["bias"] + 3)).float().double() if sign else (0.1 * (p["bias"] + 3).abs()).float().double()
        lengths = [sizes[1] - 3 * b for b in range(sizes[0])]
        check_scan(p, run_scan(p, TYPES[kind], gpu_device, lengths, False), lengths, False)


# ------------------------------------------------------------------------------------------------
# Gradients against differences
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("name", ["conv", "scan", "norm"])
def test_gradients_are_differences_along_themselves(name, gpu_device):
    """fp32, along the gradient itself and along a random half of it, where the derivative is the gradient's norm (that half's): central differences of steps h and
    h / 2 put together to fourth order, h = 1/4 along a direction of norm one, 1/64 for the scan's A, whose powers bend most.  The truncation, taken from the
    same differences of the oracle in 64 bits, is below 2e-5 of the derivative.  The value is a sum of n results of size one, each off by less than 400 2^-24 (the
    counts above) and of any sign: together 400 2^-24 sqrt(n), which the two steps make 1.9 / h times as much, 1.8e-4 sqrt(n) and 2.9e-3 for A; derivatives are, by
    the oracle, above 0.03 sqrt(n) and 0.19 for A: 6e-3 and 1.5e-2 of them.  So 2e-2, and a gradient a tenth too large or small is off by five times that."""
    from tests.test_gpu_recurrent_use import _operators
    call, tensors = _operators(gpu_device)[name]
    tensors = [t * 0.5 for t in tensors]
    leaves = [t.clone().requires_grad_(True) for t in tensors]
    out = call(*leaves)
    gen = torch.Generator(device=gpu_device).manual_seed(53)
    given = [torch.randn(o.shape, generator=gen, device=gpu_device) for o in out]
    grads = torch.autograd.grad(out, leaves, given)
    value = lambda ts: sum(float((o.double() * g.double()).sum()) for o, g in zip(call(*ts), given))
    for i, t in enumerate(tensors):
        for half in (False, True):
            print(f"[case] difference along itself {name} {i} {half}", flush=True)
            d = grads[i].double()
            if half:
                d = d * (torch.rand(d.shape, generator=gen, device=gpu_device) < 0.5)
            want = float(d.norm())
            d = d / want

            def difference(h):
                with torch.no_grad():
                    more, less = ((t.double() + s * d).float() for s in (h, -h))
                    return (value([*tensors[:i], more, *tensors[i + 1:]]) - value([*tensors[:i], less, *tensors[i + 1:]])) / (2 * h)

            h = 2.0 ** -6 if (name, i) == ("scan", 2) else 2.0 ** -2
            num = (4 * difference(h / 2) - difference(h)) / 3
            for factor, fits in ((1.0, True), (1.1, False), (0.9, False)):
                assert (abs(num - factor * want) <= 2e-2 * want) == fits, (i, half, factor, num, want)


# ------------------------------------------------------------------------------------------------
# What is not finite
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", list(TYPES))
def test_nan_reaches_gradients_of_its_group_and_sequence_only(kind, gpu_device):
    """NaN in x, the step or the gate of one channel at a token: gradients of B and C of another group, of another sequence, and of B behind the token (of C in
    front of it; for the gate, which no state sees, anywhere but at the token) are what they are without."""
    dtype, T, C, N = TYPES[kind], 70, 20, 5
    for at in (0, 33, T - 1):
        p = scan_problem(33, 2, T, C, N, 2, dtype)
        clean = run_scan(p, dtype, gpu_device)
        for n in ("x", "delta", "z"):
            print(f"[case] NaN in {n} at {at} {kind}", flush=True)
            bad = {m: None if t is None else t.clone() for m, t in p.items()}
            bad[n][0, at, 3] = math.nan
            got = run_scan(bad, dtype, gpu_device)
            seen = {m: torch.zeros(2, T, 2, N, dtype=torch.bool, device=gpu_device) for m in ("dB", "dC")}
            # (an x or a step that is NaN is in the states from there on; the adjoint sees the step on the way to what is in front, the gate likewise)
            seen["dB"][0, at:at + 1 if n == "x" else 0, 0] = True
            if n != "x":
                seen["dB"][0, :at + 1, 0] = True
            seen["dC"][0, at:at + 1 if n == "z" else T, 0] = True
            for m in ("dB", "dC"):
                assert torch.equal(got[m][~seen[m]], clean[m][~seen[m]]), (n, m)
                assert torch.isnan(got[m][0, at, 0]).all(), (n, m)


@pytest.mark.parametrize("kind", list(TYPES))
def test_norm_of_gates_that_are_not_finite(kind, gpu_device):
    """NaN in a gate is NaN in y and, where the activation has a slope that depends on it, in the gate's own gradient, and the rest of the row is what it is without; a
    sigmoid of an infinite gate is one or zero, and its gradient zero."""
    dtype, C = TYPES[kind], 24
    for act in ("silu", "sigmoid", None):
        for value in (math.nan, math.inf, -math.inf):
            if act != "sigmoid" and not math.isnan(value):
                continue
            print(f"[case] gate {value} {act} {kind}", flush=True)
            p = norm_problem(59, (3,), C, dtype, next=False)
            clean = run_norm(p, dtype, gpu_device, group=8, activation=act)
            p["gate"][1, 5] = value
            got = run_norm(p, dtype, gpu_device, group=8, activation=act)
            rest = torch.ones(3, C, dtype=torch.bool, device=gpu_device)
            rest[1, 5] = False
            for n in ("y", "dgate"):
                assert torch.equal(got[n][rest], clean[n][rest]), (n, act, value)
                if math.isnan(value) and (n == "y" or act is not None):
                    assert torch.isnan(got[n][1, 5]), (n, act)
            if math.isnan(value):
                assert torch.isnan(got["dx"][1, :8]).all() and torch.equal(got["dx"][1, 8:], clean["dx"][1, 8:])
            else:
                p["gate"][1, 5] = 1e4 * math.copysign(1, value)
                want = run_norm(p, dtype, gpu_device, group=8, activation=act)
                assert all(torch.allclose(got[n], want[n], rtol=0, atol=1e-30) for n in ("y", "dgate", "dx"))


# ------------------------------------------------------------------------------------------------
# States over the borders of segments
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("A", [1.0, -1.0])
@pytest.mark.parametrize("what", ["nothing", "little", "much"])
def test_scan_across_powers_that_no_float_holds(what, A, kind, gpu_device):
    """Steps of one (of minus one, for a negative A that grows): over a segment of 96 tokens a state's power is e^96 or e^-96, which is infinite or zero in 32 bits.  A state of
    nothing stays nothing under it and 2^-100 becomes a number, as they do token by token; 2^100 under a negative A fades to one.  The same for the adjoint: inputs start
    behind the tokens whose outputs' gradients count, so that neither grows out of range.  Alone, and as one of 300 sequences, which are not cut."""
    dtype = TYPES[kind]
    for grows, T in ((True, 200), (False, 130)):
        step = 1.0 if (A > 0) == grows else -1.0
        if (what == "much") == grows:
            continue
        print(f"[case] powers {what} {A} {kind} {T}", flush=True)
        p = scan_problem(61, 1, T, 10, 5, 1, dtype, gate=False)
        first = {"nothing": 0.0, "little": 2.0 ** -100, "much": 2.0 ** 100}[what]
        p["A"], p["delta"], p["bias"] = torch.full_like(p["A"], A), torch.full_like(p["delta"], step), None
        late, early = (150, 50) if grows else (T, 0)
        p["x"][:, :late], p["dy"][:, early:] = 0, 0
        p["start"], p["de"] = first * p["start"].sign(), first * p["de"].sign()
        if grows and what == "little":           # (2^-100 e^200 is a number no longer: both end where x begins)
            T = 150
            p = {n: t[:, :T].contiguous() if n in ("x", "delta", "B", "C", "dy") else t for n, t in p.items()}
        got = run_scan(p, dtype, gpu_device, None, False)
        check_scan(p, got, None, False)
        shared = ("A", "D")
        many = run_scan({n: t if t is None or n in shared else t.expand(300, *t.shape[1:]) for n, t in p.items()}, dtype, gpu_device, None, False)
        size, total = O.scan_sizes(*(p[n] for n in ("x", "delta", "A", "B", "C", "D", "z", "bias", "start")), None, False, p["dy"], p["de"])
        for n in ("y", "state", "dx", "ddelta", "dB", "dC", "dstart"):
            assert torch.equal(many[n][299], many[n][0])
            a, b = got[n][0].double().cpu(), many[n][0].double().cpu()
            assert ((a - b).abs() <= torch.finfo(got[n].dtype).eps * b.abs() + 2 * (3 * T + 13 * total + 100) * 2.0 ** -24 * size[n][0] + 1e-37 + 1e-30 * (dtype == torch.float16))[
                torch.isfinite(b)].all() and (torch.isfinite(a) == torch.isfinite(b)).all(), n


# ------------------------------------------------------------------------------------------------
# Single tokens of large batches
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,C,N,G", [(8192, 2048, 16, 1), (8192, 1024, 2, 1024), (16384, 2048, 33, 2)])
def test_tokens_of_more_channels_than_sequences_take(B, C, N, G, gpu_device):
    """More than 16000000 channels of all sequences, up to a thread count of 2^31: the bits of calls of 2048 sequences each."""
    from rnn_train_ring_attractor_amd import causal_conv_step, selective_scan_step
    gen = torch.Generator(device=gpu_device).manual_seed(67)
    r = lambda *s: torch.randn(*s, generator=gen, device=gpu_device)
    print(f"[case] tokens {B} {C} {N} {G}", flush=True)
    with torch.no_grad():
        x, Bm, A, w, bias, D = r(B, C).bfloat16(), r(B, G, N).bfloat16(), -r(C, N).exp(), r(C, 4), r(C), r(C)
        for state, step in ((r(B, 3, C).bfloat16(), lambda at, s: causal_conv_step(x[at], w, s, bias=bias, activation="silu")),
                            (r(B, C, N), lambda at, s: selective_scan_step(x[at], x[at], A, Bm[at], Bm[at], s, D=D, z=x[at], delta_bias=bias, softplus=True))):
            parts, rows = [], state.clone()
            for at in range(0, B, 2048):
                parts.append(step(slice(at, at + 2048), rows[at:at + 2048]))
            assert torch.equal(step(slice(None), state), torch.cat(parts)) and torch.equal(state, rows)


# ------------------------------------------------------------------------------------------------
# Rows that lie on each other
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("name", ["conv", "scan", "norm"])
def test_rows_that_overlap_and_one_tensor_twice(name, kind, gpu_device):
    """Inputs and gradients that are one token's values for all tokens, or windows that move up by eight values a token, the same memory in several places: the results of their
    copies.  (Rows' results to the bit, each place's gradient by itself, as autograd adds them in an order of its own; a parameter's sums in another order, up to the counts above.)"""
    from rnn_train_ring_attractor_amd import causal_conv_func, norm_gate_func, selective_scan_func
    gen = torch.Generator(device=gpu_device).manual_seed(71)
    B, T, C, N = 2, 75, 64, 16
    r = lambda *s: torch.randn(*s, generator=gen, device=gpu_device)
    w, A, D, n = r(C, 4), -r(C, N).exp(), r(C), r(C)
    whole = lambda x: x
    ops = {"conv": (lambda x, w, D: causal_conv_func(x, w, D, activation="silu"), (whole,), (w, D)),
           "scan": (lambda x, d, z, Bm, Cm, A, D: selective_scan_func(x, d, A, Bm, Cm, D=D, z=z, softplus=True),
                    (whole, whole, whole, lambda x: x[..., None, :N], lambda x: x[..., None, N:2 * N]), (A, D)),
           "norm": (lambda x, g, e, n, D: norm_gate_func(x, n, gate=g, residual=e, scale=D), (whole, whole, whole), (n, D))}
    call, places, params = ops[name]
    flat = r(B * (8 * T + C)).to(TYPES[kind])
    for what, x in (("one token", flat[:B * C].view(B, 1, C).expand(B, T, C)), ("windows", flat.as_strided((B, T, C), (8 * T + C, 8, 1))), ("one value", flat[:1].view(1, 1, 1).expand(B, T, C))):
        print(f"[case] overlap {name} {kind} {what}", flush=True)
        results = []
        for lie in (x, x.contiguous()):
            leaves = [*(of(lie).detach().requires_grad_(True) for of in places), *(p.clone().requires_grad_(True) for p in params)]
            y = call(*leaves)
            results.append((y.detach(), *torch.autograd.grad(y, leaves, lie)))
        rows = 1 + len(places)
        assert all(torch.equal(a, b) for a, b in zip(results[0][:rows], results[1][:rows])), what
        for a, b in zip(results[0][rows:], results[1][rows:]):
            assert torch.allclose(a, b, rtol=0, atol=2 * (B * T + 256) * 2.0 ** -24 * float((a.abs().max() + b.abs().max()) * 64)), what
