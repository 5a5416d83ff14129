"""The recurrent layer's operators on the GPU against their definitions in 64 bits (oracle/recurrent_oracle.py).

Bounds.  A result is rounded once to its type, half a step: eps / 2 |y|.  What is computed on the way is fp32 and is bounded against the
result's size, the same formula over its terms' magnitudes: K additions, products and functions of 2^-24 each.  K counts, for
the convolution: K + 1 terms of a pre-activation, 16 for silu and its slope, the same again behind it, and for a weight's gradient the tokens;
the scan: for every token a power (its own 2 half steps and the product with the state), for all of them together the exponents' errors, each (raw step's
                 magnitude + 12) half steps of it, the states, the channels of a group, 64 for softplus, gates and what is left, and for a parameter the tokens;
the norm: a mean over a group and one over the row, each twice (its sum, and the quotient it goes into), 64 for the functions, and for a weight the rows."""
import math

import pytest
import torch

from oracle import recurrent_oracle as O

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _within(name, got, want, size, K):
    got = got.detach()
    dtype, got = got.dtype, got.double().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    eps = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).tiny * 2.0 ** -9 if dtype == torch.float16 else 1e-37
    bound = eps * want.abs() + (1 + eps) * K * 2.0 ** -24 * size + tiny
    fits = want.abs() * (1 + eps) + bound < torch.finfo(dtype).max
    bad = ~((got - want).abs() <= bound) & fits
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} at {bad.nonzero()[0].tolist()}, worst {float(((got - want).abs() / bound)[fits].max()):.2f} of the bound"


def _rand(gen, *shape):
    return torch.randn(*shape, generator=gen, dtype=torch.float64)


def _place(t, major):
    """The same values in [T,B,..] order, or as a slice of a wider tensor."""
    if major == "time":
        return t.transpose(0, 1).contiguous().transpose(0, 1)
    if major == "slice":
        wide = torch.full((*t.shape[:-1], t.shape[-1] + 24), math.nan, dtype=t.dtype, device=t.device)
        wide[..., 8:8 + t.shape[-1]] = t
        return wide[..., 8:8 + t.shape[-1]]
    return t


def _grads(outs, leaves, given):
    wanted = [t for t in leaves if t is not None]
    got = iter(torch.autograd.grad(outs, wanted, given, allow_unused=True))
    return [None if t is None else next(got) for t in leaves]


def _reference(call, leaves, given):
    """call(*leaves) -> outputs; their values and gradients in 64 bits"""
    leaves = [None if t is None else t.clone().requires_grad_(True) for t in leaves]
    outs = call(*leaves)
    grads = _grads(list(outs), leaves, given)
    return [o.detach() for o in outs], [None if t is None else torch.zeros_like(t) if g is None else g for t, g in zip(leaves, grads)]


# ------------------------------------------------------------------------------------------------
# Convolution
# ------------------------------------------------------------------------------------------------
def conv_problem(seed, B, T, C, K, dtype, start=True, bias=True):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: _rand(gen, *s).to(dtype).double()
    p = {"x": r(B, T, C), "weight": _rand(gen, C, K).float().double(), "bias": _rand(gen, C).float().double() if bias else None,
         "start": r(B, K - 1, C) if start else None, "dy": r(B, T, C), "de": r(B, K - 1, C)}
    return p


CONV_IN = ("x", "weight", "bias", "start")


def run_conv(p, dtype, dev, lengths=None, act=None, place="batch"):
    from rnn_train_ring_attractor_amd import causal_conv_func
    kinds = {"weight": torch.float32, "bias": torch.float32}
    leaves = [None if p[n] is None else _place(p[n].to(kinds.get(n, dtype)).to(dev), place if n == "x" else "batch").detach().requires_grad_(True) for n in CONV_IN]
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=dev)
    y, end = causal_conv_func(leaves[0], leaves[1], leaves[2], initial_state=leaves[3], lengths=lens, activation=act, return_state=True)
    grads = _grads([y, end], leaves, [_place(p["dy"].to(dtype).to(dev), place), p["de"].to(dtype).to(dev)])
    return dict(zip(("y", "state", *("d" + n for n in CONV_IN)), (y, end, *grads)))


def check_conv(p, got, lengths, act):
    clean = {n: None if t is None else t.nan_to_num() for n, t in p.items()}
    outs, grads = _reference(lambda *t: O.conv(*t, lengths, act), [clean[n] for n in CONV_IN], [clean["dy"], clean["de"]])
    want = dict(zip(("y", "state", *("d" + n for n in CONV_IN)), (*outs, *grads)))
    size = O.conv_sizes(*(clean[n] for n in CONV_IN), lengths, act, clean["dy"], clean["de"])
    B, T, _ = p["x"].shape
    K = p["weight"].shape[1]
    assert torch.equal(got["state"].double().cpu(), want["state"])
    for n in want:
        if want[n] is not None and n != "state":
            _within(n, got[n], want[n], size[n], 2 * (K + 1 + 16) + (B * T if n in ("dweight", "dbias") else 0))


CONV = [(1, 1, 1, 1), (1, 1, 1, 4), (2, 5, 3, 2), (1, 2, 8, 4), (3, 33, 24, 3), (2, 70, 33, 4), (1, 300, 64, 8), (2, 129, 520, 5), (1, 40, 1032, 4), (1, 17, 7, 7),
        (5, 9, 96, 6)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("sizes", CONV, ids=["x".join(map(str, s)) for s in CONV])
def test_conv_and_its_gradients(sizes, kind, gpu_device):
    for act in (None, "silu"):
        print(f"[case] conv {sizes} {kind} {act}", flush=True)
        p = conv_problem(3, *sizes, TYPES[kind], start=sizes[1] % 2 == 1, bias=sizes[3] != 5)
        check_conv(p, run_conv(p, TYPES[kind], gpu_device, act=act), None, act)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("K", range(1, 9))
def test_conv_with_every_number_of_taps(K, kind, gpu_device):
    for C in (16, 5):                            # rows of whole units of 16 bytes, and not
        for act in (None, "silu"):
            print(f"[case] conv taps {C} {K} {kind} {act}", flush=True)
            p = conv_problem(7, 2, 19, C, K, TYPES[kind])
            check_conv(p, run_conv(p, TYPES[kind], gpu_device, act=act), None, act)


@pytest.mark.parametrize("place", ["time", "slice"])
@pytest.mark.parametrize("kind", list(TYPES))
def test_conv_of_padded_batches(kind, place, gpu_device):
    """Lengths from none to all; rows behind a length hold NaN and are not read."""
    T = 150
    for C, K in ((40, 4), (13, 3), (16, 8)):
        lengths = [T, 0, 1, 2, 63, 64, 65, 149]
        p = conv_problem(5, len(lengths), T, C, K, TYPES[kind])
        for b, n in enumerate(lengths):
            p["x"][b, n:] = math.nan
            p["dy"][b, n:] = math.nan
        print(f"[case] padded conv {C} {K} {kind} {place}", flush=True)
        got = run_conv(p, TYPES[kind], gpu_device, [T + 9, -3] + lengths[2:], "silu", place)
        check_conv(p, got, lengths, "silu")
        for b, n in enumerate(lengths):
            assert (got["y"][b, n:] == 0).all() and (got["dx"][b, n:] == 0).all()


@pytest.mark.parametrize("kind", list(TYPES))
def test_conv_token_by_token(kind, gpu_device):
    """What a sequence gives, and the state that it leaves, token by token; places that wait stay as they are."""
    from rnn_train_ring_attractor_amd import causal_conv_func, causal_conv_step
    dtype = TYPES[kind]
    for B, T, C, K in ((1, 6, 8, 4), (3, 9, 129, 3), (2, 10, 64, 8), (2, 3, 5, 1)):
        print(f"[case] conv tokens {B} {T} {C} {K} {kind}", flush=True)
        p = conv_problem(7, B, T, C, K, dtype)
        x, start = p["x"].to(dtype).to(gpu_device), p["start"].to(dtype).to(gpu_device)
        w, bias = p["weight"].float().to(gpu_device), p["bias"].float().to(gpu_device)
        with torch.no_grad():
            want, end = causal_conv_func(x, w, bias, initial_state=start, activation="silu", return_state=True)
            state = start.clone()
            wide = torch.cat([x, x], dim=2)
            got = torch.stack([causal_conv_step(wide[:, t, C:], w, state, bias=bias, activation="silu") for t in range(T)], dim=1)
            assert torch.equal(got, want) and torch.equal(state, end)
            active = torch.arange(B, device=gpu_device) % 2 == 0
            y = causal_conv_step(x[:, 0], w, state, bias=bias, active=active, activation="silu")
            assert (y[~active] == 0).all() and torch.equal(state[~active], end[~active])
            if K > 1:
                assert torch.equal(state[active][:, -1], x[active][:, 0])


# ------------------------------------------------------------------------------------------------
# Scan
# ------------------------------------------------------------------------------------------------
SCAN_IN = ("x", "delta", "A", "B", "C", "D", "z", "bias", "start")


def scan_problem(seed, batch, T, channels, N, G, dtype, gate=True, skip=True, bias=True, start=True):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: _rand(gen, *s).to(dtype).double()
    f = lambda t: t.float().double()
    return {"x": r(batch, T, channels), "delta": r(batch, T, channels), "A": f(-torch.exp(_rand(gen, channels, N))), "B": r(batch, T, G, N), "C": r(batch, T, G, N),
            "D": f(_rand(gen, channels)) if skip else None, "z": r(batch, T, channels) if gate else None, "bias": f(_rand(gen, channels) - 3) if bias else None,
            "start": f(_rand(gen, batch, channels, N)) if start else None, "dy": r(batch, T, channels), "de": f(_rand(gen, batch, channels, N))}


def run_scan(p, dtype, dev, lengths=None, plus=True, place="batch"):
    from rnn_train_ring_attractor_amd import selective_scan_func
    kinds = {n: torch.float32 for n in ("A", "D", "bias", "start")}
    leaves = [None if p[n] is None else _place(p[n].to(kinds.get(n, dtype)).to(dev), "batch" if n in kinds else place).detach().requires_grad_(True) for n in SCAN_IN]
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=dev)
    x, delta, A, B, C, D, z, bias, start = leaves
    y, end = selective_scan_func(x, delta, A, B, C, D=D, z=z, delta_bias=bias, initial_state=start, lengths=lens, softplus=plus, return_state=True)
    grads = _grads([y, end], leaves, [_place(p["dy"].to(dtype).to(dev), place), p["de"].float().to(dev)])
    return dict(zip(("y", "state", *("d" + n for n in SCAN_IN)), (y, end, *grads)))


def check_scan(p, got, lengths, plus):
    clean = {n: None if t is None else t.nan_to_num() for n, t in p.items()}
    ins = [clean[n] for n in SCAN_IN]
    outs, grads = _reference(lambda *t: O.scan(*t, lengths, plus), ins, [clean["dy"], clean["de"]])
    want = dict(zip(("y", "state", *("d" + n for n in SCAN_IN)), (*outs, *grads)))
    size, total = O.scan_sizes(*ins, lengths, plus, clean["dy"], clean["de"])
    batch, T, channels = p["x"].shape
    N, G = p["A"].shape[1], p["B"].shape[2]
    raw = float((clean["delta"].abs() + (0 if clean["bias"] is None else clean["bias"].abs())).max())
    K = 3 * T + (raw + 12) * total + N + channels // G + 64
    for n in want:
        if want[n] is not None:
            _within(n, got[n], want[n], size[n], K + (batch * T if n in ("dA", "dD", "dbias") else 0))


SCAN = [(1, 1, 1, 1, 1), (2, 3, 5, 2, 1), (1, 16, 16, 4, 1), (1, 17, 24, 8, 3), (2, 31, 64, 16, 1), (1, 32, 66, 16, 2), (1, 33, 130, 5, 1), (2, 20, 40, 11, 4),
        (1, 48, 72, 32, 1), (1, 40, 33, 20, 3), (2, 18, 34, 64, 2), (1, 21, 15, 47, 1), (3, 95, 8, 16, 1)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("sizes", SCAN, ids=["x".join(map(str, s)) for s in SCAN])
def test_scan_and_its_gradients(sizes, kind, gpu_device):
    for k, (gate, skip, bias, start, plus) in enumerate(((True, True, True, True, True), (False, False, False, False, True), (True, False, True, False, True))):
        print(f"[case] scan {sizes} {kind} {k}", flush=True)
        p = scan_problem(11 + k, *sizes, TYPES[kind], gate, skip, bias, start)
        check_scan(p, run_scan(p, TYPES[kind], gpu_device, plus=plus), None, plus)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 48, 63, 64])
def test_scan_with_every_number_of_states(N, kind, gpu_device):
    """Every number of states a lane and waves a channel, in rows of whole units of 16 bytes and not, over one segment and several."""
    for channels, G, T in ((40, 1, 133), (24, 3, 45), (10, 2, 133)):
        print(f"[case] scan states {channels} {N} {G} {T} {kind}", flush=True)
        p = scan_problem(21, 2, T, channels, N, G, TYPES[kind])
        check_scan(p, run_scan(p, TYPES[kind], gpu_device), None, True)


@pytest.mark.parametrize("place", ["time", "slice"])
@pytest.mark.parametrize("kind", list(TYPES))
def test_scan_of_padded_batches(kind, place, gpu_device):
    """Lengths from none to all, over several segments; rows behind a length hold NaN and are not read."""
    T = 150
    for channels, N, G in ((16, 16, 1), (9, 3, 3), (24, 40, 2)):
        lengths = [T, 0, 1, 15, 16, 17, 64, 149]
        p = scan_problem(13, len(lengths), T, channels, N, G, TYPES[kind])
        for b, n in enumerate(lengths):
            for name in ("x", "delta", "B", "C", "z", "dy"):
                p[name][b, n:] = math.nan
        print(f"[case] padded scan {channels} {N} {G} {kind} {place}", flush=True)
        got = run_scan(p, TYPES[kind], gpu_device, [T + 9, -3] + lengths[2:], True, place)
        check_scan(p, got, lengths, True)
        for name in ("y", "dx", "ddelta", "dB", "dC", "dz"):
            assert all((got[name][b, n:] == 0).all() for b, n in enumerate(lengths)), name


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("sizes", [(3, 333, 70, 16, 2), (2, 700, 20, 7, 1), (1, 1030, 16, 33, 1), (9, 100, 64, 24, 1)], ids=lambda s: "x".join(map(str, s)))
def test_scan_sums_of_small_whole_numbers_are_exact(sizes, kind, gpu_device):
    """Without decay (A zero), steps of one and rows of -1, 0 and 1: states (below 2^10) and their sums are whole numbers that every step holds, so each
    result is the sum rounded once, and a token too many or too few shows, across chunks and segments."""
    batch, T, channels, N, G = sizes
    print(f"[case] whole numbers {sizes} {kind}", flush=True)
    gen = torch.Generator().manual_seed(17)
    whole = lambda *s: torch.randint(-1, 2, s, generator=gen).double()
    p = {"x": whole(batch, T, channels), "delta": torch.ones(batch, T, channels, dtype=torch.float64), "A": torch.zeros(channels, N, dtype=torch.float64),
         "B": whole(batch, T, G, N), "C": whole(batch, T, G, N), "D": whole(channels), "z": None, "bias": None, "start": whole(batch, channels, N),
         "dy": whole(batch, T, channels), "de": whole(batch, channels, N)}
    lengths = [T, 0, T - 1, T // 2, 1, 33, 64, 65, 32][:batch] if batch > 1 else [T - 3]
    got = run_scan(p, TYPES[kind], gpu_device, lengths, False)
    outs, grads = _reference(lambda *t: O.scan(*t, lengths, False), [p[n] for n in SCAN_IN], [p["dy"], p["de"]])
    for n, want in zip(("y", "state", *("d" + n for n in SCAN_IN)), (*outs, *grads)):
        if want is None:
            continue
        exact = want.round()
        assert (exact - want).abs().max() < 1e-6 and exact.abs().max() < 2 ** 24
        if n == "ddelta" or exact.abs().max() < 60000:
            assert torch.equal(got[n].double().cpu(), exact.to(got[n].dtype).double()), n


@pytest.mark.parametrize("kind", list(TYPES))
def test_scan_token_by_token(kind, gpu_device):
    """Goes on from a sequence's state: outputs within both roundings, the state within those of the tokens."""
    from rnn_train_ring_attractor_amd import selective_scan_func, selective_scan_step
    dtype = TYPES[kind]
    for batch, T, channels, N, G in ((1, 6, 8, 16, 1), (3, 9, 130, 5, 2), (2, 5, 64, 64, 1), (2, 4, 6, 1, 3)):
        print(f"[case] scan tokens {batch} {T} {channels} {N} {G} {kind}", flush=True)
        p = scan_problem(19, batch, T, channels, N, G, dtype)
        t = {n: None if x is None else x.to(torch.float32 if n in ("A", "D", "bias", "start") else dtype).to(gpu_device) for n, x in p.items()}
        outs, _ = _reference(lambda *a: O.scan(*a, None, True), [p[n] for n in SCAN_IN], [p["dy"], p["de"]])
        size, total = O.scan_sizes(*(p[n] for n in SCAN_IN), None, True)
        K = 3 * T + (float((p["delta"].abs() + p["bias"].abs()).max()) + 12) * total + N + 64
        with torch.no_grad():
            half = T // 2
            y, state = selective_scan_func(t["x"][:, :half], t["delta"][:, :half], t["A"], t["B"][:, :half], t["C"][:, :half], D=t["D"], z=t["z"][:, :half],
                                           delta_bias=t["bias"], initial_state=t["start"], softplus=True, return_state=True)
            rows = [y] + [selective_scan_step(t["x"][:, i], t["delta"][:, i], t["A"], t["B"][:, i], t["C"][:, i], state, D=t["D"], z=t["z"][:, i],
                                              delta_bias=t["bias"], softplus=True)[:, None] for i in range(half, T)]
            _within("y", torch.cat(rows, dim=1), outs[0], size["y"], K)
            _within("state", state, outs[1], size["state"], K)
            before = state.clone()
            active = (torch.arange(batch, device=gpu_device) % 2 == 1).to(torch.uint8)
            y = selective_scan_step(t["x"][:, 0], t["delta"][:, 0], t["A"], t["B"][:, 0], t["C"][:, 0], state, active=active)
            rest = active == 0
            assert (y[rest] == 0).all() and torch.equal(state[rest], before[rest]) and (batch == 1 or not torch.equal(state, before))


# ------------------------------------------------------------------------------------------------
# Norm, gate, residual
# ------------------------------------------------------------------------------------------------
NORM_IN = ("x", "weight", "gate", "residual", "scale", "next_weight")


def norm_problem(seed, lead, C, dtype, gate=True, residual=True, scale=True, next=True):
    gen = torch.Generator().manual_seed(seed)
    r = lambda: (2 * _rand(gen, *lead, C)).to(dtype).double()
    w = lambda there: _rand(gen, C).float().double() if there else None
    return {"x": (r() + 1).to(dtype).double(), "weight": w(True), "gate": r() if gate else None, "residual": r() if residual else None, "scale": w(scale), "next_weight": w(next),
            "dy": r(), "dn": r()}


def run_norm(p, dtype, dev, place="batch", **how):
    from rnn_train_ring_attractor_amd import norm_gate_func
    leaves = [None if p[n] is None else _place(p[n].to(torch.float32 if p[n].dim() == 1 and n not in ("x", "gate", "residual") else dtype).to(dev), place
                                               if n in ("x", "gate", "residual") else "batch").detach().requires_grad_(True) for n in NORM_IN]
    x, weight, gate, residual, scale, nxt = leaves
    out = norm_gate_func(x, weight, gate=gate, residual=residual, scale=scale, next_weight=nxt, **how)
    out = list(out) if nxt is not None else [out]
    grads = _grads(out, leaves, [_place(p[n].to(dtype).to(dev), place) for n in ("dy", "dn")[:len(out)]])
    return dict(zip((*("y", "n")[:len(out)], *("d" + n for n in NORM_IN)), (*out, *grads)))


def check_norm(p, got, group, kind, act):
    ins = [p[n] for n in NORM_IN]
    C = p["x"].shape[-1]
    given = [p["dy"], p["dn"]][:1 if p["next_weight"] is None else 2]
    outs, grads = _reference(lambda *t: O.norm_gate(*t, group, 1e-5, kind, act), ins, given)
    want = dict(zip((*("y", "n")[:len(outs)], *("d" + n for n in NORM_IN)), (*outs, *grads)))
    size = O.norm_sizes(*ins, group, 1e-5, kind, act, p["dy"], p["dn"])
    K = 2 * (group or C) + 2 * C + 64
    for n in want:
        if want[n] is not None:
            _within(n, got[n], want[n], size[n], K + (p["x"].numel() // C if n in ("dweight", "dscale", "dnext_weight") else 0))


NORM = [((1,), 1, None), ((3,), 7, None), ((2, 5), 64, 16), ((33,), 96, 32), ((70,), 500, 100), ((9,), 520, None), ((2, 3, 4), 130, 5), ((600,), 24, 8), ((5,), 1032, 344),
        ((3,), 2048, None), ((4,), 4100, 820), ((2,), 8192, None), ((2,), 8190, 1638), ((2,), 8187, None), ((1100,), 8, None)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("lead,C,group", NORM, ids=[f"{'x'.join(map(str, a))}x{b}-{c}" for a, b, c in NORM])
def test_norm_and_its_gradients(lead, C, group, kind, gpu_device):
    for k, (gate, residual, scale, nxt, form, act) in enumerate(((True, True, True, True, "rms", "silu"), (False, False, False, False, "layer", None),
                                                                 (True, False, True, True, "layer", "sigmoid"), (True, True, False, False, "rms", None))):
        print(f"[case] norm {lead} {C} {group} {kind} {k}", flush=True)
        if form == "layer" and (C if group is None else group) == 1:
            continue                             # (a value less its own mean: nothing but rounding)
        p = norm_problem(23 + k, lead, C, TYPES[kind], gate, residual, scale, nxt)
        check_norm(p, run_norm(p, TYPES[kind], gpu_device, group=group, kind=form, activation=act), group, form, act)


@pytest.mark.parametrize("place", ["time", "slice"])
@pytest.mark.parametrize("kind", list(TYPES))
def test_norm_of_any_strides(kind, place, gpu_device):
    print(f"[case] norm strides {kind} {place}", flush=True)
    for C, group in ((64, 32), (33, 11)):
        p = norm_problem(29, (3, 7), C, TYPES[kind])
        check_norm(p, run_norm(p, TYPES[kind], gpu_device, place, group=group), group, "rms", "silu")


# rows whose groups ask for each number of units a thread, with and without whole units of 16 bytes
LIES = [(4096, 512), (4096, 256), (4096, 64), (8192, 512), (8184, 2728), (8184, 264), (8192, 256), (8188, 356), (8188, 92), (8192, 64), (8190, 2730), (8190, 63), (2047, None),
        (1023, 341), (255, None), (127, None)]


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("C,group", LIES, ids=[f"{a}-{b}" for a, b in LIES])
def test_norm_at_every_lie_of_its_rows(C, group, kind, gpu_device):
    print(f"[case] norm lies {C} {group} {kind}", flush=True)
    p = norm_problem(31, (3,), C, TYPES[kind])
    check_norm(p, run_norm(p, TYPES[kind], gpu_device, group=group, kind="layer", activation="silu"), group, "layer", "silu")
