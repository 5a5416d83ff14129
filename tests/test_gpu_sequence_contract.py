"""What the sequence operators' documentation promises, call by call, where the tests of their formulas do not look: how exact bf16 results are,
also without a returned state.

A bf16 result is a sum in fp32, rounded once: half a step, 2^-8 of it.  Each term of it passes an operand that is computed on the way and
enters a product as the sum of two bf16 numbers (a weight or a state: x cut off behind 8 bits, 2^-7 of it left, then that rounded, 2^-8 of
it: 2^-15), and, in a state that is no result, a decayed row in two rounded ones (2^-16); K additions and products in fp32, 2^-24 each.
The last three are bounded against the same sum over the terms' magnitudes."""
import math

import pytest
import torch

from tests.test_gpu_sequence import SEGMENTED, SHAPES, TYPES, _problem, _reference

pytestmark = pytest.mark.gpu


def _call(p, dtype, dev, lengths=None, state=True, scale=None):
    """linear_attention_func and its gradients; state: whether the final one is asked for (and has a gradient)."""
    from rnn_train_ring_attractor_amd import linear_attention_func
    leaves = [p[n].to(dtype).to(dev).requires_grad_(True) for n in ("q", "k", "v")]
    s0 = None if p["s0"] is None else p["s0"].float().to(dev).requires_grad_(True)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=dev)
    got = linear_attention_func(*leaves, p["g"].float().to(dev), initial_state=s0, lengths=lens, scale=scale, return_state=state)
    outs, given = ([*got], [p["do"].to(dtype).to(dev), p["ds"].float().to(dev)]) if state else ([got], [p["do"].to(dtype).to(dev)])
    grads = torch.autograd.grad(outs, leaves + ([] if s0 is None else [s0]), given)
    return dict(zip(["o", "state"][:len(outs)] + ["dq", "dk", "dv", "ds0"], [x.detach() for x in (*outs, *grads)]))


def _without_state_gradient(p):
    return {**p, "ds": torch.zeros_like(p["ds"])}


def _lengths(T, B, count):
    first = -(-(-(-T // 64)) // count) * 64
    return [first + 1, T, 0, first, 1, first - 1, T - 1, 65][:B]


def _bf16_bound(want, size, K):
    return 2.0 ** -8 * want.abs() + (1 + 2.0 ** -8) * (2.0 ** -15 + 2.0 ** -16 + K * 2.0 ** -24) * size + 1e-37


BF16 = [(s, 1) for s in SHAPES if s[1] > 1] + [(s, n) for k, s, n in SEGMENTED if k == "bf16"]


@pytest.mark.parametrize("state", [True, False], ids=["state", "no_state"])
@pytest.mark.parametrize("sizes,count", BF16, ids=["x".join(map(str, s)) for s, _ in BF16])
def test_bf16_results_carry_their_own_rounding(sizes, count, state, gpu_device):
    print(f"[case] bf16 {sizes} state={state}", flush=True)
    B, T, H, G, Dk, Dv = sizes
    p = _problem(43, *sizes, torch.bfloat16, start=T % 2 == 0)
    p = p if state else _without_state_gradient(p)
    lengths = _lengths(T, B, count) if count > 1 else None
    got, want, size = _call(p, torch.bfloat16, gpu_device, lengths, state), _reference(p, lengths), _reference(p, lengths, magnitudes=True)
    for name in ("o", "dq", "dk", "dv"):
        err = (got[name].double().cpu() - want[name]).abs()
        bound = _bf16_bound(want[name], size[name], T + Dk + Dv + H // G + 256)
        assert (err <= bound).all(), (name, float((err / bound).max()))
        if want[name].numel() >= 10000:
            # A rounding error is even within half a step of 2^-9 to 2^-8 of a value: of numbers of even logarithms the root mean square is
            # 2^-8 (3 / (8 ln 2) / 3) ** 0.5 = 0.00166 of theirs; a tenth more for numbers that are not
            rms = math.sqrt(float((err ** 2).sum() / (want[name] ** 2).sum()))
            print(f"[rms] {name} {rms:.5f}", flush=True)
            assert rms <= 1.1 * 0.00166, (name, rms)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("sizes,count", [((2, 333, 2, 1, 40, 72), 0)] + [(s, n) for _, s, n in SEGMENTED], ids=lambda x: "x".join(map(str, x)) if isinstance(x, tuple) else str(x))
def test_sums_of_small_whole_numbers_are_exact(sizes, count, kind, gpu_device):
    """Operands of -1, 0 and 1 without decay: weights, states (below 2^16) and sums (below 2^24) are whole numbers that every step holds, so
    each result is the sum rounded once, and a token too many or too few shows."""
    print(f"[case] whole numbers {sizes} {kind}", flush=True)
    B, T, H, G, Dk, Dv = sizes
    gen = torch.Generator().manual_seed(47)
    whole = lambda *s: torch.randint(-1, 2, s, generator=gen).double()
    p = {"q": whole(B, T, H, Dk), "k": whole(B, T, G, Dk), "v": whole(B, T, G, Dv), "do": whole(B, T, H, Dv), "g": torch.zeros(H, dtype=torch.float64),
         "s0": whole(B, H, Dk, Dv), "ds": whole(B, H, Dk, Dv)}
    lengths = _lengths(T, B, max(count, 2))
    got = _call(p, TYPES[kind], gpu_device, lengths, True, 1.0)
    want = _reference({**p, "q": p["q"] * Dk ** 0.5}, lengths)           # (the oracle's scale is Dk ** -0.5)
    want["dq"] = want["dq"] * Dk ** 0.5
    for name in want:
        exact = want[name].round()
        assert (exact - want[name]).abs().max() < 1e-6 and exact.abs().max() < 60000
        assert torch.equal(got[name].cpu(), exact.to(got[name].dtype)), name


# (sizes, lengths): ends inside chunks, heads whose dv and dk go back together and not, rows of whole 16 bytes and not, segments
PADDED = [((4, 90, 2, 1, 32, 48), [45, 90, 1, 33]), ((4, 90, 2, 2, 33, 47), [45, 90, 1, 70]), ((3, 70, 2, 1, 40, 72), [37, 70, 0]),
          ((2, 70, 1, 1, 256, 136), [41, 69]), ((4, 500, 2, 2, 20, 70), [70, 500, 0, 499]), ((4, 500, 2, 1, 70, 66), [129, 65, 3, 450])]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("sizes,lengths", PADDED, ids=["x".join(map(str, s)) for s, _ in PADDED])
def test_rows_behind_a_length_are_zero_whatever_the_others_hold(sizes, lengths, kind, gpu_device):
    """An infinity or NaN in a row that counts, in the initial state or in the final one's gradient leaves everything behind the lengths zero,
    and other sequences as they were."""
    dtype = TYPES[kind]
    p = _problem(53, *sizes, dtype, start=True)
    clean = _call(p, dtype, gpu_device, lengths)
    for name in ("q", "k", "v", "do", "s0", "ds"):
        for value in (math.inf, math.nan):
            for at in ((0,) if name in ("s0", "ds") else (0, lengths[0] - 1)):
                print(f"[case] {value} in {name} at {at} {sizes} {kind}", flush=True)
                bad = {n: (None if x is None else x.clone()) for n, x in p.items()}
                (bad[name][0] if name in ("s0", "ds") else bad[name][0, at])[..., 2] = value
                got = _call(bad, dtype, gpu_device, lengths)
                for n in ("o", "dq", "dk", "dv"):
                    assert all((got[n][b, m:] == 0).all() for b, m in enumerate(lengths)), n
                assert all(torch.equal(got[n][1:], clean[n][1:]) for n in got)
                assert not all(torch.isfinite(got[n][0]).all() for n in got)


@pytest.mark.parametrize("kind", list(TYPES))
def test_a_state_that_grows_in_a_short_chunk(kind, gpu_device):
    """A decay above one: powers of places behind a chunk's last token can pass fp32's range, those of its tokens do not."""
    dtype = TYPES[kind]
    for T, lengths in ((1, None), (3, None), (5, [5, 2]), (40, [3, 1])):
        print(f"[case] growing state {T} {lengths} {kind}", flush=True)
        p = _problem(59, 2, T, 2, 1, 16, 24, dtype, start=True, decays=[6.0, 0.5])
        got, want, size = _call(p, dtype, gpu_device, lengths), _reference(p, lengths), _reference(p, lengths, magnitudes=True)
        for name in want:
            half = 2.0 ** -24 if name in ("state", "ds0") else torch.finfo(dtype).eps / 2
            path = (2.0 ** -15 + 2.0 ** -16 if kind == "bf16" else 0.0) + (T + 16 + 24 + 2 + 256) * 2.0 ** -24
            err = (got[name].double().cpu() - want[name]).abs()
            fits = want[name].abs() * (1 + half) < torch.finfo(got[name].dtype).max
            assert (err <= half * want[name].abs() + (1 + half) * path * size[name] + 1e-7)[fits].all(), (name, T)


@pytest.mark.parametrize("sizes", [(2, 9, 3, 1, 5, 7), (1, 300, 1, 1, 5, 7)])
def test_states_at_any_address(sizes, gpu_device):
    """States and their gradients that are views into a larger tensor, off 16 bytes: the same bits."""
    from rnn_train_ring_attractor_amd import linear_attention_func
    print(f"[case] states at any address {sizes}", flush=True)
    B, T, H, G, Dk, Dv = sizes
    gen = torch.Generator(device=gpu_device).manual_seed(61)
    r = lambda *s: torch.randn(*s, generator=gen, device=gpu_device)
    q, k, v = r(B, T, H, Dk).requires_grad_(True), r(B, T, G, Dk).requires_grad_(True), r(B, T, G, Dv).requires_grad_(True)
    g, pool = -torch.rand(H, generator=gen, device=gpu_device), r(4, B, H, Dk, Dv)
    assert any(pool[i].data_ptr() % 16 for i in range(4))
    for i in range(4):
        ds = r(4, B, H, Dk, Dv)
        results = []
        for s0, d in ((pool[i], ds[i]), (pool[i].clone(), ds[i].clone())):
            s0 = s0.detach().requires_grad_(True)
            o, s = linear_attention_func(q, k, v, g, initial_state=s0, return_state=True)
            results.append([o, s, *torch.autograd.grad([o, s], [q, k, v, s0], [torch.ones_like(o), d])])
        assert all(torch.equal(a, b) for a, b in zip(*results))
    # autograd hands the pieces of a stacked gradient on as views
    s0 = pool[1].detach().requires_grad_(True)
    ends = [linear_attention_func(q, k, v, g, initial_state=s0, return_state=True)[1] for _ in range(3)]
    weights = r(3, B, H, Dk, Dv)
    together, = torch.autograd.grad((torch.stack(ends) * weights).sum(), [s0], retain_graph=True)
    alone = sum(torch.autograd.grad([e], [s0], [w.clone()], retain_graph=True)[0] for e, w in zip(ends, weights))
    assert torch.allclose(together, alone, rtol=1e-5, atol=1e-5)


def _entries(dev):
    from rnn_train_ring_attractor_amd import dropout_func, linear_attention_func, rotary_func
    gen = torch.Generator(device=dev).manual_seed(67)
    k, v, g = (torch.randn(2, 5, 2, d, generator=gen, device=dev) for d in (8, 6, 1))
    g = torch.tensor([-0.1, -0.5], device=dev)
    pos, f = torch.arange(5, device=dev), torch.rand(4, generator=gen, dtype=torch.float64, device=dev)
    return {"attention": lambda x: linear_attention_func(x, k, v, g), "rotary": lambda x: rotary_func(x, pos, f), "pair": lambda x: rotary_func((k, x), pos, f)[1],
            "dropout": lambda x: dropout_func(x, 0.3, 5, 6), "residual": lambda x: dropout_func(k, 0.3, 5, 6, residual=x)}, torch.randn(2, 5, 2, 8, generator=gen, device=dev)


@pytest.mark.parametrize("name", ["attention", "rotary", "pair", "dropout", "residual"])
def test_what_watches_the_operators_sees_them(name, gpu_device):
    """Forward mode and function transforms, which they have no rules for, are refused instead of losing the derivative; a trace records the call."""
    import torch.autograd.forward_ad as forward
    entries, x = _entries(gpu_device)
    op = entries[name]
    print(f"[case] watched {name}", flush=True)
    want = op(x)
    with forward.dual_level():
        assert torch.equal(op(x), want)                          # nothing of it is differentiated
        with pytest.raises(NotImplementedError, match="jvp"):
            op(forward.make_dual(x, torch.ones_like(x)))
    for transformed in (lambda: torch.func.jvp(op, (x,), (x,)), lambda: torch.func.vmap(op)(x[None]), lambda: torch.func.grad(lambda t: op(t).sum())(x)):
        with pytest.raises(RuntimeError):
            transformed()
    traced = torch.jit.trace(op, x)
    other = x.flip(0).contiguous() * 2
    for _ in range(2):
        assert torch.equal(traced(other), op(other))


def test_what_watches_a_single_token(gpu_device):
    import torch.autograd.forward_ad as forward
    from rnn_train_ring_attractor_amd import linear_attention_step
    q, k, v, s = (torch.randn(2, 2, *d, device=gpu_device) for d in ((8,), (8,), (6,), (8, 6)))
    g = torch.tensor([-0.1, -0.5], device=gpu_device)
    step = lambda q, s: linear_attention_step(q, k, v, g, s)
    want = step(q, s.clone())
    before = s.clone()
    with forward.dual_level():
        assert torch.equal(step(q, s.clone()), want)
        for a, b in ((forward.make_dual(q, q), s), (q, forward.make_dual(s, s))):
            with pytest.raises(RuntimeError, match="no gradient"):
                step(a, b)
    for transformed in (lambda: torch.func.jvp(lambda t: step(t, s), (q,), (q,)), lambda: torch.func.vmap(lambda t: step(t, s))(q[None]),
                        lambda: torch.func.grad(lambda t: step(t, s).sum())(q), lambda: torch.jit.trace(step, (q, s))):
        with pytest.raises(RuntimeError):
            transformed()
    assert torch.equal(s, before)


def test_negated_views_are_read_as_they_are_meant(gpu_device):
    """Tensors that torch keeps negated lazily (the imaginary part of a conjugate), as inputs, positions, states and gradients."""
    from rnn_train_ring_attractor_amd import dropout_func, linear_attention_func, linear_attention_step, rotary_func
    gen = torch.Generator(device=gpu_device).manual_seed(71)
    neg = lambda *s: torch.randn(*s, dtype=torch.complex64, generator=gen, device=gpu_device).conj().imag
    whole = lambda *s: torch._neg_view(torch.randn(*s, generator=gen, device=gpu_device))
    f = torch.rand(4, generator=gen, dtype=torch.float64, device=gpu_device)
    for make in (neg, whole):
        q, k, v, s, x, res, pos = (make(*d) for d in ((2, 5, 2, 8), (2, 5, 2, 8), (2, 5, 2, 6), (2, 2, 8, 6), (2, 5, 2, 8), (2, 5, 2, 8), (2, 5)))
        g = torch._neg_view(torch.rand(2, generator=gen, device=gpu_device))
        do, ds = make(2, 5, 2, 6), make(2, 2, 8, 6)
        assert all(t.is_neg() for t in (q, k, v, s, x, res, pos, g, do, ds))

        def results(of):
            a, b, c, d, e, h = (of(t).detach().requires_grad_(True) for t in (q, k, v, s, x, res))
            o, end = linear_attention_func(a, b, c, of(g), initial_state=d, return_state=True)
            out = [o, end, *torch.autograd.grad([o, end], [a, b, c, d], [of(do), of(ds)])]
            turned = rotary_func((a, e), of(pos), of(f))
            out += [*turned, *torch.autograd.grad(turned, [a, e], [of(x), of(res)])]
            y = dropout_func(e, 0.3, 5, 6, residual=h)
            out += [y, *torch.autograd.grad([y], [e, h], [of(q)])]
            with torch.no_grad():
                out += [linear_attention_func(of(q), of(k), of(v), of(g)), rotary_func(of(x), of(pos), torch._neg_view(-f) if of is plain else f),
                        dropout_func(of(x), 0.3, 5, 6, residual=of(res))]
                state = torch.ones(2, 2, 8, 6, device=gpu_device)
                out += [linear_attention_step(of(q)[:, 0], of(k)[:, 0], of(v)[:, 0], of(g), state), state]
            return out

        plain = lambda t: t
        print("[case] negated views", flush=True)
        for i, (a, b) in enumerate(zip(results(plain), results(lambda t: t.resolve_neg()))):
            assert torch.equal(a, b), i
    state = torch._neg_view(torch.ones(2, 2, 8, 6, device=gpu_device))
    with pytest.raises(RuntimeError, match="in place"), torch.no_grad():
        linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, state)


def test_sizes_past_31_bits_are_refused(gpu_device):
    from rnn_train_ring_attractor_amd import linear_attention_func, linear_attention_step, rotary_func
    n = (1 << 32) + 2
    one = lambda *s: torch.zeros(1, device=gpu_device, dtype=torch.bfloat16).expand(*s)
    g = torch.zeros(1, device=gpu_device)
    print("[case] sizes past 31 bits", flush=True)
    with torch.no_grad():
        with pytest.raises(ValueError, match="2\\^31"):
            rotary_func(one(1, n, 1, 2), torch.zeros(1, device=gpu_device).expand(n), torch.ones(1, device=gpu_device, dtype=torch.float64))
        with pytest.raises(ValueError, match="2\\^31"):
            linear_attention_func(one(1, n, 1, 1), one(1, n, 1, 1), one(1, n, 1, 1), g)
        with pytest.raises(ValueError, match="2\\^31"):
            linear_attention_step(one(n, 1, 1), one(n, 1, 1), one(n, 1, 1), g, torch.zeros(1, device=gpu_device).expand(n, 1, 1, 1))


class _Spy:
    """The library, with a note of every call of a backward and of rotary positions."""

    def __init__(self, lib, calls):
        self.lib, self.calls = lib, calls

    def __getattr__(self, name):
        fn = getattr(self.lib, name)

        def call(*args):
            if name in ("ringattr_linear_attention_bwd", "ringattr_rotary"):
                self.calls.append(args)
            return fn(*args)

        return call


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("sizes", [(2, 90, 4, 2, 32, 48), (2, 70, 2, 2, 40, 72), (4, 500, 2, 1, 70, 66), (4, 500, 2, 2, 20, 70), (3, 70, 2, 1, 136, 140)],
                         ids=lambda s: "x".join(map(str, s)))
def test_gradients_that_nobody_asks_for(sizes, kind, gpu_device, monkeypatch):
    """What is frozen gets no gradient and costs no pass; the others are what they are all together."""
    from rnn_train_ring_attractor_amd import _lib, linear_attention_func
    print(f"[case] frozen {sizes} {kind}", flush=True)
    dtype = TYPES[kind]
    p = _problem(73, *sizes, dtype, start=True)
    t = {n: p[n].to(torch.float32 if n in ("s0", "ds", "g") else dtype).to(gpu_device) for n in ("q", "k", "v", "s0", "do", "ds", "g")}
    calls = []
    spy = _Spy(_lib.load(), calls)
    monkeypatch.setattr(_lib, "load", lambda: spy)
    names = ("q", "k", "v", "s0")
    for with_state in (True, False):
        full = None
        for mask in (15, *range(1, 15)):
            leaves = {n: t[n].detach().requires_grad_(bool(mask >> i & 1)) for i, n in enumerate(names)}
            o, s = linear_attention_func(leaves["q"], leaves["k"], leaves["v"], t["g"], initial_state=leaves["s0"], return_state=True)
            wanted = [n for n in names if leaves[n].requires_grad]
            outs, given = ([o, s], [t["do"], t["ds"]]) if with_state else ([o], [t["do"]])
            if not any(x.requires_grad for x in outs):
                continue
            calls.clear()
            got = dict(zip(wanted, torch.autograd.grad(outs, [leaves[n] for n in wanted], given, allow_unused=True)))
            args, = calls
            asked = [n for n, x in zip(names, args[10:14]) if x is not None]
            assert asked == [n for n in names if n in wanted or (n == "v" and "s0" in wanted)], mask
            full = got if mask == 15 else full
            for n in wanted:
                # (bf16: a state that is a result as well is exact to 2^-24 in place of 2^-16, which a gradient can show as its last bit)
                a, b = got[n].double(), full[n].double()
                assert torch.equal(a, b) if kind != "bf16" or n == "q" else ((a - b).norm() <= 2.0 ** -8 * b.norm()), (mask, n)


def test_turned_tensors_that_nobody_asks_a_gradient_of(gpu_device, monkeypatch):
    from rnn_train_ring_attractor_amd import _lib, rotary_func
    q, k = torch.randn(2, 5, 3, 8, device=gpu_device), torch.randn(2, 5, 1, 8, device=gpu_device)
    pos, f = torch.arange(5, device=gpu_device), torch.rand(4, dtype=torch.float64, device=gpu_device)
    calls = []
    spy = _Spy(_lib.load(), calls)
    a, b = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
    both = torch.autograd.grad(rotary_func((a, b), pos, f), [a, b], [q, k])
    monkeypatch.setattr(_lib, "load", lambda: spy)
    for i, pair in enumerate(((a, k), (q, b))):
        out = rotary_func(pair, pos, f)
        calls.clear()
        got, = torch.autograd.grad([out[i]], [pair[i]], [(q, k)[i]])
        assert torch.equal(got, both[i])
        args, = calls
        assert args[1] is None and args[9] is None           # one tensor


@pytest.mark.parametrize("kind,sizes,count", [(k, s, n) for k, s, n in SEGMENTED if s[0] <= 4 and k != "fp16"],
                         ids=["-".join([k] + [str(x) for x in s]) for k, s, n in SEGMENTED if s[0] <= 4 and k != "fp16"])
def test_a_backward_that_forms_the_states_again(kind, sizes, count, gpu_device):
    """The C ABI's backward without the forward's states against the definition, and next to one that is given them."""
    import ctypes
    from rnn_train_ring_attractor_amd import _lib
    B, T, H, G, Dk, Dv = sizes
    dtype, lib = TYPES[kind], _lib.load()
    code = _lib.SEQUENCE_TYPES[dtype]
    print(f"[case] states again {kind} {sizes}", flush=True)
    p = _without_state_gradient(_problem(79, *sizes, dtype, start=True))
    lengths = _lengths(T, B, count)
    t = {n: p[n].to(torch.float32 if n in ("g", "s0") else dtype).to(gpu_device) for n in ("q", "k", "v", "do", "g", "s0")}
    lens = torch.tensor(lengths, dtype=torch.int32, device=gpu_device)
    room = lambda n: torch.full((n // 4,), math.nan, device=gpu_device)
    need = lib.ringattr_linear_attention_fwd_workspace_bytes(code, *sizes)
    assert need > 0
    ws, o = room(need), torch.empty(B, T, H, Dv, dtype=dtype, device=gpu_device)
    strides = lambda names: (ctypes.c_longlong * (3 * len(names)))(*(s for n in names for s in t[n].stride()[:3]))
    scale, stream = Dk ** -0.5, _lib.stream_handle(torch.device("cuda", 0))
    _lib.check(lib.ringattr_linear_attention_fwd(t["q"].data_ptr(), t["k"].data_ptr(), t["v"].data_ptr(), strides("qkv"), t["g"].data_ptr(),
                                                 t["s0"].data_ptr(), lens.data_ptr(), o.data_ptr(), None, scale, code, *sizes, ws.data_ptr(), need, stream))
    results = []
    for states in (None, ws):
        nbytes = lib.ringattr_linear_attention_bwd_workspace_bytes(code, *sizes, states is not None)
        own, out = room(nbytes), {n: torch.full_like(t[n], math.nan) for n in "qkv"}
        _lib.check(lib.ringattr_linear_attention_bwd(
            t["q"].data_ptr(), t["k"].data_ptr(), t["v"].data_ptr(), t["do"].data_ptr(), strides(["q", "k", "v", "do"]), t["g"].data_ptr(),
            t["s0"].data_ptr(), lens.data_ptr(), None if states is None else states.data_ptr(), None, *(out[n].data_ptr() for n in "qkv"), None, scale,
            code, *sizes, own.data_ptr(), nbytes, stream))
        results.append(out)
    want, size = _reference(p, lengths), _reference(p, lengths, magnitudes=True)
    for n in "qkv":
        assert torch.equal(results[0][n], results[1][n])
        err = (results[0][n].double().cpu() - want["d" + n]).abs()
        K = T + Dk + Dv + H // G + 256
        bound = _bf16_bound(want["d" + n], size["d" + n], K) if kind == "bf16" else 2.0 ** -24 * (want["d" + n].abs() + K * 1.01 * size["d" + n]) + 1e-37
        assert (err <= bound).all(), n


def _turned_exactly(x, positions, frequencies):
    """x [B,T,H,D] turned in halves by the exact product of positions and frequencies, 1 / (2 pi) to 60 digits."""
    from fractions import Fraction
    pi = Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")
    out, r = x.clone(), len(frequencies)
    for m, f in enumerate(frequencies.tolist()):
        turns = [Fraction(p) * Fraction(f) / (2 * pi) for p in positions.tolist()]
        angle = 2 * math.pi * torch.tensor([float(t - round(t)) for t in turns], dtype=torch.float64)[None, :, None]
        a, b = x[..., m], x[..., m + r]
        out[..., m], out[..., m + r] = a * torch.cos(angle) - b * torch.sin(angle), b * torch.cos(angle) + a * torch.sin(angle)
    return out


def test_positions_however_far(gpu_device):
    """Bound: an angle known to 2^-24 turns, cosine and sine in fp32, two products and a sum: (2 pi + 4) 2^-24 of |a| + |b|, then half a step."""
    from rnn_train_ring_attractor_amd import rotary_func
    print("[case] far positions", flush=True)
    far = torch.tensor([0, 3, -(1 << 31), (1 << 40) + 1, 987654321987654321, (1 << 53) + 1, (1 << 62) + 12345, (1 << 63) - 1, -(1 << 63), -(1 << 40) - 77])
    angles = torch.tensor([0.0, 1e7, -3.3e6, 16777215.0, 1e-3, 12345.678, -7.5, 1e9, 3e4, -1e-20], dtype=torch.float32)
    gen = torch.Generator().manual_seed(83)
    for positions, f in ((far, 10000.0 ** (-torch.arange(8, dtype=torch.float64) / 8)), (far, 1000 * torch.rand(8, generator=gen, dtype=torch.float64)),
                         (far.clamp(-(1 << 31), (1 << 31) - 1).int(), torch.rand(8, generator=gen, dtype=torch.float64)),
                         (angles, torch.arange(1, 9, dtype=torch.float64) * 125)):
        x = torch.randn(1, 10, 2, 16, generator=gen, dtype=torch.float64).float()
        got = rotary_func(x.to(gpu_device), positions.to(gpu_device), f.to(gpu_device)).double().cpu()
        want = _turned_exactly(x.double(), positions, f)
        size = (x[..., :8].abs() + x[..., 8:].abs()).repeat(1, 1, 1, 2).double()
        err = (got - want).abs()
        assert (err <= 2.0 ** -24 * 1.0001 * want.abs() + (2 * math.pi + 4) * 2.0 ** -24 * size).all(), (positions.dtype, float((err / size).max()))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("sizes", [(1, 100, 2, 2, 128, 128), (2, 90, 2, 1, 33, 47), (1, 70, 2, 1, 40, 72), (1, 70, 1, 1, 256, 136), (4, 500, 2, 2, 20, 70),
                                   (4, 500, 2, 1, 70, 66), (4, 500, 2, 2, 130, 9)], ids=lambda s: "x".join(map(str, s)))
def test_what_is_not_finite_reaches_rows_that_see_it_only(sizes, kind, gpu_device):
    """At every width, within a chunk, across chunks and across segments."""
    dtype, T = TYPES[kind], sizes[1]
    p = _without_state_gradient(_problem(89, *sizes, dtype, start=True))
    clean = _call(p, dtype, gpu_device, None, state=False)
    for at in (0, 45, T - 1):
        for name in ("q", "k", "v", "do"):
            for value in (-math.inf, math.nan):
                print(f"[case] {value} in {name} at {at} {sizes} {kind}", flush=True)
                bad = {n: (None if x is None else x.clone()) for n, x in p.items()}
                bad[name][0, at, :, -1] = value
                got = _call(bad, dtype, gpu_device, None, state=False)
                front, back, other = slice(0, at), slice(at + 1, T), slice(0, T)
                same = {"q": {"o": (front, back), "dq": (other,), "dk": (back,), "dv": (back,)}, "k": {"o": (front,), "dq": (front,), "dk": (other,), "dv": (front, back)},
                        "v": {"o": (front,), "dq": (front,), "dk": (front, back), "dv": (other,)}, "do": {"o": (other,), "dq": (front, back), "dk": (back,), "dv": (back,)}}[name]
                for n, rows in same.items():
                    assert torch.equal(got[n][1:], clean[n][1:]), n
                    assert all(torch.equal(got[n][0, r], clean[n][0, r]) for r in rows), n
                if name in ("k", "v"):
                    assert not torch.isfinite(got["o"][0, at:]).all(-1).any(), "rows that see it"


def test_forward_mode_over_a_backward_is_refused(gpu_device):
    """A gradient that carries a tangent goes into no backward without a rule for it; one that carries none does."""
    import torch.autograd.forward_ad as forward
    entries, x = _entries(gpu_device)
    for name, op in entries.items():
        print(f"[case] forward over backward {name}", flush=True)
        leaf = x.clone().requires_grad_(True)
        y = op(leaf)
        g = torch.ones_like(y)
        want, = torch.autograd.grad(y, leaf, g, retain_graph=True)
        with forward.dual_level():
            assert torch.equal(torch.autograd.grad(y, leaf, g, retain_graph=True)[0], want)
            if name != "residual":                               # (whose gradient is the one that comes in)
                with pytest.raises((RuntimeError, NotImplementedError)):
                    torch.autograd.grad(y, leaf, forward.make_dual(g, g))
