"""The sequence operators on the GPU against their definitions in 64 bits (oracle/sequence_oracle.py).

Bounds.  A result y = sum of terms is rounded once to its type, half a step: eps / 2 |y|.  What is computed on the way is bounded
against A, the same sum over the terms' magnitudes (the operator of the inputs' magnitudes): K additions and products in fp32 give at most
K 2^-24 A, where K counts the contraction over a head, the tokens and the powers of the decay (a power is off by its exponent's
rounding: up to 256 half steps at the decays here).  With bfloat16 operands every term of an output passes one operand that is rounded to
bfloat16, its weight (tokens of its chunk) or the state (earlier ones): half a step, 2^-8; what a chunk adds to such a state enters
as two bf16 numbers, 2^-16 for the second.  A state that is itself a result enters no output and takes three, 2^-24 among the additions."""
import math

import pytest
import torch

from oracle import sequence_oracle as O

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _within(name, got, want, size, dtype, K):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, name
    eps = torch.finfo(dtype).eps / 2
    path = K * 2.0 ** -24 + (2.0 ** -8 + 2.0 ** -16 if dtype == torch.bfloat16 else 0.0)
    tiny = torch.finfo(dtype).tiny if dtype == torch.float16 else 1e-37
    bound = eps * want.abs() + (1 + eps) * path * size + tiny
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()}, worst {float(((got - want).abs() / bound).max()):.2f} of the bound"


def _rand(gen, *shape):
    return torch.randn(*shape, generator=gen, dtype=torch.float64)


def _problem(seed, B, T, H, G, Dk, Dv, dtype, start, decays=None):
    gen = torch.Generator().manual_seed(seed)
    p = {"q": _rand(gen, B, T, H, Dk), "k": _rand(gen, B, T, G, Dk), "v": _rand(gen, B, T, G, Dv), "do": _rand(gen, B, T, H, Dv)}
    p = {n: x.to(dtype).double() for n, x in p.items()}
    if decays is None:
        decays = torch.log1p(-torch.exp2(-torch.linspace(1.0, 9.0, H)))
    p["g"] = torch.as_tensor(decays, dtype=torch.float32).double()
    p["s0"] = _rand(gen, B, H, Dk, Dv).float().double() if start else None
    p["ds"] = _rand(gen, B, H, Dk, Dv).float().double()
    return p


def _reference(p, lengths, want_grads=True, magnitudes=False):
    f = (lambda x: None if x is None else x.abs()) if magnitudes else (lambda x: x)
    leaves = {n: f(p[n]).clone().requires_grad_(True) for n in ("q", "k", "v")}
    s0 = None if p["s0"] is None else f(p["s0"]).clone().requires_grad_(True)
    o, s = O.attention(leaves["q"], leaves["k"], leaves["v"], p["g"], s0, lengths)
    out = {"o": o.detach(), "state": s.detach()}
    if want_grads:
        torch.autograd.backward([o, s], [f(p["do"]), f(p["ds"])])
        zero = lambda x: torch.zeros_like(x) if x.grad is None else x.grad
        out.update({"d" + n: zero(x) for n, x in leaves.items()})
        if s0 is not None:
            out["ds0"] = zero(s0)
    return out


def _run(p, dtype, dev, lengths, place=lambda x: x):
    from rnn_train_ring_attractor_amd import linear_attention_func
    leaves = [place(p[n].to(dtype).to(dev)).detach().requires_grad_(True) for n in ("q", "k", "v")]
    s0 = None if p["s0"] is None else p["s0"].float().to(dev).requires_grad_(True)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=dev)
    o, s = linear_attention_func(*leaves, p["g"].float().to(dev), initial_state=s0, lengths=lens, return_state=True)
    wanted = leaves + ([] if s0 is None else [s0])
    grads = torch.autograd.grad([o, s], wanted, [place(p["do"].to(dtype).to(dev)), p["ds"].float().to(dev)])
    out = {"o": o, "state": s, "dq": grads[0], "dk": grads[1], "dv": grads[2]}
    if s0 is not None:
        out["ds0"] = grads[3]
    return out


def _compare(p, got, lengths, dtype, share):
    want, size = _reference(p, lengths), _reference(p, lengths, magnitudes=True)
    T, Dk, Dv = p["q"].shape[1], p["q"].shape[3], p["v"].shape[3]
    K = T + Dk + Dv + share + 256
    for name in want:
        kind = torch.float32 if name in ("state", "ds0") else dtype
        _within(name, got[name], want[name], size[name], kind, K)


SHAPES = [(1, 1, 1, 1, 1, 1), (2, 5, 2, 1, 3, 7), (1, 31, 2, 2, 16, 16), (2, 32, 2, 2, 64, 64), (1, 33, 3, 1, 33, 65), (2, 64, 2, 2, 128, 128),
          (1, 100, 2, 2, 250, 31), (1, 97, 1, 1, 40, 256), (1, 70, 2, 1, 256, 256), (3, 129, 4, 2, 80, 112), (1, 1100, 1, 1, 24, 72)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("B,T,H,G,Dk,Dv", SHAPES, ids=["x".join(map(str, s)) for s in SHAPES])
def test_attention_and_its_gradients(B, T, H, G, Dk, Dv, kind, gpu_device):
    print(f"[case] linear attention {B} {T} {H} {G} {Dk} {Dv} {kind}", flush=True)
    dtype = TYPES[kind]
    p = _problem(7, B, T, H, G, Dk, Dv, dtype, start=T % 2 == 1)
    _compare(p, _run(p, dtype, gpu_device, None), None, dtype, H // G)


@pytest.mark.parametrize("kind", list(TYPES))
def test_padded_batches(kind, gpu_device):
    """Lengths from none to all, one past the ends of the range (clamped); rows behind a length hold NaN and are not read."""
    dtype, T = TYPES[kind], 150
    lengths = [T, 0, 1, 31, 32, 33, 149]
    p = _problem(11, len(lengths), T, 2, 1, 48, 72, dtype, start=True)
    for n in ("q", "k", "v", "do"):
        for b, m in enumerate(lengths):
            p[n][b, m:] = math.nan
    print(f"[case] padded batch {kind}", flush=True)
    got = _run(p, dtype, gpu_device, [T + 9, -3] + lengths[2:])
    clean = {n: (x.nan_to_num() if n in ("q", "k", "v", "do") else x) for n, x in p.items()}
    _compare(clean, got, lengths, dtype, 2)
    for n in ("o", "dq", "dk", "dv"):
        for b, m in enumerate(lengths):
            assert (got[n][b, m:] == 0).all()


# (kind, sizes, segments that the tokens are cut into)
SEGMENTED = [("fp32", (8, 500, 8, 4, 4, 130), 2), ("bf16", (8, 500, 8, 8, 4, 130), 2), ("fp32", (4, 500, 64, 64, 10, 6), 2),
             ("bf16", (8, 1000, 32, 8, 10, 6), 2), ("fp32", (4, 200, 32, 32, 70, 66), 2), ("bf16", (4, 800, 32, 16, 70, 66), 2),
             ("fp32", (4, 500, 2, 1, 20, 70), 8), ("bf16", (4, 500, 2, 2, 20, 70), 8), ("fp16", (4, 500, 2, 2, 70, 66), 8),
             ("bf16", (4, 500, 2, 1, 70, 66), 8), ("fp16", (4, 500, 4, 4, 16, 30), 8), ("bf16", (4, 500, 4, 2, 16, 30), 8),
             ("fp32", (4, 500, 2, 2, 130, 9), 8), ("bf16", (4, 500, 2, 2, 9, 130), 8)]


@pytest.mark.parametrize("kind,sizes,count", SEGMENTED, ids=["-".join([k] + [str(x) for x in s]) for k, s, _ in SEGMENTED])
def test_lengths_that_end_in_any_segment(kind, sizes, count, gpu_device):
    """Sequences cut into two segments and into many, heads whose dv and dk go back together and not: lengths that end in front of, at and
    behind a segment's first token, in the last one, and none."""
    from rnn_train_ring_attractor_amd import _lib
    B, T, H, G, Dk, Dv = sizes
    dtype = TYPES[kind]
    nbytes = _lib.load().ringattr_linear_attention_fwd_workspace_bytes(_lib.SEQUENCE_TYPES[dtype], *sizes)
    each = B * H * Dk * Dv * 4
    assert (count - 1) * each <= nbytes < (count - 1) * each + 256, "the tokens are cut otherwise than this case is for"
    first = -(-(-(-T // 64)) // count) * 64
    lengths = [first + 1, T, 0, first, 1, first - 1, T - 1, 65][:B]
    print(f"[case] segments {kind} {sizes} {lengths}", flush=True)
    p = _problem(37, *sizes, dtype, start=True)
    for n in ("q", "k", "v", "do"):
        for b, m in enumerate(lengths):
            p[n][b, m:] = math.nan
    got = _run(p, dtype, gpu_device, lengths)
    clean = {n: (x.nan_to_num() if n in ("q", "k", "v", "do") else x) for n, x in p.items()}
    _compare(clean, got, lengths, dtype, H // G)


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("decays", [[0.0, 0.0], [-math.inf, -1e-7], [-40.0, -3.0]], ids=["none", "all_and_hardly", "strong"])
def test_decays_at_their_ends(decays, kind, gpu_device):
    dtype = TYPES[kind]
    p = _problem(13, 2, 90, 2, 2, 32, 32, dtype, start=True, decays=decays)
    print(f"[case] decays {decays} {kind}", flush=True)
    _compare(p, _run(p, dtype, gpu_device, None), None, dtype, 1)


@pytest.mark.parametrize("kind", list(TYPES))
def test_strided_rows(kind, gpu_device):
    """Time-major memory, slices of a wider row that start off 16 bytes, heads stepped over: the same bits as from contiguous tensors."""
    dtype = TYPES[kind]
    p = _problem(17, 2, 75, 2, 2, 64, 64, dtype, start=False)
    want = _run(p, dtype, gpu_device, None)

    def wide(x):
        big = torch.full((*x.shape[:-1], x.shape[-1] + 3), math.nan, dtype=x.dtype, device=x.device)
        big[..., 1:-2] = x
        return big[..., 1:-2]

    def stepped(x):
        big = torch.full((x.shape[0], x.shape[1], 2 * x.shape[2], x.shape[3]), math.nan, dtype=x.dtype, device=x.device)
        big[:, :, ::2] = x
        return big[:, :, ::2]

    for name, place in (("time", lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)), ("wide", wide), ("stepped", stepped)):
        print(f"[case] strides {name} {kind}", flush=True)
        got = _run(p, dtype, gpu_device, None, place)
        assert all(torch.equal(got[n], want[n]) for n in want), name


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_values_that_are_not_finite_stay_where_they_are_seen(kind, gpu_device):
    """A row of v (k, q, grad_o) that holds infinities or NaN changes nothing in front of it (in gradients: behind it)."""
    from rnn_train_ring_attractor_amd import linear_attention_func
    dtype, T, at = TYPES[kind], 80, 45
    p = _problem(19, 1, T, 2, 2, 32, 48, dtype, start=True)
    clean = _run(p, dtype, gpu_device, None)
    for name in ("v", "k", "q", "do"):
        for value in (math.inf, math.nan):
            print(f"[case] {value} in {name} {kind}", flush=True)
            bad = {n: (None if x is None else x.clone()) for n, x in p.items()}
            bad[name][0, at, :, 5] = value
            got = _run(bad, dtype, gpu_device, None)
            if name in ("v", "k"):
                assert torch.equal(got["o"][:, :at], clean["o"][:, :at])
                assert not torch.isfinite(got["o"][:, at:]).all()
                assert torch.equal(got["dq"][:, :at], clean["dq"][:, :at])
            elif name == "q":
                assert torch.equal(got["o"][:, :at], clean["o"][:, :at]) and torch.equal(got["o"][:, at + 1:], clean["o"][:, at + 1:])
                assert torch.equal(got["state"], clean["state"]) and torch.equal(got["dk"][:, at + 1:], clean["dk"][:, at + 1:])
                assert torch.equal(got["dv"][:, at + 1:], clean["dv"][:, at + 1:])
            else:
                assert torch.equal(got["o"], clean["o"])
                assert torch.equal(got["dq"][:, :at], clean["dq"][:, :at]) and torch.equal(got["dq"][:, at + 1:], clean["dq"][:, at + 1:])
                assert torch.equal(got["dk"][:, at + 1:], clean["dk"][:, at + 1:]) and torch.equal(got["dv"][:, at + 1:], clean["dv"][:, at + 1:])
    # an infinite value is an infinity in the rows that see it, of the weight's sign
    bad = p["v"].clone()
    bad[0, at, :, 5] = math.inf
    t = lambda x: x.to(dtype).to(gpu_device)
    o = linear_attention_func(t(p["q"]), t(p["k"]), t(bad), p["g"].float().to(gpu_device)).double().cpu()
    w = (p["q"][0, at] * p["k"][0, at]).sum(-1)
    assert torch.equal(o[0, at, :, 5], torch.sign(w) * math.inf)


def test_gradients_are_differences_of_the_outputs(gpu_device):
    """Central differences of a scalar of the outputs along random directions.  The scalar is linear in each input alone, so the
    difference has no error of its own but the outputs' rounding: K 2^-24 of the scalar's terms over the step."""
    from rnn_train_ring_attractor_amd import linear_attention_func
    p = _problem(23, 2, 70, 2, 1, 20, 28, torch.float32, start=True)
    got = _run(p, torch.float32, gpu_device, None)
    size = _reference(p, None, want_grads=False, magnitudes=True)
    total = float((size["o"] * p["do"].abs()).sum() + (size["state"] * p["ds"].abs()).sum())
    f32 = lambda x: x.float().to(gpu_device)

    def scalar(**over):
        x = {**p, **over}
        o, s = linear_attention_func(f32(x["q"]), f32(x["k"]), f32(x["v"]), f32(x["g"]), initial_state=f32(x["s0"]), return_state=True)
        return float((o.double().cpu() * p["do"]).sum() + (s.double().cpu() * p["ds"]).sum())

    gen = torch.Generator().manual_seed(1)
    for name, grad in (("q", "dq"), ("k", "dk"), ("v", "dv"), ("s0", "ds0")):
        print(f"[case] differences {name}", flush=True)
        way = _rand(gen, *p[name].shape).sign()
        up, down = (p[name] + way).float().double(), (p[name] - way).float().double()
        want = (scalar(**{name: up}) - scalar(**{name: down}))
        have = float((got[grad].double().cpu() * (up - down)).sum())
        K = 70 + 48 + 256
        assert abs(want - have) <= 4 * K * 2.0 ** -24 * 4 * total, name


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("B,H,G,Dk,Dv", [(1, 1, 1, 1, 1), (3, 4, 2, 33, 47), (2, 2, 2, 64, 64), (1, 8, 1, 128, 128), (40, 16, 4, 256, 256),
                                         (300, 8, 8, 20, 12)])
def test_single_tokens_go_on_from_a_prompt(B, H, G, Dk, Dv, kind, gpu_device):
    """Tokens one by one behind a prompt: each against the definition, places that wait as they were, and the whole sequence at once."""
    from rnn_train_ring_attractor_amd import linear_attention_func, linear_attention_step
    dtype, T, first = TYPES[kind], 9, 6
    print(f"[case] step {B} {H} {G} {Dk} {Dv} {kind}", flush=True)
    p = _problem(29, B, T, H, G, Dk, Dv, dtype, start=True)
    t = lambda x: x.to(dtype).to(gpu_device)
    q, k, v, g = t(p["q"]), t(p["k"]), t(p["v"]), p["g"].float().to(gpu_device)
    o0, state = linear_attention_func(q[:, :first], k[:, :first], v[:, :first], g, initial_state=p["s0"].float().to(gpu_device),
                                      return_state=True)
    outs = [o0]
    for i in range(first, T):
        outs.append(linear_attention_step(q[:, i], k[:, i], v[:, i], g, state)[:, None])
    want, want_s = O.attention(p["q"], p["k"], p["v"], p["g"], p["s0"])
    size, size_s = O.attention(*(p[n].abs() for n in ("q", "k", "v")), p["g"], p["s0"].abs())
    K = T + Dk + Dv + 256
    _within("o", torch.cat(outs, dim=1), want, size, dtype, K)
    _within("state", state, want_s, size_s, torch.float32, K)
    active = torch.arange(B, device=gpu_device) % 2 == 1
    before = state.clone()
    o = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, state, active=active)
    assert torch.equal(state[~active], before[~active]) and (o[~active] == 0).all()
    alone = before.clone()
    o_all = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, alone)
    assert torch.equal(state[active], alone[active]) and torch.equal(o[active], o_all[active])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("B,T,H,G,D,r,pos", [(1, 1, 1, 1, 2, 1, "shared"), (2, 7, 3, 1, 33, 16, "each"), (3, 5, 4, 2, 64, 32, "each"),
                                             (2, 130, 2, 2, 128, 32, "shared"), (2, 3, 5, 5, 96, 24, "angle"), (1, 4, 1, 1, 520, 260, "angle"),
                                             (2, 9, 3, 1, 64, 25, "each"), (1, 600, 2, 2, 62, 10, "shared"), (3, 33, 4, 1, 128, 26, "angle"),
                                             (500, 1, 2, 1, 16, 3, "each"), (1, 2, 7, 3, 20, 5, "shared"), (1, 1, 900, 7, 6, 2, "each")])
def test_rotary(B, T, H, G, D, r, pos, layout, kind, gpu_device):
    """Bound: cos and sin are fp32 numbers of an angle known to 2^-24 turns (2 pi 2^-24 rad) and each product and the sum are rounded:
    (2 pi + 4) 2^-24 of |a| + |b|, then the type's half step."""
    from rnn_train_ring_attractor_amd import rotary_func
    dtype = TYPES[kind]
    print(f"[case] rotary {B} {T} {H} {G} {D} {r} {pos} {layout} {kind}", flush=True)
    gen = torch.Generator().manual_seed(31)
    q, k, dq, dk = (_rand(gen, B, T, h, D).to(dtype) for h in (H, G, H, G))
    f = torch.arange(1, r + 1, dtype=torch.float64) if pos == "angle" else 10000.0 ** (-torch.arange(r, dtype=torch.float64) / r)
    if pos == "angle":
        positions = (10 * torch.randn(B, T, generator=gen)).float()
    elif pos == "each":
        positions = torch.randint(-5, 1 << 31, (B, T), generator=gen)
    else:
        positions = torch.arange(1 << 20, (1 << 20) + T, dtype=torch.int32)
    scale = 1.25
    dev = lambda x: x.to(gpu_device)
    leaves = [dev(q).requires_grad_(True), dev(k).requires_grad_(True)]
    out = rotary_func(tuple(leaves), dev(positions), dev(f), layout=layout, scale=scale)
    grads = torch.autograd.grad(out, leaves, [dev(dq), dev(dk)])
    for x, y in ((q, out[0]), (k, out[1])):
        want = O.rotary(x.double(), positions, f, layout, scale)
        size = torch.zeros_like(want)
        i, j = (slice(0, r), slice(r, 2 * r)) if layout == "half" else (slice(0, 2 * r, 2), slice(1, 2 * r, 2))
        both = scale * (x.double()[..., i].abs() + x.double()[..., j].abs())
        size[..., i], size[..., j] = both, both
        err = (y.detach().double().cpu() - want).abs()
        assert (err <= torch.finfo(dtype).eps / 2 * want.abs() * 1.0001 + (2 * math.pi + 4) * 2.0 ** -24 * size + 1e-7 * (dtype == torch.float16)).all()
        assert torch.equal(y.detach().cpu()[..., 2 * r:], x[..., 2 * r:])
    for x, y in ((dq, grads[0]), (dk, grads[1])):
        want = O.rotary(x.double(), -positions, f, layout, scale)
        want[..., 2 * r:] = x.double()[..., 2 * r:]
        i, j = (slice(0, r), slice(r, 2 * r)) if layout == "half" else (slice(0, 2 * r, 2), slice(1, 2 * r, 2))
        size = torch.zeros_like(want)
        both = scale * (x.double()[..., i].abs() + x.double()[..., j].abs())
        size[..., i], size[..., j] = both, both
        err = (y.double().cpu() - want).abs()
        assert (err <= torch.finfo(dtype).eps / 2 * want.abs() * 1.0001 + (2 * math.pi + 4) * 2.0 ** -24 * size + 1e-7 * (dtype == torch.float16)).all()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_of_rows_at_any_address(layout, kind, gpu_device):
    """Rows that start on 16 bytes, on two values and on one, heads stepped over, time-major: the same bits as contiguous ones."""
    from rnn_train_ring_attractor_amd import rotary_func
    gen = torch.Generator().manual_seed(41)
    pos = torch.arange(19, device=gpu_device)
    for D, r in ((64, 24), (64, 20), (64, 23), (62, 8)):
        f = torch.rand(r, generator=gen, dtype=torch.float64).to(gpu_device)
        x = _rand(gen, 3, 19, 5, D).to(TYPES[kind]).to(gpu_device)
        want = rotary_func(x, pos, f, layout)
        for lead, row in ((8, 80), (2, 72), (2, 71), (1, 72), (4, 66)):
            print(f"[case] rotary rows {layout} {kind} {D} {r} {lead} {row}", flush=True)
            wide = torch.full((19, 3, 10, row), math.nan, dtype=x.dtype, device=gpu_device)
            placed = wide.transpose(0, 1)[:, :, ::2, lead:lead + D] if lead + D <= row else wide.transpose(0, 1)[:, :, ::2, :D]
            placed.copy_(x)
            assert torch.equal(rotary_func(placed, pos, f, layout), want)
            both = rotary_func((placed, x[:, :, :2]), pos, f, layout)
            assert torch.equal(both[0], want) and torch.equal(both[1], want[:, :, :2])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape,p", [((1,), 0.5), ((7, 3), 0.25), ((5, 129), 0.9), ((64, 1000), 0.1), ((9,), 0.0)])
def test_dropout(shape, p, kind, gpu_device):
    """The mask equals the definition's, kept values are the product's rounding (1 / (1 - p) is an fp32 number: one more half step of
    fp32), dropped ones are zero whatever they held."""
    from rnn_train_ring_attractor_amd import dropout_func
    dtype = TYPES[kind]
    print(f"[case] dropout {shape} {p} {kind}", flush=True)
    gen = torch.Generator().manual_seed(37)
    x, res, do = (_rand(gen, *shape).to(dtype) for _ in range(3))
    seed, offset = 0xFEDCBA9876543210, 0x0123456789ABCDEF
    keep = torch.from_numpy(O.keep_mask(x.numel(), p, seed, offset)).view(shape)
    dev = lambda t: t.to(gpu_device)
    a, b = dev(x).requires_grad_(True), dev(res).requires_grad_(True)
    y = dropout_func(a, p, seed, offset, residual=b)
    ga, gb = torch.autograd.grad([y], [a, b], [dev(do)])
    plain = dropout_func(dev(x), p, seed, offset)
    counted = dropout_func(dev(x), p, seed, torch.tensor([offset], device=gpu_device))
    assert torch.equal(plain, counted) and torch.equal(gb.cpu(), do)
    scale = torch.where(keep, 1.0 / (1.0 - p), 0.0).double()
    half = torch.finfo(dtype).eps / 2
    none = torch.zeros(shape, dtype=dtype)
    for got, x_, rest in ((plain, x, none), (ga, do, none), (y, x, res)):
        got, want = got.detach().cpu(), rest.double() + x_.double() * scale
        size = rest.double().abs() + x_.double().abs() * scale
        assert ((got.double() - want).abs() <= half * want.abs() * 1.0001 + 3 * 2.0 ** -24 * size + 6e-8 * (dtype == torch.float16)).all()
        assert torch.equal(got[~keep], rest[~keep])
    odd = dev(torch.cat([torch.zeros(1, dtype=dtype), x.flatten()]))[1:].view(shape)       # off 16 bytes
    assert torch.equal(dropout_func(odd, p, seed, offset), plain)
    wild = torch.where(keep, x, torch.tensor(math.inf, dtype=dtype))
    assert torch.equal(dropout_func(dev(wild), p, seed, offset), plain)
