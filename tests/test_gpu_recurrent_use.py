"""The recurrent layer's operators as they are used: together in a block, for prompts and tokens, recorded into graphs, on streams of their own, far into large
tensors, with frozen and broadcast inputs, under what watches operators, and what they refuse on a GPU."""
import math

import pytest
import torch

from oracle import recurrent_oracle as O
from tests.test_gpu_recurrent import TYPES, conv_problem, norm_problem, run_conv, run_norm, run_scan, scan_problem

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------
# A block: convolution, scan with its gate, norm and scaled residual, the next block's norm
# ------------------------------------------------------------------------------------------------
def block_problem(seed, B, T, C, N, G, K, dtype, dev):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64).to(dtype).to(dev)
    f = lambda t: t.float().to(dev)
    rows = {"x": r(B, T, C), "delta": r(B, T, C), "Bm": r(B, T, G, N), "Cm": r(B, T, G, N), "z": r(B, T, C), "res": r(B, T, C)}
    n = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)
    weights = {"w": f(n(C, K) * K ** -0.5), "wb": f(0.1 * n(C)), "A": f(-torch.exp(n(C, N))), "D": f(n(C)), "bias": f(n(C) - 3), "nw": f(1 + 0.1 * n(C)),
               "scale": f(0.3 + 0.1 * n(C)), "nx": f(1 + 0.1 * n(C))}
    return rows, weights


ROWS, WEIGHTS = ("x", "delta", "Bm", "Cm", "z", "res"), ("w", "wb", "A", "D", "bias", "nw", "scale", "nx")


def block(r, w, start=None, lengths=None, states=False):
    from rnn_train_ring_attractor_amd import causal_conv_func, norm_gate_func, selective_scan_func
    a, b = (None, None) if start is None else start
    u, a = causal_conv_func(r["x"], w["w"], w["wb"], initial_state=a, lengths=lengths, activation="silu", return_state=True)
    y, b = selective_scan_func(u, r["delta"], w["A"], r["Bm"], r["Cm"], D=w["D"], z=r["z"], delta_bias=w["bias"], initial_state=b, lengths=lengths,
                               softplus=True, return_state=True)
    out = norm_gate_func(y, w["nw"], residual=r["res"], scale=w["scale"], next_weight=w["nx"])
    return (*out, a, b) if states else out


def block_token(r, w, t, a, b):
    from rnn_train_ring_attractor_amd import causal_conv_step, norm_gate_func, selective_scan_step
    u = causal_conv_step(r["x"][:, t], w["w"], a, bias=w["wb"], activation="silu")
    y = selective_scan_step(u, r["delta"][:, t], w["A"], r["Bm"][:, t], r["Cm"][:, t], b, D=w["D"], z=r["z"][:, t], delta_bias=w["bias"], softplus=True)
    return norm_gate_func(y, w["nw"], residual=r["res"][:, t], scale=w["scale"], next_weight=w["nx"])


def exact_block(r, w):
    r, w = ({n: t.detach().double().cpu().requires_grad_(True) for n, t in d.items()} for d in (r, w))
    u, _ = O.conv(r["x"], w["w"], w["wb"], act="silu")
    y, _ = O.scan(u, r["delta"], w["A"], r["Bm"], r["Cm"], w["D"], r["z"], w["bias"], plus=True)
    return O.norm_gate(y, w["nw"], residual=r["res"], scale=w["scale"], next_weight=w["nx"]), r, w


def test_block_and_its_gradients(gpu_device):
    """fp32.  Bound, of norms: the stages' errors add up, to first order; each is K 2^-24 of its terms' sizes (K: 3 T + 2 C + 300 for the three together,
    as their own tests count, forwards and back), sizes are up to 2^4 times the values for sums of this many terms of any sign, and the two norms
    divide by values of order one."""
    B, T, C, N, G, K = 2, 70, 48, 16, 2, 4
    print("[case] block", flush=True)
    rows, weights = block_problem(3, B, T, C, N, G, K, torch.float32, gpu_device)
    gen = torch.Generator(device=gpu_device).manual_seed(4)
    given = [torch.randn(B, T, C, generator=gen, device=gpu_device) for _ in range(2)]
    r, w = ({n: t.clone().requires_grad_(True) for n, t in d.items()} for d in (rows, weights))
    out = block(r, w)
    grads = torch.autograd.grad(out, [*(r[n] for n in ROWS), *(w[n] for n in WEIGHTS)], given)
    want, er, ew = exact_block(rows, weights)
    exact = torch.autograd.grad(want, [*(er[n] for n in ROWS), *(ew[n] for n in WEIGHTS)], [g.double().cpu() for g in given])
    bound = 2 * (3 * T + 2 * C + 300) * 2.0 ** -24 * 2 ** 4
    for name, a, b in zip(("y", "n", *ROWS, *WEIGHTS), (*out, *grads), (*want, *exact)):
        err = float((a.detach().double().cpu() - b).norm() / b.norm())
        assert err <= bound, (name, err, bound)


@pytest.mark.parametrize("kind", list(TYPES))
def test_block_for_a_prompt_and_its_tokens(kind, gpu_device):
    """The tokens behind a prompt of several lengths, one by one, give what the whole sequences give: in fp32 up to the order of a segment's sums, otherwise up
    to the roundings between the stages (u, y and the outputs, half a step each, in both ways)."""
    B, T, C, N, G, K, dtype = 3, 150, 72, 16, 1, 4, TYPES[kind]
    print(f"[case] prompt and tokens {kind}", flush=True)
    rows, weights = block_problem(5, B, T, C, N, G, K, dtype, gpu_device)
    with torch.no_grad():
        whole = block(rows, weights)
        for half in (1, 2, 37, 149):
            y, n, a, b = block({m: t[:, :half] for m, t in rows.items()}, weights, states=True)
            assert all(torch.allclose(p.float(), q[:, :half].float(), rtol=0, atol=8 * torch.finfo(dtype).eps * float(q.abs().max())) for p, q in zip((y, n), whole))
            for t in range(half, min(T, half + 5)):
                got = block_token(rows, weights, t, a, b)
                for p, q in zip(got, whole):
                    q = q[:, t].float()
                    assert float((p.float() - q).norm() / q.norm()) <= (2.0 ** -16 if kind == "fp32" else 6 * torch.finfo(dtype).eps / 2), (half, t)


def test_recorded_training_step(gpu_device):
    """A block's forward and backward recorded once and replayed over other inputs, eager work and waits between: the bits of the eager step each time."""
    print("[case] graph", flush=True)
    B, T, C, N, G, K = 2, 300, 64, 16, 1, 4
    rows, weights = block_problem(7, B, T, C, N, G, K, torch.bfloat16, gpu_device)
    rows["dy"], rows["dn"] = torch.randn_like(rows["x"]), torch.randn_like(rows["x"])
    lengths = torch.tensor([T, 123], dtype=torch.int32, device=gpu_device)

    def step(d):
        r, w = ({n: t.detach().requires_grad_(True) for n, t in x.items()} for x in ({n: d[n] for n in ROWS}, weights))
        out = block(r, w, lengths=lengths)
        return [*out, *torch.autograd.grad(out, [*(r[n] for n in ROWS), *(w[n] for n in WEIGHTS)], [d["dy"], d["dn"]])]

    static = {n: t.clone() for n, t in rows.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    gen = torch.Generator(device=gpu_device).manual_seed(9)
    for i in range(4):
        for t in static.values():
            t.copy_(torch.randn(t.shape, generator=gen, device=gpu_device))
        want = [t.detach().clone() for t in step(static)]
        other = {n: t[:, :7 + i].contiguous() for n, t in static.items()}
        y = block({n: other[n] for n in ROWS}, weights)[0]               # other eager work of the same operators
        graph.replay()
        torch.cuda.synchronize()
        assert torch.isfinite(y).all()
        for a, b in zip(out, want):
            assert torch.equal(a, b), i


def test_two_graphs_and_two_streams_at_once(gpu_device):
    """Calls side by side have the bits of calls alone: workspaces are a call's own."""
    print("[case] streams", flush=True)
    sets = [block_problem(11 + i, 1, 2000, 64, 16, 1, 4, torch.bfloat16, gpu_device) for i in range(2)]
    with torch.no_grad():
        want = [block(*s, states=True) for s in sets]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in sets]
        got = [[], []]
        for st in streams:
            st.wait_stream(torch.cuda.current_stream())
        for _ in range(5):
            for i, st in enumerate(streams):
                with torch.cuda.stream(st):
                    got[i].append(block(*sets[i], states=True))
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for g in got[i] for a, b in zip(g, want[i]))
        graphs, outs = [], []
        for s in sets:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(block(*s, states=True))
            graphs.append(graph)
        for _ in range(3):
            for i, st in enumerate(streams):
                with torch.cuda.stream(st):
                    graphs[i].replay()
            torch.cuda.synchronize()
            for i in range(2):
                assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))


def test_recorded_tokens(gpu_device):
    """A served token recorded once: states move on in place at every replay."""
    print("[case] recorded tokens", flush=True)
    rows, weights = block_problem(15, 2, 9, 64, 16, 1, 4, torch.bfloat16, gpu_device)
    with torch.no_grad():
        whole = block(rows, weights, states=True)
        static = {n: t[:, :1].clone() for n, t in rows.items()}
        a, b = torch.zeros_like(whole[2]), torch.zeros_like(whole[3])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block_token(static, weights, 0, a, b)
        a.zero_(), b.zero_()
        for t in range(9):
            for n in static:
                static[n].copy_(rows[n][:, t:t + 1])
            graph.replay()
            torch.cuda.synchronize()
            assert all(float((p.float() - q[:, t].float()).norm() / q[:, t].float().norm()) <= 6 * 2.0 ** -8 for p, q in zip(out, whole)), t
        assert torch.equal(a, whole[2])


# ------------------------------------------------------------------------------------------------
# Segments, sizes
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_sequences_alone_and_in_a_batch(kind, gpu_device):
    """One sequence is cut into segments, 300 of them are not: the two differ by the roundings of a state (16 2^-24 of its terms a segment's border) in
    what is fp32, and in rows by a last bit besides."""
    print(f"[case] alone and in a batch {kind}", flush=True)
    T, C, N = 700, 40, 16
    p = scan_problem(17, 1, T, C, N, 1, TYPES[kind])
    one = run_scan(p, TYPES[kind], gpu_device, [T - 5])
    shared = ("A", "D", "bias")
    many = {n: t if t is None or n in shared else t.expand(300, *t.shape[1:]) for n, t in p.items()}
    batch = run_scan(many, TYPES[kind], gpu_device, [T - 5] * 300)
    size, _ = O.scan_sizes(*(p[n] for n in ("x", "delta", "A", "B", "C", "D", "z", "bias", "start")), [T - 5], True, p["dy"], p["de"])
    for n in ("y", "state", "dx", "ddelta", "dB", "dC", "dz", "dstart"):
        assert all(torch.equal(batch[n][i], batch[n][0]) for i in (1, 150, 299)), n
        a, b = one[n][0].double().cpu(), batch[n][0].double().cpu()
        step = torch.finfo(one[n].dtype).eps
        assert ((a - b).abs() <= step * b.abs() + 32 * 16 * 2.0 ** -24 * size[n][0] + 1e-30).all(), n


def test_results_are_the_same_from_run_to_run(gpu_device):
    print("[case] twice", flush=True)
    p, q, r = scan_problem(19, 2, 333, 200, 16, 2, torch.bfloat16), conv_problem(19, 3, 700, 200, 4, torch.bfloat16), norm_problem(19, (700,), 200, torch.bfloat16)
    for run in (lambda: run_scan(p, torch.bfloat16, gpu_device), lambda: run_conv(q, torch.bfloat16, gpu_device, act="silu"), lambda: run_norm(r, torch.bfloat16, gpu_device)):
        a, b = run(), run()
        assert all(torch.equal(a[n], b[n]) for n in a if a[n] is not None)


def test_far_into_large_tensors(gpu_device):
    """Strides past 32 bits."""
    from rnn_train_ring_attractor_amd import causal_conv_func, causal_conv_step, norm_gate_func, selective_scan_func, selective_scan_step
    print("[case] far strides", flush=True)
    B, T, C, N = 2, 40, 64, 16
    far = torch.empty((1 << 31) + 8 * B * T * C, dtype=torch.bfloat16, device=gpu_device)
    rows, weights = block_problem(21, B, T, C, N, 1, 4, torch.bfloat16, gpu_device)
    at, placed = 0, {}
    for n, t in rows.items():
        width = t[0, 0].numel()
        stride = (1 << 31, width, *((N, 1) if t.dim() == 4 else (1,)))
        placed[n] = far.as_strided(t.shape, stride, at).copy_(t)
        at += T * width
    with torch.no_grad():
        for a, b in zip(block(placed, weights, states=True), block(rows, weights, states=True)):
            assert torch.equal(a, b)
        states = [(torch.ones(B, 3, C, device=gpu_device, dtype=torch.bfloat16), torch.ones(B, C, N, device=gpu_device)) for _ in range(2)]
        for a, b in zip(block_token(placed, weights, 3, *states[0]), block_token(rows, weights, 3, *states[1])):
            assert torch.equal(a, b)
        assert all(torch.equal(a, b) for a, b in zip(*states))
    given = [torch.randn(B, T, C, device=gpu_device).bfloat16() for _ in range(2)]
    grads = []
    for r in (placed, rows):
        leaves = {n: t.detach().requires_grad_(True) for n, t in r.items()}
        grads.append(torch.autograd.grad(block(leaves, weights), list(leaves.values()), given))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_results_past_32_bits(gpu_device):
    """More than 2^32 results: equal sequences, equal results."""
    from rnn_train_ring_attractor_amd import causal_conv_func, norm_gate_func, selective_scan_func
    gen = torch.Generator(device=gpu_device).manual_seed(23)
    r = lambda *s: torch.randn(*s, generator=gen, device=gpu_device)
    B, T, C = 65, 1 << 14, 4096 + 8
    x = r(1, T, C).bfloat16()
    many = x.expand(B, T, C)
    assert many.numel() > 1 << 32
    with torch.no_grad():
        print("[case] convolution of 2^32 results", flush=True)
        w = r(C, 4)
        y, one = causal_conv_func(many, w), causal_conv_func(x, w)
        assert all(torch.equal(y[b], one[0]) for b in (0, 1, 63, 64))
        del y
        print("[case] norm of 2^32 results", flush=True)
        w = r(C)
        y, n = norm_gate_func(many, w, gate=many, residual=many, next_weight=w)
        a, b = norm_gate_func(x, w, gate=x, residual=x, next_weight=w)
        assert all(torch.equal(y[i], a[0]) and torch.equal(n[i], b[0]) for i in (0, 1, 63, 64))
        del y, n
        print("[case] scan of 2^32 results", flush=True)
        A, Bm = -torch.rand(C, 4, generator=gen, device=gpu_device), r(1, T, 1, 4).bfloat16()
        y = selective_scan_func(many, many, A, Bm.expand(B, T, 1, 4), Bm.expand(B, T, 1, 4), softplus=True)
        assert torch.equal(y[64], y[0]) and torch.equal(y[31], y[1]) and torch.equal(y[0], y[1]) and torch.isfinite(y[64]).all()
        part = selective_scan_func(x[:, :500], x[:, :500], A, Bm[:, :500], Bm[:, :500], softplus=True)
        # (cut into segments or not: a state's roundings)
        assert torch.allclose(part[0].float(), y[64, :500].float(), rtol=2.0 ** -7, atol=1e-3)


def test_sizes_past_31_bits_are_refused(gpu_device):
    from rnn_train_ring_attractor_amd import causal_conv_func, causal_conv_step, norm_gate_func, selective_scan_func, selective_scan_step
    n = (1 << 32) + 2
    one = lambda *s, dtype=torch.bfloat16: torch.zeros(1, device=gpu_device, dtype=dtype).expand(*s)
    w, A = torch.zeros(1, 4, device=gpu_device), torch.zeros(1, 2, device=gpu_device)
    print("[case] sizes past 31 bits", flush=True)
    with torch.no_grad():
        for call in (lambda: causal_conv_func(one(1, n, 1), w), lambda: causal_conv_step(one(n, 1), w, one(n, 3, 1)),
                     lambda: selective_scan_func(one(1, n, 1), one(1, n, 1), A, one(1, n, 1, 2), one(1, n, 1, 2)),
                     lambda: selective_scan_step(one(n, 1), one(n, 1), A, one(n, 1, 2), one(n, 1, 2), one(n, 1, 2, dtype=torch.float32)),
                     lambda: norm_gate_func(one(n * 2, 1), w[:, 0])):
            with pytest.raises((ValueError, torch.OutOfMemoryError)):
                call()


def test_empty_batches_and_sequences(gpu_device):
    from rnn_train_ring_attractor_amd import causal_conv_func, norm_gate_func, selective_scan_func
    print("[case] empty", flush=True)
    for B, T in ((0, 5), (2, 0)):
        for start in (False, True):
            p, q = scan_problem(25, B, T, 8, 4, 1, torch.float32, start=start), conv_problem(25, B, T, 8, 4, torch.float32, start=start)
            got, conv = run_scan(p, torch.float32, gpu_device), run_conv(q, torch.float32, gpu_device)
            assert got["y"].shape == (B, T, 8) and conv["y"].shape == (B, T, 8)
            for g in (got, conv):
                assert all((g[n] == 0).all() for n in g if n in ("dA", "dD", "dbias", "dweight"))
            if start:
                assert torch.equal(got["state"].double().cpu(), p["start"]) and torch.equal(got["dstart"].double().cpu(), p["de"])
                assert torch.equal(conv["state"].double().cpu(), q["start"]) and torch.equal(conv["dstart"].double().cpu(), q["de"])
            else:
                assert (got["state"] == 0).all() and (conv["state"] == 0).all()
    got = run_norm(norm_problem(25, (0, 3), 8, torch.float32), torch.float32, gpu_device)
    assert got["y"].shape == (0, 3, 8) and (got["dweight"] == 0).all() and (got["dnext_weight"] == 0).all()


# ------------------------------------------------------------------------------------------------
# Gradients asked for and not, broadcast inputs, runs again
# ------------------------------------------------------------------------------------------------
def _operators(dev):
    """{name: (call of tensors, tensors)}; a call's first outputs are differentiated"""
    from rnn_train_ring_attractor_amd import causal_conv_func, norm_gate_func, selective_scan_func
    gen = torch.Generator(device=dev).manual_seed(27)
    r = lambda *s: torch.randn(*s, generator=gen, device=dev)
    B, T, C, N, G, K = 2, 90, 24, 6, 2, 4
    return {
        "conv": (lambda x, w, b, s: causal_conv_func(x, w, b, initial_state=s, activation="silu", return_state=True), [r(B, T, C), r(C, K), r(C), r(B, K - 1, C)]),
        "scan": (lambda x, d, A, Bm, Cm, D, z, b, s: selective_scan_func(x, d, A, Bm, Cm, D=D, z=z, delta_bias=b, initial_state=s, softplus=True, return_state=True),
                 [r(B, T, C), r(B, T, C), -r(C, N).exp(), r(B, T, G, N), r(B, T, G, N), r(C), r(B, T, C), r(C), r(B, C, N)]),
        "norm": (lambda x, w, g, e, s, n: norm_gate_func(x, w, gate=g, residual=e, scale=s, next_weight=n), [r(B, T, C), r(C), r(B, T, C), r(B, T, C), r(C), r(C)]),
    }


@pytest.mark.parametrize("name", ["conv", "scan", "norm"])
def test_gradients_that_nobody_asks_for_and_runs_again(name, gpu_device):
    """What is frozen gets no gradient, the others what they are all together; a backward twice, a checkpoint and inference mode give the same bits."""
    from torch.utils.checkpoint import checkpoint
    call, tensors = _operators(gpu_device)[name]
    leaves = [t.clone().requires_grad_(True) for t in tensors]
    out = call(*leaves)
    given = [torch.randn_like(o) for o in out]
    full = torch.autograd.grad(out, leaves, given, retain_graph=True)
    again = torch.autograd.grad(out, leaves, given)
    kept = torch.autograd.grad(checkpoint(call, *leaves, use_reentrant=False), leaves, given)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(full, again, kept))
    with torch.inference_mode():
        assert all(torch.equal(a, b) for a, b in zip(call(*tensors), out))
    n = len(tensors)
    for mask in [1 << i for i in range(n)] + [(1 << n) - 1 - (1 << i) for i in range(n)]:
        print(f"[case] frozen {name} {mask}", flush=True)
        some = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate(tensors)]
        wanted = [t for t in some if t.requires_grad]
        got = iter(torch.autograd.grad(call(*some), wanted, given))
        for i, t in enumerate(some):
            if t.requires_grad:
                assert torch.equal(next(got), full[i]), (mask, i)
    # each output's gradient alone: the two add up (sums of two parts of up to T N terms, in one order and another)
    parts = []
    for k in range(2):
        some = [t.clone().requires_grad_(True) for t in tensors]
        g = torch.autograd.grad(call(*some)[k], some, given[k], allow_unused=True)
        parts.append([torch.zeros_like(t) if x is None else x for t, x in zip(some, g)])
    for a, b, c in zip(full, *parts):
        assert ((b + c - a).norm() <= 2.0 ** -24 * 400 * (b.norm() + c.norm()) + 1e-30)


@pytest.mark.parametrize("name", ["conv", "scan", "norm"])
def test_broadcast_inputs(name, gpu_device):
    """A broadcast input reads like its copy, and its gradient is the sum over what it was broadcast to; a gradient that is one expanded value likewise."""
    call, tensors = _operators(gpu_device)[name]
    for i, t in enumerate(tensors):
        if t.dim() < 2 or t.shape[0] != 2:
            continue
        print(f"[case] broadcast {name} {i}", flush=True)
        one = t[:1].clone().requires_grad_(True)
        full = one.detach().expand_as(t).contiguous().requires_grad_(True)
        out = [call(*tensors[:i], x, *tensors[i + 1:]) for x in (one.expand_as(t), full)]
        assert all(torch.equal(a, b) for a, b in zip(*out))
        given = [torch.randn_like(o) for o in out[0]]
        part, whole = torch.autograd.grad(out[0], one, given)[0], torch.autograd.grad(out[1], full, given)[0]
        assert torch.allclose(part, whole.sum(0, keepdim=True), rtol=2.0 ** -22, atol=2.0 ** -22 * float(whole.abs().max()))
    leaves = [t.clone().requires_grad_(True) for t in tensors]
    out = call(*leaves)
    a = torch.autograd.grad(out[0].sum(), leaves, retain_graph=True, allow_unused=True)
    b = torch.autograd.grad(out[0], leaves, torch.ones_like(out[0]), allow_unused=True)
    assert all(x is y or torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("name", ["conv", "scan", "norm"])
def test_gradients_are_differences(name, gpu_device):
    """Along random directions, in fp32 with a step of 2^-7: the difference's own error is the step squared (third derivatives of order ten) and the
    results' roundings over the step; of directions of thousands of elements the norm is a hundred."""
    call, tensors = _operators(gpu_device)[name]
    tensors = [t * 0.5 for t in tensors]
    leaves = [t.clone().requires_grad_(True) for t in tensors]
    out = call(*leaves)
    given = [torch.randn_like(o) for o in out]
    grads = torch.autograd.grad(out, leaves, given)
    value = lambda ts: sum(float((o.double() * g.double()).sum()) for o, g in zip(call(*ts), given))
    for i, t in enumerate(tensors):
        print(f"[case] difference {name} {i}", flush=True)
        d = torch.randn_like(t)
        d, step = d / d.norm(), 2.0 ** -4
        with torch.no_grad():
            num = (value([*tensors[:i], t + step * d, *tensors[i + 1:]]) - value([*tensors[:i], t - step * d, *tensors[i + 1:]])) / (2 * step)
        got = float((grads[i].double() * d.double()).sum())
        assert abs(num - got) <= 0.02 * float(grads[i].norm()) + 1e-3, (i, num, got)


# ------------------------------------------------------------------------------------------------
# What watches operators
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("name", ["conv", "scan", "norm"])
def test_what_watches_the_operators_sees_them(name, gpu_device):
    """Forward mode and function transforms, which they have no rules for, are refused instead of losing the derivative; a trace records the call."""
    import torch.autograd.forward_ad as forward
    call, tensors = _operators(gpu_device)[name]
    x = tensors[0]
    op = lambda t: call(t, *tensors[1:])[0]
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
    leaf = x.clone().requires_grad_(True)
    y = op(leaf)
    g = torch.ones_like(y)
    want, = torch.autograd.grad(y, leaf, g, retain_graph=True)
    with forward.dual_level():
        assert torch.equal(torch.autograd.grad(y, leaf, g, retain_graph=True)[0], want)
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.autograd.grad(y, leaf, forward.make_dual(g, g))
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(op(leaf).sum(), leaf, create_graph=True)


def test_what_watches_single_tokens(gpu_device):
    import torch.autograd.forward_ad as forward
    from rnn_train_ring_attractor_amd import causal_conv_step, selective_scan_step
    r = lambda *s: torch.randn(*s, device=gpu_device)
    w, A, Bm = r(8, 4), -r(8, 6).exp(), r(2, 1, 6)
    for step, x, s in ((lambda x, s: causal_conv_step(x, w, s), r(2, 8), r(2, 3, 8)), (lambda x, s: selective_scan_step(x, x, A, Bm, Bm, s), r(2, 8), r(2, 8, 6))):
        want, before = step(x, s.clone()), s.clone()
        with forward.dual_level():
            assert torch.equal(step(x, s.clone()), want)
            for a, b in ((forward.make_dual(x, x), s), (x, forward.make_dual(s, s))):
                with pytest.raises(RuntimeError, match="no gradient"):
                    step(a, b)
        for transformed in (lambda: torch.func.jvp(lambda t: step(t, s), (x,), (x,)), lambda: torch.func.vmap(lambda t: step(t, s))(x[None]),
                            lambda: torch.func.grad(lambda t: step(t, s).sum())(x), lambda: torch.jit.trace(step, (x, s))):
            with pytest.raises(RuntimeError):
                transformed()
        assert torch.equal(s, before)
        with pytest.raises(RuntimeError, match="no gradient"):
            step(x.clone().requires_grad_(True), s)
        version = s._version
        step(x, s)
        assert s._version > version                              # autograd sees that the state was written to


@pytest.mark.parametrize("name", ["conv", "scan", "norm"])
def test_negated_views_are_read_as_they_are_meant(name, gpu_device):
    """Tensors that torch keeps negated lazily, as inputs, parameters and gradients."""
    call, tensors = _operators(gpu_device)[name]
    print(f"[case] negated {name}", flush=True)
    results = []
    for of in (lambda t: torch._neg_view(-t), lambda t: t):
        leaves = [of(t).detach().requires_grad_(True) for t in tensors]
        assert results or all(t.is_neg() for t in leaves)
        gen = torch.Generator(device=gpu_device).manual_seed(29)
        out = call(*leaves)
        given = [of(torch.randn(o.shape, generator=gen, device=gpu_device)) for o in out]
        results.append([*out, *torch.autograd.grad(out, leaves, given)])
        with torch.no_grad():
            results[-1] += call(*leaves)
    for i, (a, b) in enumerate(zip(*results)):
        assert torch.equal(a, b), i


# ------------------------------------------------------------------------------------------------
# Infinities and NaN
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", list(TYPES))
def test_what_is_not_finite_reaches_rows_that_see_it_only(kind, gpu_device):
    """Of a channel at a token: the convolution's next taps, the scan's tokens from there on in that channel, the norm's row."""
    dtype, T, C, N = TYPES[kind], 70, 20, 5
    for at in (0, 33, T - 1):
        for value in (math.inf, math.nan):
            print(f"[case] {value} at {at} {kind}", flush=True)
            p = conv_problem(31, 2, T, C, 4, dtype)
            clean = run_conv(p, dtype, gpu_device, act="silu")
            bad = {n: None if t is None else t.clone() for n, t in p.items()}
            bad["x"][0, at, 3] = value
            got = run_conv(bad, dtype, gpu_device, act="silu")
            seen = torch.zeros(2, T, C, dtype=torch.bool, device=gpu_device)
            seen[0, at:at + 4, 3] = True
            assert torch.equal(got["y"][~seen], clean["y"][~seen]) and not torch.isfinite(got["y"][0, at, 3])
            back = torch.zeros_like(seen)                                # gradients behind the slope of what saw it
            back[0, max(0, at - 3):at + 4, 3] = True
            assert torch.equal(got["dx"][~back], clean["dx"][~back])
            for n in ("dweight", "dbias"):
                rest = [c for c in range(C) if c != 3]
                assert torch.equal(got[n][rest], clean[n][rest]), n
            p = scan_problem(33, 2, T, C, N, 2, dtype)
            clean = run_scan(p, dtype, gpu_device)
            for n in ("x", "delta", "z"):
                bad = {m: None if t is None else t.clone() for m, t in p.items()}
                bad[n][0, at, 3] = value
                got = run_scan(bad, dtype, gpu_device)
                seen = torch.zeros(2, T, C, dtype=torch.bool, device=gpu_device)
                seen[0, at:at + 1 if n == "z" else T, 3] = True
                assert torch.equal(got["y"][~seen], clean["y"][~seen]), n
                if n != "delta" or math.isnan(value):
                    assert not torch.isfinite(got["y"][0, at, 3]) or n == "z", n
                rest = [c for c in range(C) if c != 3]
                for m in ("dx", "ddelta", "dz", "dstart", "state"):
                    assert torch.equal(got[m][1], clean[m][1]), (n, m)
                    a, b = (t[m][0] if m in ("dstart", "state") else t[m][0].transpose(0, 1) for t in (got, clean))
                    assert torch.equal(a[rest], b[rest]), (n, m)
                assert torch.equal(got["dA"][rest], clean["dA"][rest]) and torch.equal(got["dD"][rest], clean["dD"][rest])
                assert torch.equal(got["dB"][1], clean["dB"][1]) and torch.equal(got["dC"][:, :at], clean["dC"][:, :at]) or n == "z"
                if n == "x" and at == T - 1:                             # (no state that holds it takes part in dA)
                    assert torch.equal(got["dA"], clean["dA"])
            p = norm_problem(35, (2, T), C, dtype)
            clean = run_norm(p, dtype, gpu_device, group=5)
            bad = {m: None if t is None else t.clone() for m, t in p.items()}
            bad["x"][0, at, 3] = value
            got = run_norm(bad, dtype, gpu_device, group=5)
            rows = torch.ones(2, T, dtype=torch.bool, device=gpu_device)
            rows[0, at] = False
            for m in ("y", "n", "dx", "dgate", "dresidual"):
                assert torch.equal(got[m][rows], clean[m][rows]), m
            assert torch.equal(got["y"][0, at, 5:], clean["y"][0, at, 5:]) and not torch.isfinite(got["y"][0, at, :5]).all()


# ------------------------------------------------------------------------------------------------
# Refusals
# ------------------------------------------------------------------------------------------------
def test_refusals_on_the_gpu(gpu_device):
    from rnn_train_ring_attractor_amd import causal_conv_func, causal_conv_step, norm_gate_func, selective_scan_func, selective_scan_step
    z = lambda *s, **k: torch.zeros(*s, device=gpu_device, **k)
    x, w = z(2, 3, 8), z(8, 4)
    ok = lambda **o: causal_conv_func(**{**dict(x=x, weight=w), **o})
    assert ok().shape == (2, 3, 8) and torch.equal(ok(lengths=torch.tensor([1, 1 << 40], device=gpu_device)), ok())
    for error, bad in ((ValueError, dict(x=x[0])), (ValueError, dict(weight=z(8))), (ValueError, dict(weight=z(7, 4))), (ValueError, dict(weight=z(8, 9))), (ValueError, dict(weight=z(8, 0))),
                       (TypeError, dict(weight=w.bfloat16())), (TypeError, dict(x=x.long())), (ValueError, dict(bias=z(7))), (TypeError, dict(bias=z(8).half())),
                       (ValueError, dict(initial_state=z(2, 4, 8))), (TypeError, dict(initial_state=z(2, 3, 8).bfloat16())), (ValueError, dict(lengths=z(3, dtype=torch.int32))),
                       (TypeError, dict(lengths=z(2))), (RuntimeError, dict(lengths=torch.zeros(2, dtype=torch.int32))), (ValueError, dict(activation="relu")),
                       (RuntimeError, dict(weight=w.cpu())), (ValueError, dict(x=z(2, 3, 0), weight=z(0, 4)))):
        with pytest.raises(error):
            ok(**bad)
    step = lambda **o: causal_conv_step(**{**dict(x=x[:, 0], weight=w, state=z(2, 3, 8)), **o})
    assert step().shape == (2, 8) and causal_conv_step(x[:0, 0], w, z(0, 3, 8)).shape == (0, 8)
    for error, bad in ((ValueError, dict(state=z(2, 4, 8))), (RuntimeError, dict(state=z(2, 8, 3).transpose(1, 2))), (RuntimeError, dict(state=z(1, 1, 8).expand(2, 3, 8))),
                       (TypeError, dict(state=z(2, 3, 8).half())), (TypeError, dict(active=z(2))), (ValueError, dict(active=z(3, dtype=torch.bool))),
                       (RuntimeError, dict(state=torch._neg_view(z(2, 3, 8))))):
        with pytest.raises(error):
            step(**bad)
    A, Bm = z(8, 4), z(2, 3, 2, 4)
    ok = lambda **o: selective_scan_func(**{**dict(x=x, delta=x, A=A, B=Bm, C=Bm), **o})
    assert ok().shape == (2, 3, 8)
    for error, bad in ((ValueError, dict(x=x[0])), (ValueError, dict(delta=z(2, 3, 7))), (TypeError, dict(delta=x.half())), (ValueError, dict(A=z(8))), (ValueError, dict(A=z(7, 4))),
                       (TypeError, dict(A=A.double())), (ValueError, dict(B=z(2, 3, 2, 5))), (ValueError, dict(C=z(2, 3, 1, 4))), (ValueError, dict(B=z(2, 3, 4))),
                       (ValueError, dict(B=z(2, 3, 3, 4), C=z(2, 3, 3, 4))), (TypeError, dict(C=Bm.half())), (ValueError, dict(D=z(7))), (ValueError, dict(z=z(2, 3, 7))),
                       (ValueError, dict(delta_bias=z(1))), (ValueError, dict(initial_state=z(2, 4, 8))), (TypeError, dict(initial_state=z(2, 8, 4).half())),
                       (ValueError, dict(A=z(8, 65), B=z(2, 3, 2, 65), C=z(2, 3, 2, 65))), (ValueError, dict(lengths=z(1, dtype=torch.int64)))):
        with pytest.raises(error):
            ok(**bad)
    step = lambda **o: selective_scan_step(**{**dict(x=x[:, 0], delta=x[:, 0], A=A, B=Bm[:, 0], C=Bm[:, 0], state=z(2, 8, 4)), **o})
    assert step().shape == (2, 8)
    for error, bad in ((ValueError, dict(state=z(2, 4, 8))), (RuntimeError, dict(state=z(2, 4, 8).transpose(1, 2))), (RuntimeError, dict(A=A.clone().requires_grad_(True))),
                       (ValueError, dict(active=z(3, dtype=torch.uint8))), (RuntimeError, dict(state=z(1, 8, 4).expand(2, 8, 4)))):
        with pytest.raises(error):
            step(**bad)
    ok = lambda **o: norm_gate_func(**{**dict(x=x, weight=z(8)), **o})
    assert ok().shape == (2, 3, 8) and len(ok(next_weight=z(8))) == 2 and norm_gate_func(z(8), z(8)).shape == (8,)
    for error, bad in ((ValueError, dict(weight=z(7))), (TypeError, dict(weight=z(8).half())), (TypeError, dict(weight=None)), (ValueError, dict(gate=z(2, 3, 7))),
                       (TypeError, dict(residual=x.half())), (ValueError, dict(scale=z(1))), (ValueError, dict(next_weight=z(7))), (ValueError, dict(group=3)), (ValueError, dict(group=0)),
                       (ValueError, dict(kind="batch")), (ValueError, dict(activation="relu")), (ValueError, dict(eps=-1.0)), (ValueError, dict(eps=math.nan)),
                       (ValueError, dict(x=z(1, 8193), weight=z(8193))), (ValueError, dict(x=z(2, 0), weight=z(0))), (RuntimeError, dict(gate=x.cpu())), (ValueError, dict(x=z(())))):
        with pytest.raises(error):
            ok(**bad)
