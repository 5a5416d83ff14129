"""The sequence operators as they are used: together in a layer, recorded into graphs, on streams of their own, far into large tensors,
in the training driver, and what they refuse on a GPU."""
import math

import pytest
import torch

from oracle import sequence_oracle as O

pytestmark = pytest.mark.gpu

SEED = 0x1234567890ABCDEF


def _layer_problem(seed, B, T, H, G, D, dtype):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64).to(dtype).double()
    return {"q": r(B, T, H, D), "k": r(B, T, G, D), "v": r(B, T, G, D), "x": r(B, T, H * D), "dy": r(B, T, H * D),
            "g": torch.log1p(-torch.exp2(-torch.linspace(2.0, 7.0, H))).double()}


def _layer(q, k, v, x, g, positions, f, p, offset):
    """x + dropout(attention of turned queries and keys)"""
    from rnn_train_ring_attractor_amd import dropout_func, linear_attention_func, rotary_func
    q, k = rotary_func((q, k), positions, f)
    o = linear_attention_func(q, k, v, g)
    return dropout_func(o.flatten(2), p, SEED, offset, residual=x)


def _on(dev, dtype, problem):
    return [problem[n].to(dtype).to(dev).requires_grad_(True) for n in ("q", "k", "v", "x")]


def test_layer_and_its_gradients(gpu_device):
    """fp32.  Bound: the operators' own (K 2^-24 of the terms' magnitudes each, K = 128 tokens + heads' widths + 256) one behind the
    other; magnitudes bounded by the operator of magnitudes with turned pairs replaced by |a| + |b| on both places."""
    B, T, H, G, D, p, offset = 2, 130, 4, 2, 32, 0.25, 77
    print("[case] layer", flush=True)
    z = _layer_problem(3, B, T, H, G, D, torch.float32)
    f = 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))
    positions = torch.arange(50000, 50000 + T)
    keep = torch.from_numpy(O.keep_mask(B * T * H * D, p, SEED, offset)).view(B, T, H * D)

    def reference(q, k, v, x, dy, magnitudes):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v, x)]
        turn = (lambda t: torch.cat([t[..., :D // 2] + t[..., D // 2:]] * 2, -1)) if magnitudes else \
               (lambda t: _rotary_differentiable(t, positions, f))
        o, _ = O.attention(turn(leaves[0]), turn(leaves[1]), leaves[2], z["g"])
        y = leaves[3] + torch.where(keep, o.flatten(2) / (1 - p), 0.0)
        y.backward(dy)
        return [y.detach()] + [t.grad for t in leaves]

    want = reference(*(z[n] for n in ("q", "k", "v", "x", "dy")), False)
    size = reference(*(z[n].abs() for n in ("q", "k", "v", "x", "dy")), True)
    leaves = _on(gpu_device, torch.float32, z)
    y = _layer(*leaves, z["g"].float().to(gpu_device), positions.to(gpu_device), f.to(gpu_device), p, offset)
    grads = torch.autograd.grad([y], leaves, [z["dy"].float().to(gpu_device)])
    for name, got, w, s in zip(("y", "dq", "dk", "dv", "dx"), [y, *grads], want, size):
        err = (got.detach().double().cpu() - w).abs()
        assert (err <= 3 * (T + 2 * D + 256) * 2.0 ** -24 * s).all(), (name, float((err / s).max() * 2 ** 24))


def _rotary_differentiable(x, positions, f):
    a = positions.double()[:, None] * f
    c, s = torch.cos(a)[None, :, None], torch.sin(a)[None, :, None]
    h = x.shape[-1] // 2
    u, w = x[..., :h], x[..., h:]
    return torch.cat([u * c - w * s, w * c + u * s], -1)


@pytest.mark.parametrize("T", [60, 2100])
def test_recorded_layer_replays_as_it_runs(T, gpu_device):
    """Forward and backward of the layer in a graph, the dropout's offset advanced by the graph: every replay on new inputs has the bits of
    the eager call, with eager calls of other sizes between the replays."""
    B, H, G, D = 2, 2, 1, 64
    print(f"[case] recorded layer T={T}", flush=True)
    dtype = torch.bfloat16
    f = (10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))).to(gpu_device)
    positions = torch.arange(T, device=gpu_device)
    z = _layer_problem(5, B, T, H, G, D, dtype)
    g = z["g"].float().to(gpu_device)
    static = [t.detach().clone() for t in _on(gpu_device, dtype, z)]
    dy = z["dy"].to(dtype).to(gpu_device)
    counter = torch.zeros(1, dtype=torch.int64, device=gpu_device)

    def step(tensors, offset):
        leaves = [t.detach().requires_grad_(True) for t in tensors]
        y = _layer(*leaves, g, positions, f, 0.2, offset)
        return [y.detach()] + list(torch.autograd.grad([y], leaves, [dy]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static, counter)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static, counter)
        counter.add_(1)
    gen = torch.Generator(device=gpu_device).manual_seed(9)
    for i in range(4):
        for t in static:
            t.copy_(torch.randn(t.shape, generator=gen, device=gpu_device))
        want = step(static, i)
        other = [t[:, :7 + i].contiguous() for t in static]
        y = _layer(*other, g, positions[:7 + i], f, 0.2, 3)          # other eager work of the same operators
        graph.replay()
        torch.cuda.synchronize()
        assert torch.isfinite(y).all()
        for a, b in zip(out, want):
            assert torch.equal(a, b), i
    assert int(counter) == 4


def test_two_graphs_and_two_streams_at_once(gpu_device):
    """Calls side by side have the bits of calls alone: workspaces are a call's own."""
    from rnn_train_ring_attractor_amd import linear_attention_func
    print("[case] streams", flush=True)
    gen = torch.Generator(device=gpu_device).manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=gen, device=gpu_device).bfloat16()
    g = -torch.rand(4, generator=gen, device=gpu_device) * 0.1
    sets = [[r(1, 3000, 4, 64) for _ in range(3)] for _ in range(2)]
    with torch.no_grad():
        want = [linear_attention_func(*s, g, return_state=True) for s in sets]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in sets]
        got = [[], []]
        for st in streams:
            st.wait_stream(torch.cuda.current_stream())
        for _ in range(5):
            for i, st in enumerate(streams):
                with torch.cuda.stream(st):
                    got[i].append(linear_attention_func(*sets[i], g, return_state=True))
        torch.cuda.synchronize()
        for i in range(2):
            for o, s in got[i]:
                assert torch.equal(o, want[i][0]) and torch.equal(s, want[i][1])
        graphs, outs = [], []
        for s in sets:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(linear_attention_func(*s, g, return_state=True))
            graphs.append(graph)
        for _ in range(3):
            for i, st in enumerate(streams):
                with torch.cuda.stream(st):
                    graphs[i].replay()
            torch.cuda.synchronize()
            for i in range(2):
                assert torch.equal(outs[i][0], want[i][0]) and torch.equal(outs[i][1], want[i][1])


def test_far_into_large_tensors(gpu_device):
    """Strides and element numbers past 32 bits."""
    from rnn_train_ring_attractor_amd import dropout_func, linear_attention_func, linear_attention_step, rotary_func
    print("[case] far strides", flush=True)
    gen = torch.Generator(device=gpu_device).manual_seed(6)
    B, T, H, D = 2, 40, 2, 64
    small = torch.randn(3, B, T, H, D, generator=gen, device=gpu_device).bfloat16()
    g = torch.tensor([-0.1, -0.01], device=gpu_device)
    far = torch.empty((1 << 31) + 3 * B * T * H * D, dtype=torch.bfloat16, device=gpu_device)

    def place(x, at):
        y = far.as_strided(x.shape, (1 << 31, H * D, D, 1), at)
        y.copy_(x)
        return y

    q, k, v = (place(small[i], i * T * H * D) for i in range(3))
    with torch.no_grad():
        want, got = linear_attention_func(*small, g, return_state=True), linear_attention_func(q, k, v, g, return_state=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        states = [torch.zeros(B, H, D, D, device=gpu_device) for _ in range(2)]
        steps = [linear_attention_step(a[:, 3], b[:, 3], c[:, 3], g, s) for (a, b, c), s in zip(((q, k, v), small), states)]
        assert torch.equal(*steps) and torch.equal(*states)
        f = torch.ones(D // 2, dtype=torch.float64, device=gpu_device)
        pos = torch.arange(T, device=gpu_device)
        assert torch.equal(rotary_func(q, pos, f), rotary_func(small[0], pos, f))
        print("[case] dropout past 2^32 values", flush=True)
        del far, q, k, v
        n = (1 << 32) + 1003
        x = torch.ones(n, dtype=torch.bfloat16, device=gpu_device)
        y = dropout_func(x, 0.5, SEED, 5)
        for first in (0, (1 << 32) - 500, n - 1003):
            keep = torch.from_numpy(O.keep_mask(1000, 0.5, SEED, 5, first=first)).to(gpu_device)
            assert torch.equal(y[first:first + 1000] != 0, keep)


def test_results_past_32_bits_and_more_tokens_than_workgroups(gpu_device):
    from rnn_train_ring_attractor_amd import dropout_func, linear_attention_func, linear_attention_step, rotary_func
    gen = torch.Generator(device=gpu_device).manual_seed(16)
    with torch.no_grad():
        print("[case] attention of 2^32 results: equal heads, equal results", flush=True)
        T, H, D = 1 << 20, 65, 64
        q, k, v = (torch.randn(1, T, 1, D, generator=gen, device=gpu_device).bfloat16().expand(1, T, H, D) for _ in range(3))
        o, s = linear_attention_func(q, k, v, torch.full((H,), -0.05, device=gpu_device), return_state=True)
        assert o.numel() > 1 << 32
        for at in (slice(0, 1000), slice(T // 2, T // 2 + 1000), slice(T - 1000, T)):
            assert all(torch.equal(o[:, at, h], o[:, at, 0]) for h in (1, 31, 63, 64))
        assert torch.equal(s, s[:, :1].expand_as(s))
        part = linear_attention_func(*(x[:, T - 1000:, :1] for x in (q, k, v)), torch.full((1,), -0.05, device=gpu_device), return_state=True)
        # exp(-0.05 * 500) of what came before is left: the two differ by their roundings
        assert torch.allclose(o[:, -500:, :1].float(), part[0][:, -500:].float(), rtol=2.0 ** -6, atol=2.0 ** -4)
        del o, s
        print("[case] step of 2^32 state values", flush=True)
        B, D = 66000, 256
        state = torch.zeros(B, 1, D, D, device=gpu_device)
        row = torch.randn(3, 1, 1, D, generator=gen, device=gpu_device)
        g, few = torch.full((1,), -0.1, device=gpu_device), torch.zeros(3, 1, D, D, device=gpu_device)
        for _ in range(2):
            got = linear_attention_step(*(x.expand(B, 1, D) for x in row), g, state)
            want = linear_attention_step(*(x.expand(3, 1, D) for x in row), g, few)
        assert torch.allclose(got[-3:], want, rtol=1e-4, atol=1e-4) and torch.allclose(got[:3], want, rtol=1e-4, atol=1e-4)
        assert torch.equal(state[-3:], few) and torch.equal(state[B // 2:B // 2 + 3], few)
        del state
        print("[case] positions of more tokens than workgroups", flush=True)
        T, D = (1 << 20) + 1003, 512                                     # a token fills a workgroup
        x = torch.randn(1, T, 1, D, generator=gen, device=gpu_device).bfloat16()
        f = torch.rand(D // 2, generator=gen, device=gpu_device, dtype=torch.float64)
        pos = torch.arange(T, device=gpu_device)
        for layout in ("half", "interleaved"):
            y = rotary_func(x, pos, f, layout)
            for at in (slice(0, 2000), slice((1 << 20) - 1000, (1 << 20) + 1003)):
                assert torch.equal(y[:, at], rotary_func(x[:, at], pos[at], f, layout))
        del x, y
        print("[case] results that pass the caches", flush=True)
        for dtype in (torch.float32, torch.float16):
            x = torch.randn(5, 4097, 4100, generator=gen, device=gpu_device).to(dtype)
            y, both = dropout_func(x, 0.25, SEED, 9), dropout_func(x, 0.25, SEED, 9, residual=x)
            n = 1000 * 4100
            assert torch.equal(y.view(-1)[:n], dropout_func(x.view(-1)[:n], 0.25, SEED, 9))      # (a mask by index: the same from the front)
            keep = torch.from_numpy(O.keep_mask(1000, 0.25, SEED, 9, first=y.numel() - 1000)).to(gpu_device)
            assert torch.equal(y.view(-1)[-1000:] != 0, keep & (x.view(-1)[-1000:] != 0))
            kept = y != 0
            assert torch.equal(both[~kept], x[~kept]) and (both[kept] != x[kept]).float().mean() > 0.99
            scaled = x[kept].float() * (1 / (1 - 0.25))
            assert torch.equal(y[kept], scaled.to(dtype))
            # product and sum in fp32, half a step each (none for the product where both are one instruction), then half a step of the type
            total = x[kept].double() * (1 + float(torch.tensor(1 / (1 - 0.25))))
            bound = 2.0 ** -24 * (scaled.abs().double() + 1.001 * total.abs()) + 1.001 * torch.finfo(dtype).eps / 2 * total.abs() + 2.0 ** -25
            assert ((both[kept].double() - total).abs() <= bound).all()


def test_positions_of_every_kind_and_gradients_of_gradients(gpu_device):
    from rnn_train_ring_attractor_amd import dropout_func, linear_attention_func, rotary_func
    print("[case] positions", flush=True)
    gen = torch.Generator(device=gpu_device).manual_seed(8)
    x = torch.randn(3, 6, 2, 16, generator=gen, device=gpu_device)
    f = torch.rand(4, generator=gen, device=gpu_device, dtype=torch.float64)
    pos = torch.randint(0, 1 << 20, (6,), generator=gen, device=gpu_device)
    want = rotary_func(x, pos, f)
    for p in (pos.int(), pos[None].expand(3, 6), pos.float(), pos.repeat(3, 1).t().contiguous().t()):
        assert torch.equal(rotary_func(x, p, f), want)
    assert torch.equal(rotary_func((x, x[:, :, :1]), pos, f)[1], want[:, :, :1])
    timed = x.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(rotary_func(timed, pos, f), want)
    a = x.clone().requires_grad_(True)
    for op in (lambda t: rotary_func(t, pos, f), lambda t: dropout_func(t, 0.3, 5, 6)):
        grad, = torch.autograd.grad([(op(a) ** 2).sum()], [a], create_graph=True)
        second, = torch.autograd.grad([grad.sum()], [a])
        # y = M x with M fixed: the gradient is 2 M^T M x, its sum's 2 M^T M 1
        ones = torch.ones_like(a).requires_grad_(True)
        want2, = torch.autograd.grad([(op(ones) ** 2).sum()], [ones])
        assert torch.allclose(second, want2, rtol=1e-5, atol=1e-5)
    q = x[..., :8].clone().requires_grad_(True)
    o = linear_attention_func(q, q, q, torch.zeros(2, device=gpu_device))
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad([o.sum()], [q], create_graph=True)


def test_backward_twice_broadcast_inputs_checkpoints_and_inference(gpu_device):
    """The same bits from a backward run twice over one forward (which kept its states), from a forward that is formed again, and under
    inference mode; a broadcast input's gradient is the sum over what it was broadcast to; inputs that ask for no gradient get none."""
    from torch.utils.checkpoint import checkpoint
    from rnn_train_ring_attractor_amd import dropout_func, linear_attention_func, linear_attention_step, rotary_func
    gen = torch.Generator(device=gpu_device).manual_seed(18)
    B, T, H, D = 2, 700, 4, 32
    q, k, v, do = (torch.randn(B, T, H, D, generator=gen, device=gpu_device) for _ in range(4))
    g, f = torch.linspace(-0.3, -0.001, H, device=gpu_device), torch.rand(8, generator=gen, device=gpu_device, dtype=torch.float64)
    pos = torch.arange(T, device=gpu_device)

    def layer(q, k, v):
        a, b = rotary_func((q, k), pos, f)
        return dropout_func(linear_attention_func(a, b, v, g), 0.2, 3, 4, residual=q)

    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    print("[case] twice", flush=True)
    o = layer(*leaves)
    first = torch.autograd.grad(o, leaves, do, retain_graph=True)
    second = torch.autograd.grad(o, leaves, do)
    print("[case] checkpoint", flush=True)
    again = torch.autograd.grad(checkpoint(layer, *leaves, use_reentrant=False), leaves, do)
    for other in (second, again):
        assert all(torch.equal(a, b) for a, b in zip(first, other))
    print("[case] some gradients", flush=True)
    only, = torch.autograd.grad(layer(q, k, leaves[2]), leaves[2:], do)
    assert torch.equal(only, first[2])
    print("[case] broadcast", flush=True)
    one = torch.randn(1, T, 1, D, generator=gen, device=gpu_device).requires_grad_(True)
    o1 = linear_attention_func(leaves[0], one.expand(B, T, H, D), leaves[2], g)
    full = one.detach().expand(B, T, H, D).contiguous().requires_grad_(True)
    o2 = linear_attention_func(leaves[0], full, leaves[2], g)
    assert torch.equal(o1, o2)
    whole, = torch.autograd.grad(o2, full, do)
    part, = torch.autograd.grad(o1, one, do)
    # two orders of a sum of B H terms: off by at most B H half steps of the terms' magnitudes each
    assert ((part - whole.sum((0, 2), keepdim=True)).abs() <= 2 * B * H * 2.0 ** -24 * whole.abs().sum((0, 2), keepdim=True)).all()
    print("[case] broadcast gradient", flush=True)
    summed, = torch.autograd.grad(linear_attention_func(q, k, leaves[2], g).sum(), leaves[2:])
    ones, = torch.autograd.grad(linear_attention_func(q, k, leaves[2], g), leaves[2:], torch.ones_like(do))
    assert torch.equal(summed, ones)
    print("[case] inference", flush=True)
    with torch.inference_mode():
        assert torch.equal(layer(q, k, v), o)
        state = torch.zeros(B, H, D, D, device=gpu_device)
        steps = [linear_attention_step(q[:, t], k[:, t], v[:, t], g, state) for t in range(3)]
    with torch.no_grad():
        want = linear_attention_func(q[:, :3], k[:, :3], v[:, :3], g)
    size = linear_attention_func(q[:, :3].abs(), k[:, :3].abs(), v[:, :3].abs(), g)
    assert ((torch.stack(steps, dim=1) - want).abs() <= 2 * (3 + 2 * D + 256) * 2.0 ** -24 * size).all()


def test_refusals_on_the_gpu(gpu_device):
    from rnn_train_ring_attractor_amd import dropout_func, linear_attention_func, linear_attention_step, rotary_func
    z = lambda *s, **k: torch.zeros(*s, device=gpu_device, **k)
    q, k, v, g, s = z(2, 3, 4, 8), z(2, 3, 2, 8), z(2, 3, 2, 6), z(4), z(2, 4, 8, 6)
    ok = lambda **o: linear_attention_func(**{**dict(q=q, k=k, v=v, log_decay=g), **o})
    assert ok().shape == (2, 3, 4, 6) and ok(q=q[:, :0], k=k[:, :0], v=v[:, :0]).shape == (2, 0, 4, 6)
    assert torch.equal(ok(q=q[:0], k=k[:0], v=v[:0], return_state=True)[1], z(0, 4, 8, 6))
    for error, bad in ((ValueError, dict(k=z(2, 3, 3, 8), v=z(2, 3, 3, 6))), (ValueError, dict(k=z(2, 3, 2, 7))), (ValueError, dict(v=z(2, 4, 2, 6))),
                       (TypeError, dict(k=k.bfloat16())), (TypeError, dict(q=q.long())), (ValueError, dict(log_decay=z(3))),
                       (TypeError, dict(log_decay=g.double())), (ValueError, dict(log_decay=g.clone().requires_grad_(True))),
                       (ValueError, dict(initial_state=z(2, 4, 6, 8))), (TypeError, dict(initial_state=s.bfloat16())),
                       (ValueError, dict(lengths=z(3, dtype=torch.int32))), (TypeError, dict(lengths=z(2))),
                       (RuntimeError, dict(lengths=torch.zeros(2, dtype=torch.int32))),
                       (ValueError, dict(q=z(1, 1, 1, 300), k=z(1, 1, 1, 300), v=z(1, 1, 1, 6), log_decay=z(1)))):
        with pytest.raises(error):
            ok(**bad)
    assert torch.equal(ok(lengths=torch.tensor([1, 1 << 40], device=gpu_device)), ok())
    step = lambda **o: linear_attention_step(**{**dict(q=q[:, 0], k=k[:, 0], v=v[:, 0], log_decay=g, state=s), **o})
    before = s._version
    assert step().shape == (2, 4, 6) and s._version > before             # autograd sees that the state was written to
    for error, bad in ((RuntimeError, dict(state=z(2, 4, 6, 8).transpose(2, 3))), (RuntimeError, dict(q=q[:, 0].clone().requires_grad_(True))),
                       (ValueError, dict(state=z(2, 4, 8, 7))), (TypeError, dict(active=z(2))), (ValueError, dict(active=z(3, dtype=torch.bool))),
                       (RuntimeError, dict(state=z(1, 1, 8, 6).expand(2, 4, 8, 6)))):
        with pytest.raises(error):
            step(**bad)
    f, pos = z(4, dtype=torch.float64), torch.arange(3, device=gpu_device)
    for error, args in ((ValueError, (q, pos[:2], f)), (TypeError, (q, pos.double(), f)), (TypeError, (q, pos, f.float())), (ValueError, (q, pos, z(5, dtype=torch.float64))),
                        (ValueError, ((q, z(2, 3, 1, 6)), pos, f)), (ValueError, ((q, q, q), pos, f)), (RuntimeError, (q, pos.cpu(), f)),
                        (ValueError, (q, pos.float().requires_grad_(True), f)), (ValueError, (q[0], pos, f)),
                        (ValueError, (q, pos, f.clone().requires_grad_(True)))):
        with pytest.raises(error):
            rotary_func(*args)
    for error, kw in ((ValueError, dict(p=1.0)), (ValueError, dict(p=-0.1)), (ValueError, dict(seed=-1)), (ValueError, dict(seed=1 << 64)),
                      (ValueError, dict(offset=z(2, dtype=torch.int64))), (ValueError, dict(residual=z(2, 3, 4, 7))), (TypeError, dict(residual=q.bfloat16()))):
        with pytest.raises(error):
            dropout_func(**{**dict(x=q, p=0.1, seed=1), **kw})
    assert dropout_func(q[:0], 0.1, 1).shape == (0, 3, 4, 8)
    counter = z(1, dtype=torch.int64)
    y = dropout_func(q.clone().requires_grad_(True), 0.1, 1, counter)
    counter.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()                                               # (it would be another mask)


@pytest.mark.parametrize("hip_graph", [False, True])
def test_training_driver_with_dropped_inputs(hip_graph, gpu_device):
    """The driver drops parts of the action signal, another mask every step, recorded or not: the same losses both ways."""
    from train_general_ring_no_gain import run_training
    print(f"[case] driver with input dropout, hip_graph={hip_graph}", flush=True)
    kw = dict(action_dim=2, num_neurons=64, training_steps=6, batch_size=16, seq_len=20, log_every=0, fused_loss=True, fused_optimizer=True)
    _, plain = run_training(**kw, hip_graph=hip_graph)
    _, dropped = run_training(**kw, hip_graph=hip_graph, input_dropout=0.5)
    _, again = run_training(**kw, hip_graph=not hip_graph, input_dropout=0.5)
    assert all(math.isfinite(x) for x in dropped) and dropped != plain
    assert dropped == pytest.approx(again, rel=1e-5)


def test_dropped_action_signal_keeps_its_statement(gpu_device):
    from rnn_train_ring_attractor_amd import host
    from rnn_train_ring_attractor_amd.ring_rnn_cuda import DRIVEN_ATTR
    action = host.av_to_action_signal_ND(torch.randn(8, 30, device=gpu_device), 16)
    dropped = host.drop_action_signal(action, 0.5, 3, 4)
    assert getattr(dropped, DRIVEN_ATTR) == getattr(action, DRIVEN_ATTR)
    keep = torch.from_numpy(O.keep_mask(action.numel(), 0.5, 3, 4)).view(action.shape).to(gpu_device)
    assert torch.equal(dropped, torch.where(keep, 2 * action, 0.0))
    assert host.drop_action_signal(action, 0.0, 3) is action
