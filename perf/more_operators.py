"""A recurrent layer's operators beside linear attention, as measurable cases: a short causal convolution, a selective state space scan
(each for whole sequences with their gradients, for prompts and for single tokens) and the norm, gate and scaled residual around a block.

`listed()` names pieces of real work over the range the operators are used in, `draw(rng)` gives further ones from the same
ranges, `prepare` makes what a program holds before the call, `run` is one pass, `work` what such a pass cannot do without and
`exact` the pass's outputs from the definition in 64 bits.  With `own` set, `run` calls the framework's operators; otherwise it
computes them by elementary tensor operations in 32 bits.

A case's fields:
  op      "conv"       y_t = act(bias + sum_k weight_k x_(t - K + 1 + k)), a channel by itself, with the K - 1 inputs in front
          "scan"       h_t = exp(d_t A) h_(t-1) + d_t x_t B_t, y_t = (C_t h_t + D x_t) silu(z_t), d = softplus(delta + bias)
          "norm"       y = residual + scale norm(x) weight act(gate), and the next block's norm(y) next_weight
          "conv_token", "scan_token"   one token for each sequence of a batch, the state updated in place
  B, T, C sequences, tokens, channels;  type: of what is not a state or a parameter (those are float32)
  train   forward and backward under given gradients of all outputs
  ragged  sequences of their own lengths (zero among them) in a padded batch
  start   a state to start from, and the one at the end as a result;  major "time": the tensors lie [T, B, ...] in memory, as the
          ring's history does
  K       taps;  act: activation
  N, G    a channel's states; groups of channels that share B and C;  gate: z is there
  group   how many neighbouring values a norm spans (a head's width, or all C);  kind "rms" or "layer"
  gate, residual, scale, next   whether these are there
"""
import math

import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def _conv(name, B, T, C, K, act, type, train, ragged=False, start=False, major="batch"):
    c = {"op": "conv", "B": B, "T": T, "C": C, "K": K, "act": act, "type": type, "train": train, "ragged": ragged, "start": start, "major": major}
    return dict(c, name=name) if name else c


def _scan(name, B, T, C, N, G, gate, type, train, ragged=False, start=False, major="batch"):
    c = {"op": "scan", "B": B, "T": T, "C": C, "N": N, "G": G, "gate": gate, "type": type, "train": train, "ragged": ragged,
         "start": start, "major": major}
    return dict(c, name=name) if name else c


def _token(name, op, B, C, type, **more):
    c = dict({"op": op, "B": B, "T": 1, "C": C, "type": type, "train": False}, **more)
    return dict(c, name=name) if name else c


def _norm(name, B, T, C, group, kind, gate, residual, scale, next, type, train):
    c = {"op": "norm", "B": B, "T": T, "C": C, "group": group, "kind": kind, "gate": gate, "residual": residual, "scale": scale,
         "next": next, "type": type, "train": train}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user's session, token by token: pure latency
        _token("scan_token_b1", "scan_token", 1, 1024, "bfloat16", N=16, G=1, gate=True),
        # a full batch served token by token: the states stream through memory
        _token("scan_token_b256", "scan_token", 256, 4096, "bfloat16", N=16, G=1, gate=True),
        # trials of the length and number the ring is trained on, in the ring's own type and layout
        _scan("scan_trials", 128, 120, 256, 16, 1, False, "float32", True, start=True, major="time"),
        # a padded batch of odd lengths and widths in groups, continuing from earlier states
        _scan("scan_ragged", 5, 777, 630, 11, 3, True, "float16", True, ragged=True, start=True),
        # a long prompt of one user
        _scan("scan_prompt", 1, 32768, 2048, 16, 1, True, "bfloat16", False, start=True),
        # the ordinary large training step: the largest
        _scan("scan_train", 8, 2048, 2048, 16, 1, True, "bfloat16", True),
        # the convolution's share of a served batch's token
        _token("conv_token_b64", "conv_token", 64, 2048, "bfloat16", K=4, act="silu"),
        # an odd padded batch in the ring's type
        _conv("conv_ragged", 7, 1001, 515, 3, "silu", "float32", True, ragged=True, start=True),
        # the large training step's convolution
        _conv("conv_train", 8, 4096, 4096, 4, "silu", "bfloat16", True),
        # the norm behind a served batch's token
        _norm("norm_token_b64", 64, 1, 2048, 2048, "rms", False, True, True, True, "bfloat16", False),
        # heads of linear attention normalised one by one and gated, an odd batch in the ring's type
        _norm("norm_heads", 33, 241, 480, 96, "layer", True, False, False, False, "float32", True),
        # the large training step's norms, gate and residual
        _norm("norm_train", 8, 4096, 2048, 2048, "rms", True, True, True, True, "bfloat16", True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    type = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    size = torch.empty((), dtype=_TYPES[type]).element_size()
    op = rng.choice(["scan", "scan", "scan", "scan_token", "conv", "conv", "conv_token", "norm", "norm"])
    C = rng.choice([256, 512, 1024, 2048, 4096, _log_int(rng, 24, 5000), 8 * _log_int(rng, 3, 600)])
    if op in ("scan", "scan_token"):
        G = rng.choice([1, 1, 2, 3, 4])
        C, N = max(G, C // G * G), rng.choice([16, 16, 16, 8, 32, rng.randint(1, 64)])
        gate = rng.random() < 0.7
        if op == "scan_token":
            return _token(None, op, _log_int(rng, 1, max(1, 256 * 4096 * 16 // (C * N))), C, type, N=N, G=G, gate=gate)
        train = rng.random() < 0.6
        B, T = _log_int(rng, 1, 64), _log_int(rng, 1, 32768)
        # no more than the large training step's states and rows
        while B * T * C * max(N * (3 if train else 1), 32 * size) > 8 * 2048 * 2048 * 16 * 3 or B * T * C * N > 8 * 2048 * 2048 * 32:
            B, T = max(1, B // 2), max(1, T * 2 // 3)
        return _scan(None, B, T, C, N, G, gate, type, train, rng.random() < 0.4, rng.random() < 0.5, rng.choice(["batch", "time"]))
    if op == "conv_token":
        return _token(None, op, _log_int(rng, 1, 512), C, type, K=rng.randint(2, 8), act=rng.choice(["silu", "none"]))
    B, T = _log_int(rng, 1, 64), _log_int(rng, 1, 16384)
    if op == "conv":
        while B * T * C * size > 8 * 4096 * 4096 * 2:
            B, T = max(1, B // 2), max(1, T * 2 // 3)
        return _conv(None, B, T, C, rng.choice([4, 4, 2, 3, rng.randint(1, 8)]), rng.choice(["silu", "silu", "none"]), type, rng.random() < 0.6,
                     rng.random() < 0.4, rng.random() < 0.5, rng.choice(["batch", "time"]))
    while B * T * C * size > 8 * 4096 * 2048 * 2:
        B, T = max(1, B // 2), max(1, T * 2 // 3)
    group = rng.choice([C, C, rng.choice([g for g in range(1, C + 1) if C % g == 0 and (g >= 16 or g == C)])])
    residual = rng.random() < 0.7
    return _norm(None, B, T, C, group, rng.choice(["rms", "rms", "layer"]), rng.random() < 0.5, residual, residual and rng.random() < 0.6,
                 rng.random() < 0.5, type, rng.random() < 0.6)


def _normal(gen, dtype, *shape, major="batch"):
    if major == "time":
        return torch.randn(shape[1], shape[0], *shape[2:], generator=gen, device="cuda").to(dtype).transpose(0, 1)
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def _lengths(gen, c):
    if not c["ragged"]:
        return None
    n = torch.randint(0, c["T"] + 1, (c["B"],), generator=gen, device="cuda", dtype=torch.int32)
    n[0] = c["T"]
    if c["B"] > 2:
        n[c["B"] // 2] = 0
    return n


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    c, dt = case, _TYPES[case["type"]]
    B, T, C, f32 = c["B"], c["T"], c["C"], torch.float32
    s = {"case": c}
    if c["op"] in ("conv", "conv_token"):
        K = c["K"]
        s["weight"], s["bias"] = _normal(gen, f32, C, K) * K ** -0.5, 0.1 * _normal(gen, f32, C)
        if c["op"] == "conv_token":
            # one projection's output, the gate's half beside it
            s["x"], s["state"] = _normal(gen, dt, B, 2 * C)[:, :C], _normal(gen, dt, B, K - 1, C)
            return s
        m = c["major"]
        s["x"], s["lengths"] = _normal(gen, dt, B, T, C, major=m), _lengths(gen, c)
        s["start"] = _normal(gen, dt, B, K - 1, C) if c["start"] else None
        if c["train"]:
            s["dy"], s["de"] = _normal(gen, dt, B, T, C, major=m), _normal(gen, dt, B, K - 1, C)
    elif c["op"] in ("scan", "scan_token"):
        N, G = c["N"], c["G"]
        # rates -1 ... -N, steps between 1 / 1000 and 1 / 10 of a unit: memories of a few tokens to a thousand
        s["A"] = -torch.arange(1, N + 1, device="cuda", dtype=f32).repeat(C, 1) * (1 + 0.1 * torch.rand(C, N, generator=gen, device="cuda"))
        step = torch.exp(math.log(1e-3) + math.log(1e2) * torch.rand(C, generator=gen, device="cuda"))
        s["bias"], s["D"] = step + torch.log(-torch.expm1(-step)), 1 + 0.1 * _normal(gen, f32, C)
        if c["op"] == "scan_token":
            row = _normal(gen, dt, B, 2 * G * N)
            s["Bm"], s["Cm"] = row[:, :G * N].view(B, G, N), row[:, G * N:].view(B, G, N)
            s["x"], s["delta"], s["state"] = _normal(gen, dt, B, C), _normal(gen, dt, B, C), _normal(gen, f32, B, C, N)
            s["z"] = _normal(gen, dt, B, 2 * C)[:, C:] if c["gate"] else None
            return s
        m = c["major"]
        s["x"], s["delta"], s["lengths"] = _normal(gen, dt, B, T, C, major=m), _normal(gen, dt, B, T, C, major=m), _lengths(gen, c)
        s["z"] = _normal(gen, dt, B, T, C, major=m) if c["gate"] else None
        row = _normal(gen, dt, B, T, 2 * G * N, major=m)        # one projection's output
        s["Bm"], s["Cm"] = row[..., :G * N].unflatten(2, (G, N)), row[..., G * N:].unflatten(2, (G, N))
        s["start"] = _normal(gen, f32, B, C, N) if c["start"] else None
        if c["train"]:
            s["dy"], s["de"] = _normal(gen, dt, B, T, C, major=m), _normal(gen, f32, B, C, N)
    else:
        s["x"], s["weight"] = 3 * _normal(gen, dt, B, T, C), 1 + 0.1 * _normal(gen, f32, C)
        s["gate"] = _normal(gen, dt, B, T, C) if c["gate"] else None
        s["residual"] = _normal(gen, dt, B, T, C) if c["residual"] else None
        s["scale"] = 0.2 + 0.05 * _normal(gen, f32, C) if c["scale"] else None
        s["next"] = 1 + 0.1 * _normal(gen, f32, C) if c["next"] else None
        if c["train"]:
            s["dy"] = _normal(gen, dt, B, T, C)
            s["dn"] = _normal(gen, dt, B, T, C) if c["next"] else None
    return s


# ------------------------------------------------------------------------------------------------
# The plain forms
# ------------------------------------------------------------------------------------------------
def _here(lengths, T):
    return None if lengths is None else (torch.arange(T, device=lengths.device)[None, :] < lengths[:, None])[..., None]


def _silu(x):
    return x / (1 + torch.exp(-x))


def _softplus(x):
    return x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))


def _plain_conv(x, weight, bias, start, lengths, act):
    """fp32 -> y [B,T,C], the last K - 1 inputs [B,K-1,C]"""
    B, T, C = x.shape
    K = weight.shape[1]
    front = x.new_zeros(B, K - 1, C) if start is None else start
    row = torch.cat([front, x], dim=1)
    y = bias + sum(weight[:, k] * row[:, k:k + T] for k in range(K))
    y = _silu(y) if act == "silu" else y
    here = _here(lengths, T)
    at = torch.arange(K - 1, device=x.device)[None, :] + (T if lengths is None else lengths[:, None])
    return y if here is None else torch.where(here, y, 0.0), row[torch.arange(B, device=x.device)[:, None], at]


def _plain_recurrence(a, b):
    """h_t = a_t h_(t-1) + b_t along dimension 1, from pairs of tokens: half as many, then those between."""
    n = a.shape[1]
    if n == 1:
        return b
    if n % 2:
        h = _plain_recurrence(a[:, :-1], b[:, :-1])
        return torch.cat([h, a[:, -1:] * h[:, -1:] + b[:, -1:]], dim=1)
    odd = _plain_recurrence(a[:, 1::2] * a[:, 0::2], a[:, 1::2] * b[:, 0::2] + b[:, 1::2])
    even = torch.cat([b[:, :1], a[:, 2::2] * odd[:, :-1] + b[:, 2::2]], dim=1)
    return torch.stack([even, odd], dim=2).flatten(1, 2)


def _plain_scan(x, delta, A, Bm, Cm, D, z, bias, start, lengths):
    """fp32 -> y [B,T,C], state [B,C,N]"""
    B, T, C = x.shape
    share = C // Bm.shape[2]
    d, u, here = _softplus(delta + bias), x, _here(lengths, T)
    if here is not None:
        d, u = torch.where(here, d, 0.0), torch.where(here, u, 0.0)
    a = torch.exp(d[..., None] * A)
    b = (d * u)[..., None] * Bm.repeat_interleave(share, dim=2)
    if start is not None:
        b = torch.cat([b[:, :1] + a[:, :1] * start[:, None], b[:, 1:]], dim=1)
    h = _plain_recurrence(a, b)
    y = (h * Cm.repeat_interleave(share, dim=2)).sum(3) + D * u
    y = y if z is None else y * _silu(z)
    return y if here is None else torch.where(here, y, 0.0), h[:, -1]


def _plain_normed(x, group, kind):
    rows = x.unflatten(-1, (-1, group))
    if kind == "layer":
        rows = rows - rows.mean(-1, keepdim=True)
    return (rows * torch.rsqrt((rows * rows).mean(-1, keepdim=True) + 1e-5)).flatten(-2)


def _plain_norm(x, weight, gate, residual, scale, next, c):
    y = _plain_normed(x, c["group"], c["kind"]) * weight
    y = y if gate is None else y * _silu(gate)
    y = y if scale is None else y * scale
    y = y if residual is None else residual + y
    return [y] if next is None else [y, _plain_normed(y, c["C"], c["kind"]) * next]


def _leaves(*tensors):
    return [t if t is None else t.detach().float().requires_grad_(True) for t in tensors]


def _own_leaves(*tensors):
    return [t if t is None else t.detach().requires_grad_(True) for t in tensors]


def _grads(outputs, leaves, gradients):
    return list(torch.autograd.grad(outputs, [x for x in leaves if x is not None], gradients))


def _float(t):
    return t if t is None else t.float()


def _rounded(values, like):
    return [v.to(t.dtype) for v, t in zip(values, [t for t in like if t is not None])]


def _run_plain(s):
    c, dt = s["case"], _TYPES[s["case"]["type"]]
    if c["op"] == "conv_token":
        x, K = s["x"].float(), c["K"]
        row = torch.cat([s["state"].float(), x[:, None]], dim=1)
        y = s["bias"] + (row * s["weight"].t()).sum(1)
        s["state"].copy_(row[:, 1:])
        return [(_silu(y) if c["act"] == "silu" else y).to(dt), s["state"]]
    if c["op"] == "scan_token":
        x, share = s["x"].float(), c["C"] // c["G"]
        d = _softplus(s["delta"].float() + s["bias"])
        Bm, Cm = (t.float().repeat_interleave(share, dim=1) for t in (s["Bm"], s["Cm"]))
        s["state"].mul_(torch.exp(d[..., None] * s["A"])).add_((d * x)[..., None] * Bm)
        y = (s["state"] * Cm).sum(2) + s["D"] * x
        return [(y if s["z"] is None else y * _silu(s["z"].float())).to(dt), s["state"]]
    if c["op"] == "conv":
        held = [s["x"], s["weight"], s["bias"], s["start"]]
        call = lambda x, weight, bias, start: _plain_conv(x, weight, bias, start, s["lengths"], c["act"])
        given, kinds = ("dy", "de") if c["start"] else ("dy",), [dt, dt]
    elif c["op"] == "scan":
        held = [s[n] for n in ("x", "delta", "A", "Bm", "Cm", "D", "z", "bias", "start")]
        call = lambda *leaves: _plain_scan(*leaves, s["lengths"])
        given, kinds = ("dy", "de") if c["start"] else ("dy",), [dt, torch.float32]
    else:
        held = [s[n] for n in ("x", "weight", "gate", "residual", "scale", "next")]
        call = lambda *leaves: _plain_norm(*leaves, c)
        given, kinds = ("dy", "dn") if c["next"] else ("dy",), [dt, dt]
    if not c["train"]:
        with torch.no_grad():
            return [y.to(k) for y, k in zip(call(*(_float(t) for t in held))[:len(given) if c["op"] == "norm" else 1 + c["start"]], kinds)]
    leaves = _leaves(*held)
    out = list(call(*leaves))[:len(given)]
    grads = _grads(out, leaves, [s[n].float() for n in given])
    return [y.detach().to(k) for y, k in zip(out, kinds)] + _rounded(grads, held)


# ------------------------------------------------------------------------------------------------
# The framework's operators
# ------------------------------------------------------------------------------------------------
def _run_own(s):
    from rnn_train_ring_attractor_amd import causal_conv_func, causal_conv_step, norm_gate_func, selective_scan_func, selective_scan_step
    c = s["case"]
    act = None if c.get("act") == "none" else c.get("act")
    if c["op"] == "conv_token":
        with torch.no_grad():
            return [causal_conv_step(s["x"], s["weight"], s["state"], bias=s["bias"], activation=act), s["state"]]
    if c["op"] == "scan_token":
        with torch.no_grad():
            y = selective_scan_step(s["x"], s["delta"], s["A"], s["Bm"], s["Cm"], s["state"], D=s["D"], z=s["z"], delta_bias=s["bias"],
                                    softplus=True)
        return [y, s["state"]]
    listing = lambda y: list(y) if isinstance(y, tuple) else [y]
    if c["op"] == "conv":
        held = [s["x"], s["weight"], s["bias"], s["start"]]
        call = lambda x, weight, bias, start: causal_conv_func(x, weight, bias, initial_state=start, lengths=s["lengths"], activation=act,
                                                               return_state=c["start"])
        given = ("dy", "de") if c["start"] else ("dy",)
    elif c["op"] == "scan":
        held = [s[n] for n in ("x", "delta", "A", "Bm", "Cm", "D", "z", "bias", "start")]
        call = lambda x, delta, A, Bm, Cm, D, z, bias, start: selective_scan_func(
            x, delta, A, Bm, Cm, D=D, z=z, delta_bias=bias, initial_state=start, lengths=s["lengths"], softplus=True, return_state=c["start"])
        given = ("dy", "de") if c["start"] else ("dy",)
    else:
        held = [s[n] for n in ("x", "weight", "gate", "residual", "scale", "next")]
        call = lambda x, weight, gate, residual, scale, next: norm_gate_func(
            x, weight, gate=gate, residual=residual, scale=scale, next_weight=next, group=c["group"], kind=c["kind"])
        given = ("dy", "dn") if c["next"] else ("dy",)
    if not c["train"]:
        with torch.no_grad():
            return listing(call(*held))
    leaves = _own_leaves(*held)
    out = listing(call(*leaves))
    return [y.detach() for y in out] + _grads(out, leaves, [s[n] for n in given])


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    c = case
    size = torch.empty((), dtype=_TYPES[c["type"]]).element_size()
    B, C = c["B"], c["C"]
    rows = B * c["T"]
    if c.get("ragged"):
        rows = rows // 2 + c["T"] // 2
    if c["op"] == "conv_token":
        return {"bytes": B * C * size * 2 * c["K"] + C * (c["K"] + 1) * 4, "flops": 2 * B * C * c["K"]}
    if c["op"] == "scan_token":
        n = B * C * c["N"]
        return {"bytes": 8 * n + 4 * C * (c["N"] + 2) + B * size * (C * (4 if c["gate"] else 3) + 2 * c["G"] * c["N"]), "flops": 7 * n}
    if c["op"] == "conv":
        states = B * (c["K"] - 1) * C * size * (2 if c["start"] else 0)
        if not c["train"]:
            return {"bytes": 2 * rows * C * size + states, "flops": 2 * rows * C * c["K"]}
        # x, dy read and y, dx written; backwards the sums again, their transpose and the weights' gradient
        return {"bytes": 4 * rows * C * size + 2 * states, "flops": 8 * rows * C * c["K"]}
    if c["op"] == "scan":
        n, once = rows * C * c["N"], rows * size * (C * (3 if c["gate"] else 2) + 2 * c["G"] * c["N"])
        states = B * C * c["N"] * 4 * (2 if c["start"] else 0)
        # a power, the products with it, with B and with C
        if not c["train"]:
            return {"bytes": once + rows * C * size + states, "flops": 7 * n}
        # dy read and the gradients written besides; the states again, theirs, and four sums of products
        return {"bytes": 2 * (once + rows * C * size) + 2 * states, "flops": 7 * n + 17 * n}
    tensors = 2 + c["gate"] + c["residual"] + c["next"]
    # backwards: the gradients of the outputs, x and the gate read (y again, for the next norm), the inputs' gradients written
    back = 1 + c["next"] + 1 + c["gate"] + c["next"] + 1 + c["gate"] + c["residual"]
    n = rows * C
    return {"bytes": n * size * (tensors + (back if c["train"] else 0)), "flops": n * (12 + (24 if c["train"] else 0))}


# ------------------------------------------------------------------------------------------------
# From the definitions, in 64 bits
# ------------------------------------------------------------------------------------------------
def _count(s, c):
    return [c["T"]] * c["B"] if s["lengths"] is None else s["lengths"].tolist()


def _gate64(z):
    """(silu, its derivative)"""
    p = 1 / (1 + torch.exp(-z))
    return z * p, p * (1 + z * (1 - p))


def _exact_conv(s, c):
    B, T, C, K = c["B"], c["T"], c["C"], c["K"]
    z = dict(dtype=torch.float64, device="cuda")
    w, bias = s["weight"].double(), s["bias"].double()
    y, end, dx = torch.zeros(B, T, C, **z), torch.zeros(B, K - 1, C, **z), torch.zeros(B, T, C, **z)
    dw, db, d0 = torch.zeros(C, K, **z), torch.zeros(C, **z), torch.zeros(B, K - 1, C, **z)
    for b, n in enumerate(_count(s, c)):
        front = torch.zeros(K - 1, C, **z) if s["start"] is None else s["start"][b].double()
        row = torch.cat([front, s["x"][b, :n].double()])
        end[b] = row[n:]
        if n == 0:
            if c["start"] and c["train"]:
                d0[b] = s["de"][b].double()
            continue
        taps = row.unfold(0, K, 1)                                    # [n,C,K]
        p = bias + torch.einsum("tck,ck->tc", taps, w)
        value, slope = _gate64(p) if c["act"] == "silu" else (p, torch.ones_like(p))
        y[b, :n] = value
        if c["train"]:
            g = s["dy"][b, :n].double() * slope
            dw += torch.einsum("tc,tck->ck", g, taps)
            db += g.sum(0)
            drow = torch.zeros(n + K - 1, C, **z)
            for k in range(K):
                drow[k:k + n] += g * w[:, k]
            if c["start"]:
                drow[n:] += s["de"][b].double()
                d0[b] = drow[:K - 1]
            dx[b, :n] = drow[K - 1:]
    out = [y, end] if c["start"] else [y]
    if c["train"]:
        out += [dx, dw, db] + ([d0] if c["start"] else [])
    return out


def _exact_scan(s, c):
    B, T, C, N, G = (c[x] for x in ("B", "T", "C", "N", "G"))
    z64 = dict(dtype=torch.float64, device="cuda")
    of = torch.arange(C, device="cuda") // (C // G)                   # a channel's group
    here = torch.tensor(_count(s, c), device="cuda")[:, None] > torch.arange(T, device="cuda")
    A, D = s["A"].double(), s["D"].double()
    raw = s["delta"].double() + s["bias"].double()
    d = torch.nn.functional.softplus(raw, threshold=100.0) * here[..., None]
    x = s["x"].double() * here[..., None]
    gate, slope = (None, None) if s["z"] is None else _gate64(s["z"].double())
    h = torch.zeros(B, C, N, **z64) if s["start"] is None else s["start"].double()
    hs = torch.empty(T + 1, B, C, N, **z64) if c["train"] else None
    inner = torch.empty(B, T, C, **z64)
    Bs, Cs = s["Bm"].double(), s["Cm"].double()
    for t in range(T):
        if c["train"]:
            hs[t] = h
        h = torch.exp(d[:, t, :, None] * A) * h
        h += (d[:, t] * x[:, t])[..., None] * Bs[:, t, of]
        torch.matmul(h[:, :, None], Cs[:, t, of][..., None], out=inner[:, t].view(B, C, 1, 1))
    inner += D * x
    y = (inner if gate is None else inner * gate) * here[..., None]
    out = [y, h] if c["start"] else [y]
    if not c["train"]:
        return out
    hs[T] = h
    dy = s["dy"].double() * here[..., None]
    dz = None if gate is None else dy * inner * slope
    q = dy if gate is None else dy * gate                             # the gradient in front of the gate
    g = s["de"].double() if c["start"] else torch.zeros(B, C, N, **z64)
    dA, dd, dx = torch.zeros(C, N, **z64), torch.empty(B, T, C, **z64), torch.empty(B, T, C, **z64)
    dB, dC = torch.empty(B, T, G, N, **z64), torch.empty(B, T, G, N, **z64)
    for t in reversed(range(T)):
        g = g + q[:, t, :, None] * Cs[:, t, of]
        dC[:, t] = (q[:, t, :, None] * hs[t + 1]).view(B, G, C // G, N).sum(2) * here[:, t, None, None]
        dB[:, t] = ((d[:, t] * x[:, t])[..., None] * g).view(B, G, C // G, N).sum(2)
        into = (g * Bs[:, t, of]).sum(2)
        back = torch.exp(d[:, t, :, None] * A) * g
        turn = back * hs[t]
        dA += (d[:, t, :, None] * turn).sum(0)
        dd[:, t] = (turn * A).sum(2) + into * x[:, t]
        dx[:, t] = into * d[:, t]
        g = back
    dx = (dx + D * q) * here[..., None]
    ddelta = dd / (1 + torch.exp(-raw)) * here[..., None]
    out += [dx, ddelta, dA, dB, dC, (q * x).sum((0, 1))]
    return out + ([] if dz is None else [dz]) + [ddelta.sum((0, 1))] + ([g] if c["start"] else [])


def _exact_normed(x, group, kind, weight, dn=None):
    """(normed x weight, and for a gradient dn of it dx and the weight's)"""
    rows = x.view(-1, x.shape[-1] // group, group)
    if kind == "layer":
        rows = rows - rows.mean(2, keepdim=True)
    r = (rows.square().mean(2, keepdim=True) + 1e-5) ** -0.5
    unit = rows * r
    out = (unit.view(x.shape) * weight)
    if dn is None:
        return out, None, None
    g = (dn * weight).view_as(rows)
    dx = r * (g - unit * (g * unit).mean(2, keepdim=True))
    if kind == "layer":
        dx = dx - dx.mean(2, keepdim=True)
    return out, dx.view_as(x), (dn * unit.view(x.shape)).sum((0, 1))


def _exact_norm(s, c):
    x, w = s["x"].double(), s["weight"].double()
    normed, _, _ = _exact_normed(x, c["group"], c["kind"], w)
    gate, slope = (1.0, None) if s["gate"] is None else _gate64(s["gate"].double())
    scale = 1.0 if s["scale"] is None else s["scale"].double()
    branch = normed * gate
    y = scale * branch if s["residual"] is None else s["residual"].double() + scale * branch
    out, total = [y], None
    if c["train"]:
        total = s["dy"].double()
    dnext = None
    if c["next"]:
        n, more, dnext = _exact_normed(y, c["C"], c["kind"], s["next"].double(), s["dn"].double() if c["train"] else None)
        out.append(n)
        total = total + more if c["train"] else None
    if not c["train"]:
        return out
    _, dx, dw = _exact_normed(x, c["group"], c["kind"], w, total * scale * gate)
    out += [dx, dw]
    if c["gate"]:
        out.append(total * scale * normed * slope)
    if c["residual"]:
        out.append(total)
    if c["scale"]:
        out.append((total * branch).sum((0, 1)))
    return out + ([dnext] if c["next"] else [])


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "conv":
        return _exact_conv(s, c)
    if c["op"] == "scan":
        return _exact_scan(s, c)
    if c["op"] == "norm":
        return _exact_norm(s, c)
    if c["op"] == "conv_token":
        row = torch.cat([s["state"].double(), s["x"].double()[:, None]], dim=1)
        y = s["bias"].double() + torch.einsum("bkc,ck->bc", row, s["weight"].double())
        return [_gate64(y)[0] if c["act"] == "silu" else y, row[:, 1:]]
    of = torch.arange(c["C"], device="cuda") // (c["C"] // c["G"])
    x, d = s["x"].double(), torch.nn.functional.softplus(s["delta"].double() + s["bias"].double(), threshold=100.0)
    h = torch.exp(d[..., None] * s["A"].double()) * s["state"].double() + (d * x)[..., None] * s["Bm"].double()[:, of]
    y = torch.einsum("bcn,bcn->bc", h, s["Cm"].double()[:, of]) + s["D"].double() * x
    return [y if s["z"] is None else y * _gate64(s["z"].double())[0], h]
