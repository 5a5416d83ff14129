"""The sequence operators beside the ring's time loop, as measurable cases: linear attention with a decay for each head
(whole sequences with their gradients, prompts, single tokens), rotary positions and dropout.

`listed()` names pieces of real work over the range the operators are used in, `draw(rng)` gives further ones from the same
ranges, `prepare` makes what a program holds before the call, `run` is one pass, `work` what such a pass cannot do without and
`exact` the pass's outputs from the definition in 64 bits.  With `own` set, `run` calls the framework's operators; otherwise it
computes them by elementary tensor operations in 32 bits.

A case's fields:
  op      "attention"  a whole sequence: o_t = scale q_t S_t, S_t = e^g S_{t-1} + k_t v_t^T, the state at the end beside it;
                       train: forward and backward under given gradients of both
          "token"      one token for each sequence of a batch, the state updated in place
          "rotary"     queries and keys turned by their positions; train: forward and backward
          "dropout"    residual + dropout(x); train: forward and backward
  B, T    sequences, tokens;  H, G: heads of q, of k and v;  Dk, Dv: their widths;  type: of what is not a state
  ragged  sequences of their own lengths (zero among them) in a padded batch
  start   a state to start from;  major "time": the tensors lie [T, B, ...] in memory, as the ring's history does
  rot     how many of a head's Dk values are turned;  layout, position: see the operator;  far: the largest position
  p       probability of dropping;  shape [B, T, H * Dk]
"""
import math

import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def _attention(name, B, T, H, G, Dk, Dv, type, train, ragged=False, start=False, major="batch"):
    c = {"op": "attention", "B": B, "T": T, "H": H, "G": G, "Dk": Dk, "Dv": Dv, "type": type, "train": train, "ragged": ragged,
         "start": start, "major": major}
    return dict(c, name=name) if name else c


def _token(name, B, H, G, Dk, Dv, type):
    c = {"op": "token", "B": B, "T": 1, "H": H, "G": G, "Dk": Dk, "Dv": Dv, "type": type}
    return dict(c, name=name) if name else c


def _rotary(name, B, T, H, G, Dk, rot, type, layout, position, far, train):
    c = {"op": "rotary", "B": B, "T": T, "H": H, "G": G, "Dk": Dk, "rot": rot, "type": type, "layout": layout,
         "position": position, "far": far, "train": train}
    return dict(c, name=name) if name else c


def _dropout(name, B, T, H, Dk, p, type, residual, train):
    c = {"op": "dropout", "B": B, "T": T, "H": H, "Dk": Dk, "p": p, "type": type, "residual": residual, "train": train}
    return dict(c, name=name) if name else c


def listed():
    return [
        # a session of one user, token by token: pure latency
        _token("token_b1", 1, 8, 8, 64, 64, "bfloat16"),
        # a full batch served token by token: the states stream through memory
        _token("token_b256", 256, 16, 4, 128, 128, "bfloat16"),
        # trials of the length the ring is trained on, a small batch, in the ring's own type and layout
        _attention("train_trials", 32, 120, 4, 4, 64, 64, "float32", True, start=True, major="time"),
        # a padded batch of odd lengths and widths with shared key heads, continuing from earlier states
        _attention("train_ragged", 6, 777, 6, 2, 80, 112, "bfloat16", True, ragged=True, start=True),
        # a long prompt of one user
        _attention("prompt_long", 1, 32768, 16, 16, 128, 128, "bfloat16", False),
        # a batch of medium prompts on wide heads in the ring's type
        _attention("prompt_wide", 8, 2000, 8, 8, 256, 256, "float32", False, start=True),
        # the ordinary large training step: the largest
        _attention("train_large", 8, 4096, 16, 16, 128, 128, "bfloat16", True),
        # positions of one token for each of a served batch, far into their contexts
        _rotary("rotary_token", 64, 1, 16, 4, 128, 128, "bfloat16", "half", "each", 1 << 20, False),
        # heads turned by an integrated heading (an angle, not a count) on an odd batch
        _rotary("rotary_heading", 33, 241, 5, 5, 96, 48, "float32", "interleaved", "angle", 7, True),
        # the large training step's queries and keys, half of each head turned
        _rotary("rotary_train", 8, 4096, 16, 4, 128, 64, "bfloat16", "half", "shared", 4096, True),
        # sensory dropout of the training script's action signal
        _dropout("dropout_signal", 128, 100, 1, 16, 0.2, "float32", False, True),
        # the large training step's residual branch
        _dropout("dropout_train", 8, 4096, 16, 128, 0.1, "bfloat16", True, True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    type = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    size = torch.empty((), dtype=_TYPES[type]).element_size()
    G = rng.choice([1, 2, 3, 4, 8])
    H = G * rng.choice([1, 1, 2, 4] if G <= 4 else [1, 1, 2])
    op = rng.choice(["attention", "attention", "attention", "token", "rotary", "rotary", "dropout"])
    Dk = rng.choice([64, 128, 256, rng.randint(8, 256), 8 * rng.randint(2, 32)])
    if op == "attention":
        Dv = rng.choice([64, 128, 256, rng.randint(8, 256), 8 * rng.randint(2, 32)])
        B, T = _log_int(rng, 1, 32), _log_int(rng, 1, 32768)
        # no more than the large training step's elements and products
        while B * T * H * max((Dk + Dv) * 32 * size, Dk * Dv) > 8 * 4096 * 16 * 128 * 128 or B * H * Dk * Dv > 32 * 16 * 128 * 128:
            B, T = max(1, B // 2), max(1, T * 2 // 3)
        return _attention(None, B, T, H, G, Dk, Dv, type, rng.random() < 0.6, rng.random() < 0.4, rng.random() < 0.5,
                          rng.choice(["batch", "time"]))
    if op == "token":
        Dv = rng.choice([64, 128, 256, rng.randint(8, 256)])
        return _token(None, _log_int(rng, 1, max(1, 256 * 16 * 128 * 128 // (H * Dk * Dv))), H, G, Dk, Dv, type)
    B, T = _log_int(rng, 1, 64), _log_int(rng, 1, 8192)
    while B * T * (H + G) * Dk * size > 8 * 4096 * 20 * 128 * 2:
        B, T = max(1, B // 2), max(1, T * 2 // 3)
    if op == "rotary":
        return _rotary(None, B, T, H, G, Dk, 2 * rng.randint(1, Dk // 2) if rng.random() < 0.5 else Dk - Dk % 2, type,
                       rng.choice(["half", "interleaved"]), rng.choice(["each", "shared", "angle"]), _log_int(rng, 8, 1 << 22),
                       rng.random() < 0.6)
    return _dropout(None, B, T, H, Dk, round(rng.uniform(0.02, 0.6), 3), type, rng.random() < 0.5, rng.random() < 0.7)


def _normal(gen, dtype, *shape, major="batch"):
    if major == "time":
        return torch.randn(shape[1], shape[0], *shape[2:], generator=gen, device="cuda").to(dtype).transpose(0, 1)
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def _log_decay(H):
    """From a memory of eight tokens to one of 1024, over the heads."""
    return torch.log1p(-torch.exp2(-torch.linspace(3.0, 10.0, H, dtype=torch.float64))).to(torch.float32).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    c, dt = case, _TYPES[case["type"]]
    B, T, H, Dk = c["B"], c["T"], c["H"], c["Dk"]
    s = {"case": c}
    if c["op"] == "attention":
        G, Dv, m = c["G"], c["Dv"], c["major"]
        s["q"], s["k"] = _normal(gen, dt, B, T, H, Dk, major=m), _normal(gen, dt, B, T, G, Dk, major=m)
        s["v"], s["g"] = _normal(gen, dt, B, T, G, Dv, major=m), _log_decay(H)
        s["start"] = _normal(gen, torch.float32, B, H, Dk, Dv) if c["start"] else None
        s["lengths"] = None
        if c["ragged"]:
            n = torch.randint(0, T + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
            n[0] = T
            if B > 2:
                n[B // 2] = 0
            s["lengths"] = n
        if c["train"]:
            s["do"], s["ds"] = _normal(gen, dt, B, T, H, Dv, major=m), _normal(gen, torch.float32, B, H, Dk, Dv)
    elif c["op"] == "token":
        G, Dv = c["G"], c["Dv"]
        # one projection's output, the heads of q, k and v side by side
        row = _normal(gen, dt, B, H * Dk + G * (Dk + Dv))
        s["q"] = row[:, :H * Dk].view(B, H, Dk)
        s["k"] = row[:, H * Dk:(H + G) * Dk].view(B, G, Dk)
        s["v"] = row[:, (H + G) * Dk:].view(B, G, Dv)
        s["g"], s["state"] = _log_decay(H), _normal(gen, torch.float32, B, H, Dk, Dv)
    elif c["op"] == "rotary":
        G, rot = c["G"], c["rot"]
        s["q"], s["k"] = _normal(gen, dt, B, T, H, Dk), _normal(gen, dt, B, T, G, Dk)
        if c["position"] == "angle":        # a heading that drifts; the head's pairs turn with its harmonics
            step = 0.3 * torch.randn(B, T, generator=gen, device="cuda", dtype=torch.float64)
            s["positions"] = (c["far"] * torch.rand(B, 1, generator=gen, device="cuda", dtype=torch.float64) + step.cumsum(1)).float()
            s["frequencies"] = torch.arange(1, rot // 2 + 1, dtype=torch.float64, device="cuda")
        else:
            if c["position"] == "each":
                s["positions"] = torch.randint(0, c["far"], (B, T), generator=gen, device="cuda")
            else:
                first = int(torch.randint(0, c["far"], (1,), generator=gen, device="cuda"))
                s["positions"] = torch.arange(first, first + T, device="cuda")
            s["frequencies"] = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64, device="cuda") * 2 / rot)
        s["scale"] = 1.0
        if c["train"]:
            s["do"] = [_normal(gen, dt, B, T, H, Dk), _normal(gen, dt, B, T, G, Dk)]
    else:
        s["x"] = _normal(gen, dt, B, T, H * Dk)
        s["residual"] = _normal(gen, dt, B, T, H * Dk) if c["residual"] else None
        s["seed"], s["offset"] = 0x9D3C5A1700000000 + seed, (seed << 33) + 12345
        if c["train"]:
            s["do"] = _normal(gen, dt, B, T, H * Dk)
    return s


# ------------------------------------------------------------------------------------------------
# The plain forms
# ------------------------------------------------------------------------------------------------
_CHUNK = 64


def _plain_attention(q, k, v, g, start, lengths):
    """fp32 [B,T,.,.] -> o [B,T,H,Dv], state [B,H,Dk,Dv]: within chunks as masked products, across them by the recurrence."""
    B, T, H, Dk = q.shape
    Dv, C = v.shape[3], _CHUNK
    k, v = (x.repeat_interleave(H // x.shape[2], dim=2) for x in (k, v))
    n = -(-T // C)
    if lengths is None:
        lengths = torch.full((B,), T, dtype=torch.int32, device=q.device)
    here = torch.arange(T, device=q.device)[None, :] < lengths[:, None]
    q, k, v = (torch.where(here[:, :, None, None], x, torch.zeros((), device=x.device)) for x in (q, k, v))
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, 0, 0, n * C - T)).view(B, n, C, H, -1).permute(0, 3, 1, 2, 4) for x in (q, k, v))
    i = torch.arange(C, device=q.device)
    apart = i[:, None] - i[None, :]
    weight = torch.where(apart >= 0, torch.exp(g[:, None, None] * apart.clamp(min=0)), 0.0)
    o = torch.matmul(torch.matmul(q, k.transpose(-1, -2)) * weight[None, :, None], v)
    full = (lengths[:, None] - torch.arange(n, device=q.device)[None] * C).clamp(0, C)            # [B,n] tokens of each chunk
    left = (full[:, None, :, None] - 1 - i).clamp(min=0)
    local = torch.matmul((k * torch.exp(g[None, :, None, None] * left)[..., None]).transpose(-1, -2), v)
    carry = torch.exp(g[None, :, None] * full[:, None])[..., None, None]
    state = torch.zeros(B, H, Dk, Dv, device=q.device) if start is None else start
    states = []
    for c in range(n):
        states.append(state)
        state = carry[:, :, c] * state + local[:, :, c]
    inner = q * torch.exp(g[:, None] * (i + 1))[None, :, None, :, None]
    o = Dk ** -0.5 * (o + torch.matmul(inner, torch.stack(states, dim=2)))
    return o.permute(0, 2, 3, 1, 4).reshape(B, n * C, H, Dv)[:, :T], state


def _plain_rotary(x, positions, frequencies, layout, scale):
    a = positions.to(torch.float64)[..., None] * frequencies
    a = a if a.dim() == 3 else a[None]
    cos, sin = (scale * torch.cos(a)).float()[:, :, None], (scale * torch.sin(a)).float()[:, :, None]
    r = frequencies.numel()
    if layout == "half":
        a, b, rest = x[..., :r], x[..., r:2 * r], x[..., 2 * r:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], dim=-1)
    a, b, rest = x[..., 0:2 * r:2], x[..., 1:2 * r:2], x[..., 2 * r:]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2), rest], dim=-1)


def _plain_keep(n, p, seed, offset, device):
    """Philox with four words and seven rounds (Salmon et al. 2011): word i % 4 of block i / 4, kept from p 2^32 up."""
    low = 0xFFFFFFFF
    block = torch.arange(-(-n // 4), device=device)
    x = [block & low, block >> 32, torch.full_like(block, offset & low), torch.full_like(block, offset >> 32)]
    k0, k1 = seed & low, seed >> 32
    for _ in range(7):
        a, b = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
        x = [((b >> 32) & low) ^ x[1] ^ k0, b & low, ((a >> 32) & low) ^ x[3] ^ k1, a & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return (torch.stack(x, dim=1).view(-1)[:n] >= int(p * 2.0 ** 32))


def _leaves(*tensors):
    return [t if t is None else t.detach().float().requires_grad_(True) for t in tensors]


def _own_leaves(*tensors):
    return [t if t is None else t.detach().requires_grad_(True) for t in tensors]


def _grads(outputs, leaves, gradients):
    leaves = [x for x in leaves if x is not None]
    return list(torch.autograd.grad(outputs, leaves, gradients))


def _run_plain(s):
    c, dt = s["case"], _TYPES[s["case"]["type"]]
    if c["op"] == "attention":
        if not c["train"]:
            with torch.no_grad():
                o, state = _plain_attention(s["q"].float(), s["k"].float(), s["v"].float(), s["g"], s["start"], s["lengths"])
            return [o.to(dt), state]
        q, k, v, start = _leaves(s["q"], s["k"], s["v"], s["start"])
        o, state = _plain_attention(q, k, v, s["g"], start, s["lengths"])
        grads = _grads([o, state], [q, k, v, start], [s["do"].float(), s["ds"]])
        return [o.detach().to(dt), state.detach()] + [x.to(dt) for x in grads[:3]] + grads[3:]
    if c["op"] == "token":
        rep = c["H"] // c["G"]
        q, k, v = s["q"].float(), s["k"].float().repeat_interleave(rep, 1), s["v"].float().repeat_interleave(rep, 1)
        s["state"].mul_(torch.exp(s["g"])[None, :, None, None]).add_(k[..., None] * v[:, :, None, :])
        return [(c["Dk"] ** -0.5 * (q[..., None] * s["state"]).sum(2)).to(dt), s["state"]]
    if c["op"] == "rotary":
        turn = lambda x: _plain_rotary(x, s["positions"], s["frequencies"], c["layout"], s["scale"])
        if not c["train"]:
            return [turn(s["q"].float()).to(dt), turn(s["k"].float()).to(dt)]
        q, k = _leaves(s["q"], s["k"])
        out = [turn(q), turn(k)]
        grads = _grads(out, [q, k], [x.float() for x in s["do"]])
        return [x.detach().to(dt) for x in out] + [x.to(dt) for x in grads]
    keep = _plain_keep(s["x"].numel(), c["p"], s["seed"], s["offset"], s["x"].device).view(s["x"].shape)
    drop = lambda x: torch.where(keep, x.float() * (1.0 / (1.0 - c["p"])), 0.0)
    y = drop(s["x"])
    out = [(y if s["residual"] is None else s["residual"].float() + y).to(dt)]
    if c["train"]:
        out.append(drop(s["do"]).to(dt))
        if s["residual"] is not None:
            out.append(s["do"])
    return out


# ------------------------------------------------------------------------------------------------
# The framework's operators
# ------------------------------------------------------------------------------------------------
def _run_own(s):
    from rnn_train_ring_attractor_amd import dropout_func, linear_attention_func, linear_attention_step, rotary_func
    c = s["case"]
    if c["op"] == "attention":
        call = lambda q, k, v, start: linear_attention_func(q, k, v, s["g"], initial_state=start, lengths=s["lengths"],
                                                            return_state=True)
        if not c["train"]:
            with torch.no_grad():
                return list(call(s["q"], s["k"], s["v"], s["start"]))
        leaves = _own_leaves(s["q"], s["k"], s["v"], s["start"])
        out = call(*leaves)
        return [x.detach() for x in out] + _grads(out, leaves, [s["do"], s["ds"]])
    if c["op"] == "token":
        return [linear_attention_step(s["q"], s["k"], s["v"], s["g"], s["state"]), s["state"]]
    if c["op"] == "rotary":
        turn = lambda q, k: rotary_func((q, k), s["positions"], s["frequencies"], layout=c["layout"], scale=s["scale"])
        if not c["train"]:
            with torch.no_grad():
                return list(turn(s["q"], s["k"]))
        leaves = _own_leaves(s["q"], s["k"])
        out = turn(*leaves)
        return [x.detach() for x in out] + _grads(out, leaves, s["do"])
    if not c["train"]:
        with torch.no_grad():
            return [dropout_func(s["x"], c["p"], s["seed"], s["offset"], residual=s["residual"])]
    leaves = _own_leaves(s["x"], s["residual"])
    y = dropout_func(leaves[0], c["p"], s["seed"], s["offset"], residual=leaves[1])
    return [y.detach()] + _grads([y], leaves, [s["do"]])


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    c = case
    size = torch.empty((), dtype=_TYPES[c["type"]]).element_size()
    rows, H, Dk = c["B"] * c["T"], c["H"], c["Dk"]
    if c["op"] in ("attention", "token"):
        G, Dv = c["G"], c["Dv"]
        if c["op"] == "attention" and c["ragged"]:
            rows = rows // 2 + c["T"] // 2
        once = rows * (H * (Dk + Dv) + G * (Dk + Dv)) * size
        states = c["B"] * H * Dk * Dv * 4
        if c["op"] == "token":
            return {"bytes": once + 2 * states, "flops": 5 * rows * H * Dk * Dv}
        if not c["train"]:
            return {"bytes": once + states * (2 if c["start"] else 1), "flops": 4 * rows * H * Dk * Dv}
        # q, k, v, do read and o, dq, dk, dv written; the states' part likewise
        return {"bytes": 2 * once + states * (4 if c["start"] else 2), "flops": 12 * rows * H * Dk * Dv}
    passes = 2 if c["train"] else 1
    if c["op"] == "rotary":
        return {"bytes": passes * 2 * rows * (H + c["G"]) * Dk * size, "flops": passes * 3 * rows * (H + c["G"]) * c["rot"]}
    n = rows * H * Dk
    return {"bytes": n * size * (2 * passes + (1 if c["residual"] else 0)), "flops": passes * n}


# ------------------------------------------------------------------------------------------------
# From the definitions, in 64 bits
# ------------------------------------------------------------------------------------------------
def _exact_attention(s, c):
    B, T, H, G, Dk, Dv = (c[x] for x in ("B", "T", "H", "G", "Dk", "Dv"))
    z = dict(dtype=torch.float64, device="cuda")
    o, state = torch.zeros(B, T, H, Dv, **z), torch.zeros(B, H, Dk, Dv, **z)
    dq, dk, dv = torch.zeros(B, T, H, Dk, **z), torch.zeros(B, T, G, Dk, **z), torch.zeros(B, T, G, Dv, **z)
    d0 = torch.zeros(B, H, Dk, Dv, **z)
    scale, rows = 1.0 / math.sqrt(Dk), 2048
    lengths = [T] * B if s["lengths"] is None else s["lengths"].tolist()
    for b in range(B):
        n = lengths[b]
        at = torch.arange(n, **z)
        for h in range(H):
            e = h // (H // G)
            lam = math.exp(float(s["g"][h].double()))
            q, k, v = s["q"][b, :n, h].double(), s["k"][b, :n, e].double(), s["v"][b, :n, e].double()
            s0 = torch.zeros(Dk, Dv, **z) if s["start"] is None else s["start"][b, h].double()
            since, until = lam ** (at + 1), lam ** (n - 1 - at)
            state[b, h] = lam ** n * s0 + (k * until[:, None]).t() @ v
            if c["train"]:
                do, ds = s["do"][b, :n, h].double(), s["ds"][b, h].double()
                d0[b, h] = lam ** n * ds + scale * (q * since[:, None]).t() @ do
                dq[b, :n, h] = scale * since[:, None] * (do @ s0.t())
                dk[b, :n, e] += until[:, None] * (v @ ds.t())
                dv[b, :n, e] += until[:, None] * (k @ ds)
            o[b, :n, h] = scale * since[:, None] * (q @ s0)
            for i in range(0, n, rows):
                m = min(n, i + rows)
                w = torch.tril(lam ** (at[i:m, None] - at[None, :m]).clamp(min=0), diagonal=i) * scale
                p = w * (q[i:m] @ k[:m].t())
                o[b, i:m, h] += p @ v[:m]
                if c["train"]:
                    r = w * (do[i:m] @ v[:m].t())
                    dq[b, i:m, h] += r @ k[:m]
                    dk[b, :m, e] += r.t() @ q[i:m]
                    dv[b, :m, e] += p.t() @ do[i:m]
    out = [o, state]
    if c["train"]:
        out += [dq, dk, dv] + ([d0] if c["start"] else [])
    return out


def _exact_rotary(x, s, c, back):
    pos = s["positions"].double().reshape(-1, c["T"])
    out = x.double().clone()
    r = c["rot"] // 2
    for m in range(r):
        i, j = (m, m + r) if c["layout"] == "half" else (2 * m, 2 * m + 1)
        turns = pos * (s["frequencies"][m] / (2 * math.pi))
        angle = (2 * math.pi * (turns - torch.floor(turns)))[:, :, None]
        cos, sin = torch.cos(angle) * s["scale"], torch.sin(angle) * (-s["scale"] if back else s["scale"])
        a, b = x[..., i].double(), x[..., j].double()
        out[..., i], out[..., j] = cos * a - sin * b, sin * a + cos * b
    return out


def _exact_keep(n, p, seed, offset):
    import numpy as np
    u = np.uint64
    low, blocks = u(0xFFFFFFFF), np.arange((n + 3) // 4, dtype=np.uint64)
    c0, c1 = blocks & low, blocks >> u(32)
    c2, c3 = np.full_like(blocks, offset % 2 ** 32), np.full_like(blocks, offset // 2 ** 32)
    for r in range(7):
        key0, key1 = u((seed % 2 ** 32 + r * 0x9E3779B9) % 2 ** 32), u((seed // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32)
        first, second = c0 * u(0xD2511F53), c2 * u(0xCD9E8D57)
        c0, c1, c2, c3 = (second >> u(32)) ^ c1 ^ key0, second & low, (first >> u(32)) ^ c3 ^ key1, first & low
    words = np.empty((blocks.size, 4), dtype=np.uint64)
    words[:, 0], words[:, 1], words[:, 2], words[:, 3] = c0, c1, c2, c3
    return words.reshape(-1)[:n] >= u(int(p * 2.0 ** 32))


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "attention":
        return _exact_attention(s, c)
    if c["op"] == "token":
        per = c["H"] // c["G"]
        state, o = s["state"].double(), torch.empty(c["B"], c["H"], c["Dv"], dtype=torch.float64, device="cuda")
        for h in range(c["H"]):
            k, v = s["k"][:, h // per].double(), s["v"][:, h // per].double()
            state[:, h] = math.exp(float(s["g"][h].double())) * state[:, h] + k[:, :, None] * v[:, None, :]
            o[:, h] = (s["q"][:, h].double()[:, None, :] @ state[:, h])[:, 0] / math.sqrt(c["Dk"])
        return [o, state]
    if c["op"] == "rotary":
        out = [_exact_rotary(s["q"], s, c, False), _exact_rotary(s["k"], s, c, False)]
        return out + ([_exact_rotary(x, s, c, True) for x in s["do"]] if c["train"] else [])
    keep = torch.from_numpy(_exact_keep(s["x"].numel(), c["p"], s["seed"], s["offset"])).cuda().view(s["x"].shape)
    kept = keep.double() / (1.0 - c["p"])
    out = [s["x"].double() * kept + (0.0 if s["residual"] is None else s["residual"].double())]
    if c["train"]:
        out.append(s["do"].double() * kept)
        if s["residual"] is not None:
            out.append(s["do"].double())
    return out
