"""The recurrent layer's operators from their definitions, in 64 bits on the CPU, token by token (test infrastructure only).  Gradients are
torch's own of these sums.  With magnitudes=True the same sums over the terms' magnitudes, which a result's error on the way is bounded against."""
import torch


def silu(x):
    return x / (1 + torch.exp(-x))


def softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def conv(x, weight, bias=None, start=None, lengths=None, act=None):
    """fp64 [B,T,C] -> (y, the last K - 1 inputs); rows behind a length are zero and are not read."""
    B, T, C = x.shape
    K = weight.shape[1]
    ys, ends = [], []
    for b in range(B):
        n = T if lengths is None else int(lengths[b])
        front = torch.zeros(K - 1, C, dtype=x.dtype) if start is None else start[b]
        row = torch.cat([front, x[b, :n]])
        p = torch.stack([(row[t:t + K] * weight.t()).sum(0) for t in range(n)]) if n else torch.zeros(0, C, dtype=x.dtype)
        p = p if bias is None else p + bias
        ys.append(torch.cat([silu(p) if act == "silu" else p, torch.zeros(T - n, C, dtype=x.dtype)]))
        ends.append(row[n:])
    return torch.stack(ys), torch.stack(ends)


def scan(x, delta, A, B, C, D=None, z=None, bias=None, start=None, lengths=None, plus=False):
    """fp64 [batch,T,channels], [batch,T,groups,N] -> (y, state)."""
    batch, T, channels = x.shape
    share, N = channels // B.shape[2], A.shape[1]
    ys, ends = [], []
    for b in range(batch):
        n = T if lengths is None else int(lengths[b])
        h = torch.zeros(channels, N, dtype=x.dtype) if start is None else start[b]
        rows = []
        for t in range(n):
            d = delta[b, t] if bias is None else delta[b, t] + bias
            d = softplus(d) if plus else d
            h = torch.exp(d[:, None] * A) * h + (d * x[b, t])[:, None] * B[b, t].repeat_interleave(share, dim=0)
            y = (h * C[b, t].repeat_interleave(share, dim=0)).sum(1)
            y = y if D is None else y + D * x[b, t]
            rows.append(y if z is None else y * silu(z[b, t]))
        ys.append(torch.cat([torch.stack(rows) if n else torch.zeros(0, channels, dtype=x.dtype), torch.zeros(T - n, channels, dtype=x.dtype)]))
        ends.append(h)
    return torch.stack(ys), torch.stack(ends)


def normed(x, group, kind, eps):
    rows = x.reshape(*x.shape[:-1], -1, group)
    if kind == "layer":
        rows = rows - rows.mean(-1, keepdim=True)
    return (rows / torch.sqrt((rows * rows).mean(-1, keepdim=True) + eps)).reshape(x.shape)


def norm_gate(x, weight, gate=None, residual=None, scale=None, next_weight=None, group=None, eps=1e-5, kind="rms", act="silu"):
    y = normed(x, x.shape[-1] if group is None else group, kind, eps) * weight
    if gate is not None:
        y = y * (silu(gate) if act == "silu" else torch.sigmoid(gate) if act == "sigmoid" else gate)
    y = y if scale is None else y * scale
    y = y if residual is None else y + residual
    return (y,) if next_weight is None else (y, normed(y, x.shape[-1], kind, eps) * next_weight)


# ------------------------------------------------------------------------------------------------
# The magnitudes of what the results are sums of: the same formulas with every term's absolute value
# ------------------------------------------------------------------------------------------------
def conv_sizes(x, weight, bias=None, start=None, lengths=None, act=None, dy=None, dend=None):
    """{name: size}: a pre-activation's terms; of a gradient in front of silu |dy| (1 + that), as the slope's own error goes with it."""
    B, T, C = x.shape
    K = weight.shape[1]
    leaves = [t if t is None else t.abs().requires_grad_(True) for t in (x, weight, bias, start)]
    p, end = conv(leaves[0], leaves[1], leaves[2], leaves[3], lengths)
    out = {"y": p.detach(), "state": end.detach()}
    if dy is not None:
        g = dy.abs() * (1 + p.detach()) if act == "silu" else dy.abs()
        if lengths is not None:
            g = g * (torch.arange(T)[None, :] < torch.as_tensor(lengths)[:, None])[..., None]
        torch.autograd.backward([p, end], [g, torch.zeros_like(end) if dend is None else dend.abs()])
        out.update({n: torch.zeros_like(t) if t.grad is None else t.grad for n, t in zip(("dx", "dweight", "dbias", "dstart"), leaves) if t is not None})
    return out


def scan_sizes(x, delta, A, B, C, D=None, z=None, bias=None, start=None, lengths=None, plus=False, dy=None, dend=None):
    batch, T, channels = x.shape
    G, N = B.shape[2], A.shape[1]
    share = channels // G
    D = torch.zeros(channels, dtype=x.dtype) if D is None else D.abs()
    zero = lambda t: torch.zeros_like(t)
    out = {n: zero(t) for n, t in (("y", x), ("dx", x), ("ddelta", x), ("dz", x), ("dA", A), ("dB", B), ("dC", B), ("dD", D), ("dbias", D))}
    out["state"] = torch.zeros(batch, channels, N, dtype=x.dtype)
    out["dstart"], total = out["state"].clone(), 0.0
    for b in range(batch):
        n = T if lengths is None else int(lengths[b])
        raw = delta[b, :n] if bias is None else delta[b, :n] + bias
        d = softplus(raw) if plus else raw
        slope = torch.sigmoid(raw) if plus else torch.ones_like(raw)
        s = torch.ones_like(raw) if z is None else silu(z[b, :n]).abs()
        Bm, Cm = (t[b, :n].abs().repeat_interleave(share, dim=1) for t in (B, C))
        xm, dm = x[b, :n].abs(), d.abs()
        h = out["state"][b].clone() if start is None else start[b].abs()
        hs, powers = [h], torch.exp(d[..., None] * A)
        inner = torch.zeros_like(raw)
        for t in range(n):
            h = powers[t] * h + (dm[t] * xm[t])[:, None] * Bm[t]
            hs.append(h)
            inner[t] = (h * Cm[t]).sum(1) + D * xm[t]
        out["y"][b, :n], out["state"][b] = inner * s, h
        total = max(total, float((dm[..., None] * A.abs()).sum(0).max()) if n else 0.0)
        if dy is None:
            continue
        q = dy[b, :n].abs() * s
        g = zero(h) if dend is None else dend[b].abs()
        if z is not None:
            sig = torch.sigmoid(z[b, :n])
            out["dz"][b, :n] = dy[b, :n].abs() * inner * sig * (1 + z[b, :n].abs() * (1 - sig))
        for t in reversed(range(n)):
            g = g + q[t][:, None] * Cm[t]
            out["dC"][b, t] = (q[t][:, None] * hs[t + 1]).view(G, share, N).sum(1)
            out["dB"][b, t] = ((dm[t] * xm[t])[:, None] * g).view(G, share, N).sum(1)
            into, g0 = (g * Bm[t]).sum(1), g
            g = powers[t] * g
            turn = g * hs[t]
            out["dA"] += dm[t][:, None] * turn
            dd = (xm[t] * into + (A.abs() * turn).sum(1)) * slope[t]
            out["ddelta"][b, t] = dd
            out["dbias"] += dd
            out["dx"][b, t] = dm[t] * into + D * q[t]
            out["dD"] += q[t] * xm[t]
        out["dstart"][b] = g
    return out, total


def _normed_sizes(x, size, group, kind, eps):
    """(unit, its size, 1 / the root) of values x whose own terms are `size`"""
    rows, big = (t.reshape(*t.shape[:-1], -1, group) for t in (x, size))
    if kind == "layer":
        rows, big = rows - rows.mean(-1, keepdim=True), big + big.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((rows * rows).mean(-1, keepdim=True) + eps)
    rho = torch.sqrt((big * big).mean(-1, keepdim=True)) * r
    unit = rows * r
    return unit.reshape(x.shape), (big * r + unit.abs() * rho).reshape(x.shape), (r * (1 + rho)).expand_as(rows).reshape(x.shape)


def norm_sizes(x, weight, gate=None, residual=None, scale=None, next_weight=None, group=None, eps=1e-5, kind="rms", act="silu", dy=None, dn=None):
    C = x.shape[-1]
    group = C if group is None else group
    lead = tuple(range(x.dim() - 1))
    mean = lambda t, g: t.reshape(*t.shape[:-1], -1, g).mean(-1, keepdim=True).expand(*t.shape[:-1], -1, g).reshape(t.shape)
    unit, big, r = _normed_sizes(x, x.abs(), group, kind, eps)
    a = torch.ones_like(x) if gate is None else (silu(gate) if act == "silu" else torch.sigmoid(gate) if act == "sigmoid" else gate)
    s = torch.ones(C, dtype=x.dtype) if scale is None else scale
    res = torch.zeros_like(x) if residual is None else residual
    y, size = unit * weight * a * s + res, big * (weight * a * s).abs() + res.abs()
    out = {"y": size}
    if next_weight is not None:
        unit2, big2, r2 = _normed_sizes(y, size, C, kind, eps)
        out["n"] = big2 * next_weight.abs()
    if dy is None:
        return out
    t = dy.abs()
    if next_weight is not None:
        g = dn.abs() * next_weight.abs()
        t = t + r2 * (g + (mean(g, C) if kind == "layer" else 0) + big2 * mean(g * big2, C))
        out["dnext_weight"] = (dn.abs() * big2).sum(lead)
    out["dresidual"], out["dscale"] = t, (t * big * (weight * a).abs()).sum(lead)
    g = t * s.abs()
    if gate is not None:
        p = torch.sigmoid(gate)
        slope = p * (1 + gate.abs() * (1 - p)) if act == "silu" else p if act == "sigmoid" else torch.ones_like(gate)
        out["dgate"] = g * big * weight.abs() * slope
    g = g * a.abs()
    out["dweight"] = (g * big).sum(lead)
    g = g * weight.abs()
    out["dx"] = r * (g + (mean(g, group) if kind == "layer" else 0) + big * mean(g * big, group))
    return out
