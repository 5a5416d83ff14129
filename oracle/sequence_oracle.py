"""The sequence operators from their definitions, in 64 bits on the CPU (test infrastructure only).

Linear attention: the sum over the tokens that a row sees; `attention_recurrent` is the same token by token.  Gradients are torch's
own of these sums.  Dropout's mask: Philox in Python's whole numbers."""
import math

import numpy as np
import torch


def _weights(g, T):
    """[H,T,T]: exp(g (i - j)) where j <= i; a row's own weight is one whatever the decay."""
    i = torch.arange(T, dtype=torch.float64)
    apart = i[:, None] - i[None, :]
    w = torch.exp(g[:, None, None] * apart.clamp(min=1.0))
    return torch.where(apart > 0, w, torch.where(apart == 0, 1.0, 0.0))


def attention(q, k, v, g, s0=None, lengths=None, scale=None):
    """fp64 [B,T,.,.] -> (o, state); rows behind a length are zero and are not read."""
    B, T, H, Dk = q.shape
    G, Dv = k.shape[2], v.shape[3]
    scale = Dk ** -0.5 if scale is None else scale
    lengths = [T] * B if lengths is None else [int(n) for n in lengths]
    outs, states = [], []
    for b in range(B):
        n = lengths[b]
        kk, vv = (x[b, :n].repeat_interleave(H // G, dim=1).transpose(0, 1) for x in (k, v))     # [H,n,.]
        qq = q[b, :n].transpose(0, 1)
        w = _weights(g, n)
        t = torch.arange(n, dtype=torch.float64)
        o = (qq @ kk.transpose(1, 2) * w) @ vv
        s = (kk * (w[:, n - 1, :, None] if n else 1.0)).transpose(1, 2) @ vv
        if s0 is not None:
            o = o + torch.exp(g[:, None] * (t + 1))[..., None] * (qq @ s0[b])
            s = s + (torch.exp(g * n)[:, None, None] if n else 1.0) * s0[b]
        outs.append(torch.cat([scale * o.transpose(0, 1), torch.zeros(T - n, H, Dv, dtype=torch.float64)]))
        states.append(s)
    return torch.stack(outs), torch.stack(states)


def attention_recurrent(q, k, v, g, s0=None, scale=None):
    B, T, H, Dk = q.shape
    rep = H // k.shape[2]
    k, v = k.repeat_interleave(rep, dim=2), v.repeat_interleave(rep, dim=2)
    s = torch.zeros(B, H, Dk, v.shape[3], dtype=torch.float64) if s0 is None else s0.clone()
    out = []
    for t in range(T):
        s = torch.exp(g)[None, :, None, None] * s + k[:, t, :, :, None] * v[:, t, :, None, :]
        out.append((Dk ** -0.5 if scale is None else scale) * (q[:, t, :, None, :] @ s)[:, :, 0])
    return torch.stack(out, dim=1), s


def rotary(x, positions, frequencies, layout, scale=1.0):
    """x [B,T,H,D] fp64; the angle's whole turns are taken off in exact arithmetic of the fp64 values."""
    B, T, H, D = x.shape
    r = len(frequencies)
    pos = positions.reshape(-1, T).expand(B, T)
    out = x.clone()
    for m in range(r):
        i, j = (m, m + r) if layout == "half" else (2 * m, 2 * m + 1)
        ang = torch.tensor([[math.fmod(float(p) * float(frequencies[m]), 2 * math.pi) for p in row] for row in pos.tolist()],
                           dtype=torch.float64)[:, :, None]
        c, s = scale * torch.cos(ang), scale * torch.sin(ang)
        a, b = x[..., i], x[..., j]
        out[..., i], out[..., j] = a * c - b * s, b * c + a * s
    return out


def philox_words(block, offset, seed, rounds=7):
    M = 0xFFFFFFFF
    x = [block & M, block >> 32, offset & M, offset >> 32]
    k = [seed & M, seed >> 32]
    for _ in range(rounds):
        a, b = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
        x = [(b >> 32) ^ x[1] ^ k[0], b & M, (a >> 32) ^ x[3] ^ k[1], a & M]
        k = [(k[0] + 0x9E3779B9) & M, (k[1] + 0xBB67AE85) & M]
    return x


def keep_mask(n, p, seed, offset, first=0):
    """bool [n]: element first + i kept."""
    t = int(p * 2.0 ** 32)
    words = {}
    out = np.empty(n, dtype=bool)
    for i in range(n):
        e = first + i
        if e // 4 not in words:
            words[e // 4] = philox_words(e // 4, offset, seed)
        out[i] = words[e // 4][e % 4] >= t
    return out
