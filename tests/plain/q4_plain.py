"""Four bits a number, stated plainly in 64 bits (CPU): the format, products, rotation, attention.

A group x of neighbouring numbers: lo = min(0, min x), hi = max(0, max x), s = (hi − lo)/15 rounded up to four significant
bits, z = round(−lo/s), c = clamp(round(x/s) + z, 0, 15) with ties to even; it stands for s·(c − z). hi − lo < 2^-100: zeros.
An entry that is not finite or beyond 2^100: NaN throughout.
"""
import math

import torch

F64 = torch.float64


def q4(x, group):
    """What ``x`` (any floating tensor, last dimension a multiple of ``group``) stands for in four bits, float64."""
    shape = x.shape
    g = x.to(F64).reshape(-1, group)
    lo = g.min(1, keepdim=True).values.clamp(max=0.0)
    hi = g.max(1, keepdim=True).values.clamp(min=0.0)
    m, e = torch.frexp((hi - lo) / 15.0)
    s = torch.ldexp(torch.ceil(m * 16.0) / 16.0, e)
    d = torch.where(s > 0, s, torch.ones_like(s))
    z = torch.round(-lo / d)
    c = (torch.round(g / d) + z).clamp(0.0, 15.0)
    out = torch.where(hi - lo < 2.0 ** -100, torch.zeros_like(g), s * (c - z))
    bad = ~(g.abs() <= 2.0 ** 100).all(1, keepdim=True)
    return torch.where(bad, torch.full_like(g, float("nan")), out).reshape(shape)


def rotate(x, positions, inv_freq, rd):
    """x [T, heads, hd]: dim i turned with dim i + rd/2 by position · inv_freq_i, in 64 bits, rounded once to 32."""
    if not rd:
        return x.float()
    h = rd // 2
    angle = positions.to(F64)[:, None] * inv_freq.to(F64)[None, :h]
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = x[..., :h].to(F64), x[..., h:rd].to(F64)
    return torch.cat([a * c - b * s, b * c + a * s, x[..., rd:].to(F64)], -1).float()


def attention(q, k, v, first, scale, window=None, sink=None):
    """q [n, nh, hd] at positions first.. over k, v [L, nkv, hd] (float64): [n, nh, hd]. A row without a key is zeros."""
    n, nh, hd = q.shape
    G = nh // k.shape[1]
    out = torch.zeros(n, nh, hd, dtype=F64)
    for i in range(n):
        p = first + i
        lowest = max(0, p + 1 - window) if window else 0
        ks, vs = k[lowest:p + 1], v[lowest:p + 1]
        for h in range(nh):
            if ks.shape[0] == 0:
                continue
            score = (ks[:, h // G] @ q[i, h].to(F64)) * scale
            top = float(score.max()) if sink is None else max(float(score.max()), float(sink[h]))
            w = torch.exp(score - top)
            total = w.sum() + (math.exp(float(sink[h]) - top) if sink is not None else 0.0)
            out[i, h] = (w[:, None] * vs[:, h // G]).sum(0) / total
    return out
