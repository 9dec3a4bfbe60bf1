"""Attention over keys and values of four bits in 64 bits (CPU), with a bound for what kernels of 32-bit sums may be off by, and an
emulation of their operands' rounding that shows what the bound tells apart.

The bound of an output, from its terms. p_k: probabilities, v_k = s_k (c_k − z_k): a group's scale and codes, n keys.
* A score passes, for every group of 32 entries, up to four tensor-core products of 16 terms, each of which may cut its 17 addends
  below the 24 bits of the largest (2^-23 of the sum of sizes each), and then one 32-bit sum a group: 70 · 2^-23 of the size of its
  terms; float32 queries are two float16 numbers, off by 2^-22 of an entry; the exponent's own product, rounding and 2^x: 4 · 2^-23 of
  the score and 2^-21.
  ``size``: Σ |q| |k|.
* So a probability is off by e^δ − 1 of itself, in the sum over the keys and in the weighted one: 2 (e^δ − 1) Σ p |v|.
* p s is one float16 number (2^-11 of itself) or two (2^-22), and no less than a smallest step off, which is 2^-33 of the largest
  p s that the group of columns has met (float32: 2^-44): a key's share of that times |c − z| <= 15.
* Sums: a page of 64 keys is a product of 16 for each of four warps, 17 addends cut as above; the lanes' and warps' sums and up to some
  dozen chunks' in 32 bits: (17 · 2^-23 · pages + 40 · 2^-24) of Σ p |v|, the sum of the probabilities likewise.
* bfloat16 outputs: half a step, 2^-8 of the output.
"""
import math

import torch

F64 = torch.float64


def scales(x, group=32):
    """Every group's s, spread over its columns, float64."""
    g = x.to(F64).reshape(-1, group)
    m, e = torch.frexp((g.amax(1).clamp(min=0) - g.amin(1).clamp(max=0)) / 15.0)
    s = torch.ldexp(torch.ceil(m * 16.0) / 16.0, e)
    return s[:, None].expand(-1, group).reshape(x.shape)


def rows(q, k, v, sv, first, scale, window=None, sink=None):
    """(want, tolerance), each [n, nh, hd], for queries ``q`` [n, nh, hd] at positions first ..; ``k``, ``v`` [L, nkv, hd] float64:
    what the codes stand for, ``sv`` the values' groups' scales."""
    n, nh, hd = q.shape
    G, bf16 = nh // k.shape[1], q.dtype == torch.bfloat16
    want, tol = torch.zeros(n, nh, hd, dtype=F64), torch.zeros(n, nh, hd, dtype=F64)
    for i in range(n):
        p, lowest = first + i, max(0, first + i + 1 - window) if window else 0
        for h in range(nh):
            ks, vs = k[lowest:p + 1, h // G], v[lowest:p + 1, h // G]
            x = q[i, h].to(F64)
            score = ks @ x * scale
            size = ks.abs() @ x.abs() * scale
            top = score.max() if sink is None else torch.maximum(score.max(), sink[h].to(F64))
            w = torch.exp(score - top)
            w = w / (w.sum() + (torch.exp(sink[h].to(F64) - top) if sink is not None else 0.0))
            mag, ps, L = w @ vs.abs(), w[:, None] * sv[lowest:p + 1, h // G], ks.shape[0]
            delta = float(((70 * 2.0 ** -23 + (0 if bf16 else 2.0 ** -22)) * size + 2.0 ** -21 * score.abs()).max()) + 2.0 ** -21
            want[i, h] = w @ vs
            tol[i, h] = (2 * math.expm1(delta) + (2.0 ** -11 if bf16 else 2.0 ** -22) + 2 * (17 * 2.0 ** -23 * (L // 64 + 2) + 40 * 2.0 ** -24)) * mag \
                + L * (2.0 ** -33 if bf16 else 2.0 ** -44) * 15 * ps.amax(0)
            if bf16:
                tol[i, h] += 2.0 ** -8 * (want[i, h].abs() + tol[i, h])
    return want, tol


def halves(x, parts):
    """float64 numbers as the sum of ``parts`` float16 ones, the second times 2^11."""
    out = x.to(torch.float16).to(F64)
    return out if parts == 1 else out + ((x - out) * 2.0 ** 11).to(torch.float16).to(F64) * 2.0 ** -11


def power_below(x, exponent):
    """The power of two that brings x > 0 into [2^(exponent − 1), 2^exponent)."""
    return torch.ldexp(torch.ones_like(x), (exponent - torch.frexp(x)[1]).to(torch.int32))


def emulated(q, k, v, sv, first, scale, q_parts, p_parts):
    """The operands' rounding alone: q as ``q_parts`` float16 numbers under a power of two for its row, p s as ``p_parts`` under one for
    each group of columns, everything else in 64 bits."""
    n, nh, hd = q.shape
    G, out = nh // k.shape[1], torch.zeros(n, nh, hd, dtype=F64)
    for i in range(n):
        for h in range(nh):
            ks, vs, s = (t[:first + i + 1, h // G] for t in (k, v, sv))
            x = q[i, h].to(F64)
            up = power_below(x.abs().amax(), 15)
            odd = torch.tensor([1.0, 1.0, 0.0625, 0.0625], dtype=F64).repeat(hd // 4)        # every other pair meets 16 c
            x = halves(x * up * odd, q_parts) / (up * odd)
            w = torch.exp(ks @ x * scale - (ks @ x).max() * scale)
            ps = w[:, None] * s
            norm = power_below(ps.amax(0), 8)
            out[i, h] = (halves(ps * norm, p_parts) / norm * torch.where(s > 0, vs / s, torch.zeros_like(vs))).sum(0) / w.sum()
    return out
