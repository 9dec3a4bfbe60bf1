"""Products and attention over four bits are as near to 64 bits as a plain evaluation in 32: no operand is held in a form that costs the
sums bits. Outputs are float32; the plain evaluation is elementary products, sums and exponentials of the same numbers."""
import math

import pytest
import torch

import kernel_harness as KH
from plain import q4_plain as Q
from test_four_bits_edges_gpu import attend
from test_four_bits_gpu import DEV, fill

pytestmark = pytest.mark.gpu
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def off(out, want):
    return float((out.double() - want).norm() / want.norm())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M", [1, 8, 16, 40])
@pytest.mark.parametrize("K,group", [(2048, 32), (2048, 128), (8192, 64)])
def test_products_are_as_near_as_plain_ones_in_32_bits(M, K, group, dtype):
    from spissa_b200.parts.linear import Linear4
    gen = torch.Generator().manual_seed(M + group)
    x, w = torch.randn(M, K, generator=gen).to(dtype).to(DEV), 0.02 * torch.randn(512, K, generator=gen)
    what = Q.q4(w, group).to(DEV)
    want, plain = x.double() @ what.T, x.float() @ what.float().T
    # (three times: a sum's error goes by its order, and both are sums of a few dozen to some thousand roundings)
    assert off(Linear4(w.to(DEV), group)(x, out_dtype=F32), want) <= 3 * off(plain, want)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("tokens,before", [(1, 2000), (1, 20000), (24, 500)])
def test_attention_is_as_near_as_a_plain_one_in_32_bits(tokens, before, hd):
    nh, nkv = 8, 2
    gen = torch.Generator().manual_seed(hd + tokens)
    n = before + tokens
    q, k, v = (torch.randn(s, h, hd, generator=gen) for s, h in ((tokens, nh), (n, nkv), (n, nkv)))
    kh, vh = Q.q4(k, 32).to(DEV), Q.q4(v, 32).to(DEV)

    def plain(dtype):
        out = torch.empty(tokens, nh, hd, dtype=dtype, device=DEV)
        hidden = torch.arange(n, device=DEV)[None] > before + torch.arange(tokens, device=DEV)[:, None]
        for h in range(nh):
            score = (q[:, h].to(DEV).to(dtype) @ kh[:, h // 4].to(dtype).T * (1.0 / math.sqrt(hd))).masked_fill(hidden, -math.inf)
            p = torch.exp(score - score.amax(1, keepdim=True))
            out[:, h] = (p / p.sum(1, keepdim=True)) @ vh[:, h // 4].to(dtype)
        return out.reshape(tokens, -1)
    want = plain(F64)
    meta = KH.paged_meta([tokens], [before], DEV)
    out = attend(meta, fill(meta, [(k, v)], nkv, hd), q, nh, nkv, hd, [tokens], None, None, None)
    assert off(out, want) <= 2 * off(plain(F32), want)
