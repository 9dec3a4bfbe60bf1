"""The bounds that the attention over four bits is held to tell apart what float32 adds (CPU, by an emulation of the operands)."""
import math

import pytest
import torch

from plain import q4_attention_bounds as B
from plain import q4_plain as Q

HD = 128


def aligned_case(kind, hd=HD):
    """Queries whose float16 parts round the same way in every entry, over keys of one sign (``q``); probabilities that no float16
    number holds, of small scores (``p``). [1, 1, hd] queries in float32, keys and values [n, 1, hd]."""
    gen = torch.Generator().manual_seed(3)
    n = 24
    q = torch.full((1, 1, hd), 1.0 + 0.95 * 2.0 ** -11)
    level = torch.linspace(0.02, 0.3, n)[torch.randperm(n, generator=gen)]
    k = level[:, None, None].expand(n, 1, hd).contiguous()
    v = torch.where(level > 0.16, 1.0, -1.0)[:, None, None].expand(n, 1, hd).contiguous()
    if kind == "p":
        q, k = torch.ones(1, 1, hd), 0.15 * k
        v = (1.0 + torch.rand(n, 1, hd // 32, generator=gen)).repeat_interleave(32, -1) * torch.where(torch.arange(n) % 3 == 0, 1.0, -0.6)[:, None, None]
    return q, k, v


@pytest.mark.parametrize("kind", ["q", "p"])
@pytest.mark.parametrize("hd", [64, 128])
def test_the_float32_bound_rejects_a_single_part(kind, hd):
    q, k, v = aligned_case(kind, hd)
    kh, vh, sv = Q.q4(k, 32), Q.q4(v, 32), B.scales(v)
    n, scale = k.shape[0], 1.0 / math.sqrt(hd)
    want, tol = B.rows(q, kh, vh, sv, n - 1, scale)
    assert torch.allclose(want, Q.attention(q, kh, vh, n - 1, scale), rtol=1e-12, atol=0)

    def off(q_parts, p_parts):
        return float(((B.emulated(q, kh, vh, sv, n - 1, scale, q_parts, p_parts) - want).abs() / tol).max())
    assert off(2, 2) < 0.5
    assert off(1, 2) > 2 if kind == "q" else off(2, 1) > 2
