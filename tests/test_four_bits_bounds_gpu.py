"""Attention over four bits: what its sums may not be off by."""
import pytest
import torch

import kernel_harness as KH
from test_four_bits_edges_gpu import attend
from test_four_bits_gpu import DEV, fill

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hd", [64, 128])
def test_columns_of_zeros_stay_zeros(hd, dtype):
    """Zero stands for itself exactly, and a weighted sum of zeros is zero, however large the other columns of the group are."""
    n, nh, nkv = 3000, 4, 2
    gen = torch.Generator().manual_seed(hd)
    q, k = torch.randn(1, nh, hd, generator=gen).to(dtype), torch.randn(n, nkv, hd, generator=gen)
    v = torch.zeros(n, nkv, hd)
    v[..., ::32] = torch.randn(n, nkv, hd // 32, generator=gen) * 5
    v[..., 1::32] = torch.randn(n, nkv, hd // 32, generator=gen) * 5
    meta = KH.paged_meta([1], [n - 1], DEV)
    pool = fill(meta, [(k, v)], nkv, hd)
    zero = (torch.arange(hd) % 32 > 1).repeat(nh)
    for plan in (None, (1, 47, 1), (2, 10, 5)):
        out = attend(meta, pool, q, nh, nkv, hd, [1], None, None, plan)
        assert bool((out[0].cpu()[zero] == 0).all()) and bool((out[0].cpu()[~zero] != 0).all())
