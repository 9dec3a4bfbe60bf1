"""Products with rows of the weight that stand for zeros beside a large number in every group: a zero adds nothing, exactly, whichever
kernel takes the product."""
import pytest
import torch

from test_four_bits_gpu import DEV

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M", [1, 8, 9, 16, 17, 300])
def test_zeros_beside_large_weights_add_nothing(M, group, dtype):
    from spissa_b200.parts.linear import GatedLinear4, Linear4
    N, K = 200, 1024
    gen = torch.Generator().manual_seed(M + group)
    x = torch.randn(M, K, generator=gen)
    x[:, ::group], x[:, 7::group] = 0.0, 0.0                         # the large weights' columns are not asked for
    w = torch.zeros(N, K)
    w[:, ::group] = 1.0 + torch.rand(N, K // group, generator=gen)
    w[:, 7::group] = -1.0 - torch.rand(N, K // group, generator=gen)
    w[40:80] = 1e-3 * torch.randn(40, K, generator=gen)              # ordinary rows among them
    lin = Linear4(w.to(DEV), group)
    out = lin(x.to(dtype).to(DEV), out_dtype=F32)
    zero = torch.ones(N, dtype=torch.bool)
    zero[40:80] = False
    assert bool((out.cpu()[:, zero] == 0).all()) and bool((out.cpu()[:, ~zero] != 0).any())
    gated = GatedLinear4(w.to(DEV), w.flip(1).to(DEV), group=group)(x.to(dtype).to(DEV), dtype)
    assert bool((gated.cpu()[:, zero] == 0).all())
