"""Rows of x as they come, columns of wider rows, at odd places or one row for all: the products of four-bit weights take each on the
kernel that its number of rows asks for."""
import pytest
import torch

from test_four_bits_gpu import DEV, product_case

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("M,dtype", [(3, BF), (3, F32), (40, BF), (40, F32), (300, BF), (1100, BF)])
def test_rows_at_odd_places_and_rows_that_overlap(M, dtype, monkeypatch):
    from spissa_b200.csrc import lib
    from spissa_b200.parts.linear import GatedLinear4, Linear4
    N, K = 128, 256
    x, w, y, mag = product_case(M, N, K, 64, dtype, M)
    lin, gated = Linear4(w.to(DEV)), GatedLinear4(w.to(DEV), w.flip(0).to(DEV))
    whole, plain = lin(x.to(DEV), out_dtype=F32), gated(x.to(DEV), dtype)
    # sums of K products in 32 bits, cut to 24 bits a step at most, as test_four_bits_gpu.py counts them
    assert bool(((whole.cpu().double() - y).abs() <= (K * 2.0 ** -23 + 2.0 ** -22) * mag).all())

    def slow(*args, **kw):
        raise AssertionError("the FFMA product was asked for")
    monkeypatch.setattr(lib, "gemm_generic", slow)
    wide = torch.full((M, K + 44), 9.0, dtype=dtype, device=DEV)
    for at in (0, 1, 3, 4, 8, 16):
        wide[:, at:at + K] = x.to(DEV)
        assert torch.equal(lin(wide[:, at:at + K], out_dtype=F32), whole), at
        assert torch.equal(gated(wide[:, at:at + K], dtype), plain), at
    row = x[:1].to(DEV)
    assert torch.equal(lin(row.expand(M, K), out_dtype=F32), lin(row.repeat(M, 1), out_dtype=F32))
    assert torch.equal(gated(row.expand(M, K), dtype), gated(row.repeat(M, 1), dtype))
