"""Weights and caches of four bits against plain 64-bit arithmetic.

What a group stands for is compared for equality: scales, zeros and codes are defined by exact quotients, and the numbers
are bfloat16 (s has four significant bits, c − z four). Tolerances of products and attention: a sum of n products whose
terms are rounded relatively by eps each is off by at most (n · eps32 + eps) times the sum of their magnitudes; an output
rounded to bfloat16 by 2^-8 of its own. In bfloat16 a probability is rounded by at most 2^-8 of itself, so an output by
2^-8 of Σ p |v|.
"""
import math

import pytest
import torch

import kernel_harness as KH
from plain import q4_plain as Q

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


def numbers(*shape, seed=0, spread=2.0, dtype=F32):
    """Normal numbers whose groups of 32 differ in size by powers of e^spread."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=gen)
    size = torch.exp(spread * torch.randn(*shape[:-1], -(-shape[-1] // 32), generator=gen)).repeat_interleave(32, -1)[..., :shape[-1]]
    return (x * size).to(dtype)


# ------------------------------------------------------------------------------------------------------------- weights
@pytest.mark.parametrize("rows,K,group,dtype", [(1, 32, 32, F32), (16, 64, 64, BF), (17, 96, 32, BF), (130, 128, 128, F32),
                                                (45, 1152, 128, BF), (64, 2048, 64, F32)])
def test_packed_weights_stand_for_the_definitions_numbers(rows, K, group, dtype):
    from spissa_b200.csrc import lib
    w = numbers(rows, K, seed=rows, dtype=dtype)
    codes, scales = lib.q4_pack(w.to(DEV), group)
    want = Q.q4(w, group)
    for dt in (F32, BF):
        out = torch.full((rows, K), 7.0, dtype=dt, device=DEV)
        lib.q4_unpack(codes, scales, out, group)
        assert torch.equal(out.cpu().double(), want)


def test_a_groups_edges():
    """Ties between two codes, zeros, one sign only, tiny and huge ranges, entries that are not finite."""
    from spissa_b200.csrc import lib
    g = torch.zeros(12, 32)
    g[0] = torch.arange(32) * 0.5 - 4.0                 # range 15.5: s = 1.125
    g[1, :2] = torch.tensor([-7.0, 8.0])                # range 15: s = 1, every half below is a tie
    g[1, 2:17] = torch.arange(15) - 6.5
    g[2] = torch.rand(32) + 3.0                         # positive: z = 0
    g[3] = -torch.rand(32) - 3.0                        # negative: z = 15
    g[4, 5] = 2.0 ** -101                               # below the smallest range
    g[5, 5] = 2.0 ** -100
    g[6, 3], g[6, 4] = 2.0 ** 100, -2.0 ** 100
    g[7, 3] = 1.1 * 2.0 ** 100
    g[8, 9] = float("nan")
    g[9, 9] = float("-inf")
    g[10, 0], g[10, 1:] = 15.0, 2.0 ** -20              # everything but one entry rounds to zero
    g[11] = torch.where(torch.arange(32) % 2 == 0, 1.0, -1.0) * (1.0 + torch.arange(32) * 2.0 ** -23)
    codes, scales = lib.q4_pack(g.to(DEV), 32)
    out = torch.empty(12, 32, device=DEV)
    lib.q4_unpack(codes, scales, out, 32)
    want = Q.q4(g, 32)
    assert torch.equal(torch.isnan(out.cpu()), torch.isnan(want))
    assert torch.equal(out.cpu().double().nan_to_num(3.0), want.nan_to_num(3.0))


def test_gate_and_up_rows_alternate_and_come_back():
    from spissa_b200.csrc import lib
    for I, block in ((40, 0), (128, 64), (256, 128), (7, 0)):
        w = numbers(2 * I, 64, seed=I)
        codes, scales = lib.q4_pack(w.to(DEV), 64, half=I)
        out = torch.empty(2 * I, 64, device=DEV)
        lib.q4_unpack(codes, scales, out, 64, half=I, block=block)
        want = Q.q4(w, 64)
        if block:
            want = torch.stack([want[:I].reshape(-1, block, 64), want[I:].reshape(-1, block, 64)], 1).reshape(2 * I, 64)
        assert torch.equal(out.cpu().double(), want)


def product_case(M, N, K, group, dtype, seed):
    x = numbers(M, K, seed=seed, spread=0.5, dtype=dtype)
    w = numbers(N, K, seed=seed + 1, spread=0.5, dtype=BF)
    what = Q.q4(w, group)
    y, mag = x.double() @ what.T, x.double().abs() @ what.abs().T
    return x, w, y, mag


PRODUCTS = [(1, 40, 32, 32), (1, 2048, 2048, 64), (2, 100, 96, 32), (5, 333, 640, 128), (8, 256, 1024, 64), (9, 72, 2176, 64), (16, 130, 4096, 128),
            (17, 128, 256, 64), (33, 200, 160, 32), (64, 384, 1024, 128), (100, 1000, 512, 64), (130, 64, 2048, 32), (301, 512, 1024, 64), (1100, 300, 256, 128)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M,N,K,group", PRODUCTS)
def test_product(M, N, K, group, dtype):
    from spissa_b200.parts.linear import Linear4
    x, w, y, mag = product_case(M, N, K, group, dtype, M + N)
    lin = Linear4(w.to(DEV), group)
    # sums: 32-bit, tensor cores may cut instead of round (2^-23 a step); float32 operands in three bfloat16 parts lose 2^-24 each
    tol = (K * 2.0 ** -23 + 2.0 ** -22) * mag
    out = lin(x.to(DEV), out_dtype=F32)
    assert out.dtype == F32 and bool(((out.cpu().double() - y).abs() <= tol).all())
    assert torch.equal(out, lin(x.to(DEV), out_dtype=F32))
    got = lin(x.to(DEV))
    assert got.dtype == dtype and bool(((got.cpu().double() - y).abs() <= tol + (2.0 ** -8 * (y.abs() + tol) if dtype == BF else 0)).all())
    base = numbers(M, N, seed=3, spread=0.1)
    acc = base.to(DEV)
    assert lin(x.to(DEV), out=acc, accumulate=True) is acc
    assert bool(((acc.cpu().double() - (base.double() + y)).abs() <= tol + 2.0 ** -23 * (base.double().abs() + y.abs() + tol)).all())


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M,I,K,group", [(1, 24, 64, 32), (1, 1024, 2048, 64), (3, 200, 384, 128), (8, 128, 1024, 128), (12, 77, 96, 32), (16, 512, 512, 64),
                                         (17, 128, 256, 64), (40, 100, 160, 32), (70, 192, 512, 128), (257, 256, 1024, 64)])
def test_gated_product(M, I, K, group, dtype, act):
    from spissa_b200.csrc import lib
    from spissa_b200.parts.linear import GatedLinear4
    x, wg, g, gm = product_case(M, I, K, group, dtype, M + I)
    _, wu, _, _ = product_case(M, I, K, group, dtype, M + I + 5)
    wg, wu = wg * (0.5 / float(g.abs().max()) ** 0.5), wu * 0.1
    wg, wu = wg.to(BF), wu.to(BF)
    pg, pu = Q.q4(wg, group), Q.q4(wu, group)
    g, u = x.double() @ pg.T, x.double() @ pu.T
    eg, eu = ((K * 2.0 ** -23 + 2.0 ** -22) * (x.double().abs() @ p.abs().T) for p in (pg, pu))
    f = (lambda z: z * torch.sigmoid(z)) if act == "silu" else (lambda z: 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))))
    y = f(g) * u * 0.75
    # |f'| <= 1.2 for both; the intermediate products of the plain way are rounded to the activations' type first (2^-8)
    r = 2.0 ** -8 if dtype == BF else 2.0 ** -22
    eg, eu = eg + r * g.abs(), eu + r * u.abs()
    tol = 0.75 * (1.2 * eg * (u.abs() + eu) + f(g).abs() * eu) + r * y.abs() + 2.0 ** -20 * (y.abs() + u.abs() * 2.0 ** -4)
    lin = GatedLinear4(wg.to(DEV), wu.to(DEV), lib.ACT_SILU if act == "silu" else lib.ACT_GELU, 0.75, group)
    out = lin(x.to(DEV), dtype)
    assert out.dtype == dtype and bool(((out.cpu().double() - y).abs() <= tol).all())


def test_products_of_rows_inside_wider_ones_and_at_odd_places():
    from spissa_b200.parts.linear import Linear4
    for dtype in (BF, F32):
        for M in (3, 40):
            x, w, y, mag = product_case(M, 96, 128, 32, dtype, 11)
            lin = Linear4(w.to(DEV), 32)
            wide = torch.full((M, 300), 9.0, dtype=dtype, device=DEV)
            tol = (128 * 2.0 ** -23 + 2.0 ** -22) * mag
            for at in (0, 8, 3):                                     # rows on and off 16-byte boundaries
                wide[:, at:at + 128] = x.to(DEV)
                out = lin(wide[:, at:at + 128], out_dtype=F32)
                assert bool(((out.cpu().double() - y).abs() <= tol).all())
            place = torch.full((M, 200), 5.0, device=DEV)
            lin(x.to(DEV), out=place[:, 13:109])                     # an output inside wider rows leaves the rest alone
            assert bool(((place[:, 13:109].cpu().double() - y).abs() <= tol).all())
            assert bool((place[:, :13] == 5).all()) and bool((place[:, 109:] == 5).all())


def test_products_without_rows_and_refusals():
    from spissa_b200.csrc.lib import KernelError
    from spissa_b200.parts.linear import GatedLinear4, Linear4
    w = numbers(64, 128, seed=1).to(DEV)
    assert Linear4(w)(torch.empty(0, 128, device=DEV, dtype=BF)).shape == (0, 64)
    assert GatedLinear4(w, w)(torch.empty(0, 128, device=DEV, dtype=BF), BF).shape == (0, 64)
    lin = Linear4(w, 32)
    x = torch.zeros(2, 128, device=DEV, dtype=BF)
    for bad in (lambda: Linear4(w[:, :100], 32), lambda: Linear4(w, 48), lambda: Linear4(w[:, :96], 64), lambda: Linear4(w.half()),
                lambda: Linear4(w.cpu()), lambda: lin(x[:, :96]), lambda: lin(x.half()), lambda: lin(x.cpu()),
                lambda: lin(torch.zeros(128, 2, device=DEV, dtype=BF).T), lambda: lin(x, out=torch.zeros(2, 63, device=DEV)),
                lambda: lin(x, out=torch.zeros(2, 64, device=DEV, dtype=BF), accumulate=True), lambda: lin(x, out_dtype=torch.float16)):
        with pytest.raises((KernelError, ValueError)):
            bad()
    with pytest.raises(ValueError):
        lin(x, accumulate=True)
    with pytest.raises(ValueError):
        GatedLinear4(w, w, act=2)
    with pytest.raises(ValueError):
        GatedLinear4(w, w[:32])


# --------------------------------------------------------------------------------------------------------------- cache
def fill(meta, kv, nkv, hd, poison=True):
    """A pool whose pages hold each sequence's keys and values; what no position owns holds bytes that read as NaN."""
    from spissa_b200.csrc import lib
    pool = lib.kv4_pool(meta.n_pages, nkv, hd, DEV)
    if poison:
        pool.fill_(0xff)
    for b, (k, v) in enumerate(kv):
        if not k.shape[0]:
            continue
        one = KH.paged_meta([k.shape[0]], [0], DEV)
        one.page_table = meta.page_table[b:b + 1].contiguous()
        lib.kv4_store(torch.cat([k, v], 1).reshape(k.shape[0], -1).to(DEV), None, pool, one, None, 0, nkv, hd, 0)
    return pool


HEADS = [(4, 2, 32), (32, 8, 64), (9, 3, 96), (8, 1, 128), (20, 2, 128), (3, 3, 64)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
@pytest.mark.parametrize("part", [0, 1, 2])
def test_store_rotates_and_quantises_and_load_reads_back(nh, nkv, hd, dtype, part):
    from spissa_b200.csrc import lib
    rd = (hd, hd // 2, 0)[part]
    new, before = [1, 70, 5], [0, 100000, 63]
    meta = KH.paged_meta(new, before, DEV, seed=hd)
    T = sum(new)
    x = numbers(T, (nh + 2 * nkv) * hd, seed=hd + nh, spread=1.0)
    freq = 1.0 / 500000.0 ** (torch.arange(0, max(rd, 2), 2).float() / max(rd, 2))
    pool = torch.randint(0, 256, (meta.n_pages, nkv, lib.kv4_tile_bytes(hd)), dtype=torch.uint8, device=DEV)
    held = pool.clone()
    q = torch.empty(T, nh * hd, dtype=dtype, device=DEV)
    lib.kv4_store(x.to(DEV), q, pool, meta, freq.to(DEV), nh, nkv, hd, rd)
    rows = x.view(T, nh + 2 * nkv, hd)
    turned = Q.rotate(rows[:, :nh + nkv], meta.positions.cpu(), freq, rd)
    # q: cos and sin rounded to 32 bits, a product and a sum each rounded: 4 half units of what the two terms come to
    want = turned[:, :nh].reshape(T, -1).double()
    size = rows[:, :nh].abs().amax(-1, keepdim=True).expand(-1, -1, hd).reshape(T, -1).double()
    assert bool(((q.cpu().double() - want).abs() <= 4 * 2.0 ** -24 * 2 * size + (2.0 ** -8 * want.abs() if dtype == BF else 0)).all())
    k, v = (torch.empty(T, nkv, hd, dtype=dtype, device=DEV) for _ in range(2))
    lib.kv4_load(pool, meta, k, v, nkv, hd)
    assert torch.equal(k.cpu().double(), Q.q4(turned[:, nh:], 32))
    assert torch.equal(v.cpu().double(), Q.q4(rows[:, nh + nkv:], 32))
    # storing the same rows into other bytes changes the same places to the same: what no token owns stayed as it was
    other = ~held
    lib.kv4_store(x.to(DEV), q, other, meta, freq.to(DEV), nh, nkv, hd, rd)
    assert bool(((pool == held) | (pool == other)).all())
    row_bytes = hd + hd // 8
    assert int((pool == other).sum()) - int(((pool == other) & (pool == held)).sum()) <= T * nkv * row_bytes
    before_q = q.clone()
    lib.kv4_store(x.to(DEV), q, held, meta, freq.to(DEV), nh, nkv, hd, rd, write_kv=False)
    assert torch.equal(q, before_q)


def attention_case(nh, nkv, hd, dtype, new, before, window, seed, sink=False):
    meta = KH.paged_meta(new, before, DEV, seed=seed)
    kv = [(numbers(n, nkv, hd, seed=seed + 3 * b, spread=0.3), numbers(n, nkv, hd, seed=seed + 3 * b + 1, spread=0.3))
          for b, n in enumerate(meta.total_len)]
    q = numbers(sum(new), nh, hd, seed=seed + 99, spread=0.2, dtype=dtype)
    sinks = numbers(1, nh, seed=seed + 7, spread=0.1)[0].contiguous() if sink else None
    scale = 1.0 / math.sqrt(hd)
    outs, mags, spans, at = [], [], [], 0
    for (k, v), n, b in zip(kv, new, before):
        kh, vh = Q.q4(k, 32), Q.q4(v, 32)
        outs.append(Q.attention(q[at:at + n], kh, vh, b, scale, window, sinks))
        mags.append(Q.attention(q[at:at + n], kh, vh.abs(), b, scale, window, sinks))
        span = v.double().reshape(*v.shape[:2], -1, 32)              # 15 s of every group: its range and up to an eighth more
        span = 1.125 * (span.amax(-1).clamp(min=0) - span.amin(-1).clamp(max=0)).repeat_interleave(32, -1)
        spans.append((b + n) * Q.attention(q[at:at + n], kh, span, b, scale, window, sinks))
        at += n
    return meta, kv, q, sinks, *(torch.cat(x).reshape(sum(new), -1) for x in (outs, mags, spans))


def run_attention(meta, pool, q, nh, nkv, hd, window, sinks, new, before):
    from types import SimpleNamespace

    from spissa_b200.cache.views import KVLayerView
    from spissa_b200.parts.attention import attend_paged
    B = len(new)
    step = SimpleNamespace(n_seqs=B, seq_len=meta.seq_len, seq_start=meta.seq_start, max_new=max(new), max_len=max(meta.total_len),
                           all_single=all(n == 1 for n in new), host=dict(new_counts=list(new), seq_len=list(meta.total_len)))
    view = KVLayerView(pool, pool, meta.page_table, 64, meta.token_seq, meta.positions, meta.seq_slot, window, True, bits=4)
    return attend_paged(q.to(DEV).reshape(sum(new), -1), step, view, nh, nkv, hd, window, 1.0 / math.sqrt(hd),
                        sinks.to(DEV) if sinks is not None else None)


CASES = [([1], [0]), ([1], [63]), ([1, 1, 1], [64, 0, 700]), ([1], [2500]), ([2, 1, 9], [5, 130, 60]), ([40], [300]), ([300, 3], [0, 200])]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(case, nh, nkv, hd, dtype):
    new, before = CASES[case]
    for window, sink in ((None, False), (70, True)):
        meta, kv, q, sinks, want, mag, span = attention_case(nh, nkv, hd, dtype, new, before, window, 10 * case + hd, sink)
        pool = fill(meta, kv, nkv, hd)
        out = run_attention(meta, pool, q, nh, nkv, hd, window, sinks, new, before)
        assert out.dtype == dtype and out.shape == want.shape
        # scores: sums of hd products and a scale, off by (hd + 8) 2^-23 of their terms' sizes, which are below 64 here, so each
        # probability by that (e^x − 1 is near x); bfloat16: probabilities and outputs rounded on top, 2^-8 each. A value enters as
        # p s c − p s z: two sums over the n keys of terms up to 15 s p, whose partial sums are cut to 24 bits at every step, so
        # that each is off by at most n 2^-23 Σ 15 s p, also where c = z leaves nothing of the value itself (``span``: n Σ 15 s p)
        eps = (hd + 8) * 2.0 ** -23 * 64
        tol = 2 * eps * mag + 2 * 2.0 ** -23 * span + (2.0 ** -8 * mag + 2.0 ** -8 * want.abs() if dtype == BF else 0)
        assert bool(((out.cpu().double() - want).abs() <= tol).all()), float(((out.cpu().double() - want).abs() / tol).max())
        assert torch.equal(out, run_attention(meta, pool, q, nh, nkv, hd, window, sinks, new, before))
