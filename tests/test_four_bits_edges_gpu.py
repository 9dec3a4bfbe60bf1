"""Weights and caches of four bits where they can go wrong: every way of a product at the borders of its sizes, chunks longer
than a ring, numbers that are not finite in masked places, pools beyond 2^32 bytes, rows behind the last sequence, other
streams, captured graphs that share no state. Tolerances as in test_four_bits_gpu.py, which states them."""
import math
from types import SimpleNamespace

import pytest
import torch

import kernel_harness as KH
from plain import q4_plain as Q
from test_four_bits_gpu import DEV, attention_case, fill, numbers, product_case, run_attention

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


# ------------------------------------------------------------------------------------------------------------- products
def product_tolerance(K, mag):
    return (K * 2.0 ** -23 + 2.0 ** -22) * mag


@pytest.mark.parametrize("M,N,K,group", [(1, 16, 32, 32), (9, 130, 160, 32), (16, 256, 128, 128), (17, 17, 96, 32), (128, 1100, 256, 64), (129, 144, 4224, 64),
                                         (160, 4096, 320, 64), (255, 40, 2048, 128), (256, 2320, 512, 128), (257, 300, 384, 64), (513, 64, 8192, 32),
                                         (1000, 528, 128, 64), (1024, 128, 1024, 128)])
def test_products_on_the_codes_as_they_lie(M, N, K, group):
    """The tcgen05 kernel itself, over its range of rows: one piece of K and several, one CTA of an SM and two, odd rings."""
    from spissa_b200.csrc import lib
    x, w, y, mag = product_case(M, N, K, group, BF, M + N)
    codes, scales = lib.q4_pack(w.to(DEV), group)
    tol = product_tolerance(K, mag)
    wide = torch.full((M, N + 7), 3.0, device=DEV)
    lib.q4_tc(x.to(DEV), codes, scales, wide[:, 2:2 + N], N, group)
    assert bool(((wide[:, 2:2 + N].cpu().double() - y).abs() <= tol).all())
    assert bool((wide[:, :2] == 3).all()) and bool((wide[:, 2 + N:] == 3).all())
    again = torch.empty(M, N, device=DEV)
    lib.q4_tc(x.to(DEV), codes, scales, again, N, group)
    assert torch.equal(again, wide[:, 2:2 + N])
    lib.q4_tc(x.to(DEV), codes, scales, again, N, group, 0, lib.TC_ACCUMULATE)
    assert bool(((again.cpu().double() - 2 * y).abs() <= 2 * tol + 2.0 ** -22 * (y.abs() + tol)).all())
    lib.check_status(DEV)


@pytest.mark.parametrize("N,K", [(28672, 512), (20000, 256), (18960, 1024)])
def test_products_of_more_rows_of_weight_than_an_sm_each(N, K):
    from spissa_b200.parts.linear import Linear4
    for M in (17, 96, 130):
        x, w, y, mag = product_case(M, N, K, 64, BF, M)
        out = Linear4(w.to(DEV), 64)(x.to(DEV), out_dtype=F32)
        assert bool(((out.cpu().double() - y).abs() <= product_tolerance(K, mag)).all())


def test_the_ways_of_a_product_agree_at_their_borders(monkeypatch):
    """The same rows of x give what the definition gives whichever way the number of rows and the sizes choose."""
    from spissa_b200.parts import linear as L
    x, w, y, mag = product_case(260, 384, 512, 64, BF, 5)
    wg = torch.cat([w, w.flip(0)])
    gated, lin, tol = L.GatedLinear4(wg[:384].to(DEV), wg[384:].to(DEV)), L.Linear4(w.to(DEV)), product_tolerance(512, mag)
    seen = set()
    kept = L.product4
    monkeypatch.setattr(L, "product4", lambda *a: seen.add(kept(*a)) or kept(*a))
    for M in (1, 8, 9, 16, 17, 255, 256, 257, 260):
        out = lin(x[:M].to(DEV), out_dtype=F32)
        assert bool(((out.cpu().double() - y[:M]).abs() <= tol[:M]).all())
    for way in ("gemv", "tc", "unpack"):
        monkeypatch.setattr(L, "product4", lambda *a: way)
        one, two = lin(x[:16].to(DEV), out_dtype=F32), gated(x[:16].to(DEV), F32)
        assert bool(((one.cpu().double() - y[:16]).abs() <= tol[:16]).all())
        g, u = y[:16], x[:16].double() @ Q.q4(w.flip(0), 64).T
        want = g * torch.sigmoid(g) * u
        # off by the products' tolerance through the activation (slope up to 1.2); the unpacked way rounds gate and up to float32
        e = tol[:16] + 2.0 ** -23 * (g.abs() + u.abs())
        e = 1.2 * e * (u.abs() + e) + g.abs() * (x[:16].double().abs() @ Q.q4(w.flip(0), 64).abs().T) * (512 * 2.0 ** -23 + 2.0 ** -22)
        assert bool(((two.cpu().double() - want).abs() <= e + 2.0 ** -20 * want.abs() + 2.0 ** -22 * u.abs()).all()), way
    assert {"gemv", "tc"} <= seen


@pytest.mark.parametrize("M", [3, 16, 40, 300])
def test_numbers_that_are_not_finite_stay_in_their_row_and_column(M):
    from spissa_b200.parts.linear import Linear4
    x, w, y, mag = product_case(M, 200, 256, 64, BF, 9)
    clean = torch.ones(M, 200, dtype=torch.bool)
    x[1, 70] = float("nan")
    x[2, 5] = float("inf")
    w[17, 100] = float("nan")
    w[150, 3] = float("-inf")
    clean[1:3], clean[:, 17], clean[:, 150] = False, False, False
    out = Linear4(w.to(DEV), 64)(x.to(DEV), out_dtype=F32).cpu().double()
    assert bool(((out - y).abs() <= product_tolerance(256, mag))[clean].all())
    assert bool(out[:, 17].isnan().all()) and bool(out[:, 150].isnan().all()) and bool((~out[1].isfinite()).all())
    assert bool((~out[2].isfinite()).any())


def test_rows_that_overlap_and_rows_of_nothing():
    from spissa_b200.parts.linear import Linear4
    w = numbers(48, 128, seed=2, dtype=BF)
    lin, row = Linear4(w.to(DEV), 32), numbers(1, 128, seed=3, spread=0.5, dtype=BF)
    for M in (1, 5, 40):
        out = lin(row.to(DEV).expand(M, 128), out_dtype=F32)
        assert torch.equal(out, lin(row.to(DEV).repeat(M, 1), out_dtype=F32))
        zero = lin(torch.zeros(M, 128, dtype=BF, device=DEV), out_dtype=F32)
        assert bool((zero == 0).all())


def test_an_outputs_rows_that_overlap_are_refused():
    from spissa_b200.csrc.lib import KernelError
    from spissa_b200.parts.linear import Linear4
    lin = Linear4(numbers(48, 128, seed=2, dtype=BF).to(DEV), 32)
    for M in (2, 20):
        with pytest.raises(KernelError):
            lin(torch.zeros(M, 128, dtype=BF, device=DEV), out=torch.zeros(1, 48, device=DEV).expand(M, 48))


def test_products_on_another_stream_and_in_graphs():
    from spissa_b200.parts.linear import GatedLinear4, Linear4
    w = numbers(512, 1024, seed=4, spread=0.5, dtype=BF).to(DEV)
    lin, gated = Linear4(w, 64), GatedLinear4(w, w.flip(0))
    for M in (1, 12, 33, 300, 1030):
        xs = [numbers(M, 1024, seed=s, spread=0.3, dtype=BF).to(DEV) for s in (1, 2)]
        want = [(lin(x), gated(x, BF)) for x in xs]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = lin(xs[0]), gated(xs[0], BF)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(other, want[0]))
        places, graphs, outs = [x.clone() for x in xs], [], []
        for x in places:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append((lin(x), gated(x, BF)))
            graphs.append(g)
        places[0].copy_(xs[1])
        places[1].copy_(xs[0])
        for _ in range(2):
            for g in graphs:
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for i in (0, 1) for a, b in zip(outs[i], want[1 - i]))


# ------------------------------------------------------------------------------------------------------------ attention
def attention_tolerance(hd, dtype, want, mag, span):
    eps = (hd + 8) * 2.0 ** -23 * 64
    return 2 * eps * mag + 2 * 2.0 ** -23 * span + (2.0 ** -8 * mag + 2.0 ** -8 * want.abs() if dtype == BF else 0)


def attend(meta, pool, q, nh, nkv, hd, new, window, sinks, plan, out=None):
    from spissa_b200.csrc import lib
    q = q.to(DEV).reshape(q.shape[0], -1).contiguous()
    out = torch.empty_like(q) if out is None else out
    single = all(n == 1 for n in new)
    lib.kv4_attend(q, pool, out, meta, None if single else meta.seq_start, len(new), max(new), max(meta.total_len), nh, nkv, hd, window,
                   1.0 / math.sqrt(hd), sinks.to(DEV) if sinks is not None else None, plan)
    return out


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 128), (6, 2, 64)])
@pytest.mark.parametrize("plan", [(1, 64, 1), (2, 64, 1), (1, 5, 12), (1, 33, 2), (2, 40, 2), (1, 1, 60)])
def test_chunks_of_any_length(plan, nh, nkv, hd, dtype):
    """Chunks longer than the ring of pages (4) and than the page numbers a warp holds (32), and of a single page."""
    new, before = [1, 3, 1], [3790, 2400, 10]
    for window in (None, 2100):
        meta, kv, q, sinks, want, mag, span = attention_case(nh, nkv, hd, dtype, new, before, window, hd + plan[1], window is not None)
        pool = fill(meta, kv, nkv, hd)
        out = attend(meta, pool, q, nh, nkv, hd, new, window, sinks, plan)
        tol = attention_tolerance(hd, dtype, want, mag, span)
        assert bool(((out.cpu().double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new,before", [([1, 1], [100, 130]), ([6], [100]), ([20, 2], [90, 127])])
def test_keys_and_values_that_are_not_finite_reach_only_who_sees_them(new, before, dtype):
    """A NaN key, an infinite value: later queries become NaN in the heads of that kv head, the others stay as they are; behind a
    window and in later tokens they may stand."""
    nh, nkv, hd, window = 6, 2, 64, 60
    meta, kv, q, _, want, mag, span = attention_case(nh, nkv, hd, dtype, new, before, window, 21)
    tol = attention_tolerance(hd, dtype, want, mag, span)
    where = [before[0] + new[0] - 1, max(0, before[0] - window - 5)]               # the first sequence's newest token; one that nobody's window reaches
    for b, pos in ((0, where[0]), (0, where[1])):
        kv[b][0][pos, 0, 3] = float("nan")
        kv[b][1][pos, 0, 40] = float("inf")
    pool = fill(meta, kv, nkv, hd)
    out = run_attention(meta, pool, q, nh, nkv, hd, window, None, new, before).cpu().double().view(-1, nh, hd)
    seen = torch.zeros(sum(new), nh, hd, dtype=torch.bool)
    seen[new[0] - 1, :3] = True                                                     # the newest token's own query, the first kv head's three heads
    assert bool(((out - want.view(-1, nh, hd)).abs() <= tol.view(-1, nh, hd))[~seen].all())
    assert bool(out[seen].isnan().all())


def test_a_value_that_is_not_finite_spoils_its_group_of_columns_only():
    nh, nkv, hd = 4, 2, 128
    meta, kv, q, _, want, mag, span = attention_case(nh, nkv, hd, BF, [1], [70], None, 22)
    kv[0][1][30, 1, 70] = float("nan")
    out = run_attention(meta, fill(meta, kv, nkv, hd), q, nh, nkv, hd, None, None, [1], [70]).cpu().double().view(nh, hd)
    bad = torch.zeros(nh, hd, dtype=torch.bool)
    bad[2:, 64:96] = True
    assert bool(out[bad].isnan().all())
    assert bool(((out - want.view(nh, hd)).abs() <= attention_tolerance(hd, BF, want, mag, span).view(nh, hd))[~bad].all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_prompts_behind_a_window_meet_no_memory_that_was_left_alone(dtype):
    """The prompt path unpacks the pages that a window reaches; whatever the memory of the others held is not seen."""
    nh, nkv, hd, new, before, window = 16, 1, 64, [70, 33, 300], [700, 1023, 5], 100
    meta, kv, q, _, want, mag, span = attention_case(nh, nkv, hd, dtype, new, before, window, 31)
    pool = fill(meta, kv, nkv, hd)
    tol = attention_tolerance(hd, dtype, want, mag, span)
    for bits in (0xff, 0x7f):                                                       # NaN as float32 and bfloat16; large numbers
        spoiled = [torch.full((1 << 20,), bits, dtype=torch.uint8, device=DEV) for _ in range(64)]
        del spoiled
        out = run_attention(meta, pool, q, nh, nkv, hd, window, None, new, before)
        # (keys and values are exact in the queries' type; the bfloat16 kernels round probabilities once, as counted)
        assert bool(((out.cpu().double() - want).abs() <= 2 * tol).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("window", [1, 2, 64, 65, 128])
def test_windows_at_the_borders_of_pages(window, dtype):
    nh, nkv, hd = 6, 2, 64
    for new, before in (([1, 1, 1], [63, 64, 191]), ([5, 1, 40], [60, 0, 100]), ([280], [70])):
        meta, kv, q, sinks, want, mag, span = attention_case(nh, nkv, hd, dtype, new, before, window, 70 + window, window == 64)
        out = run_attention(meta, fill(meta, kv, nkv, hd), q, nh, nkv, hd, window, sinks, new, before)
        assert bool(((out.cpu().double() - want).abs() <= attention_tolerance(hd, dtype, want, mag, span)).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 128), (9, 3, 96), (4, 2, 32), (16, 2, 64)])
def test_prompts_on_the_codes_and_unpacked_first_agree(nh, nkv, hd, dtype, monkeypatch):
    """Whichever way a step would take by its sizes, both give what the definition gives."""
    from spissa_b200.parts import attention as A
    for new, before in (([70, 1, 30], [10, 500, 0]), ([300], [65])):
        meta, kv, q, sinks, want, mag, span = attention_case(nh, nkv, hd, dtype, new, before, None, 80 + hd, True)
        pool = fill(meta, kv, nkv, hd)
        for codes in (True, False):
            monkeypatch.setattr(A, "reads_codes", lambda *a: codes)
            out = run_attention(meta, pool, q, nh, nkv, hd, None, sinks, new, before)
            assert bool(((out.cpu().double() - want).abs() <= attention_tolerance(hd, dtype, want, mag, span)).all()), codes


def test_the_way_of_a_prompt_step():
    from spissa_b200.parts.attention import reads_codes
    q = torch.empty(255, 8, dtype=BF, device=DEV)
    assert reads_codes(q, 1020, 8) and not reads_codes(q.new_empty(256, 8), 1024, 8) and reads_codes(q.new_empty(1024, 8), 256, 8)
    assert reads_codes(q.float(), 1 << 16, 8) and not reads_codes(q.float(), 1 << 18, 8)


def test_a_pool_beyond_four_gigabytes():
    from spissa_b200.csrc import lib
    nh, nkv, hd, new, before = 8, 8, 128, [1, 2], [200, 65]
    page_bytes = nkv * lib.kv4_tile_bytes(hd)
    meta, kv, q, _, want, mag, span = attention_case(nh, nkv, hd, BF, new, before, None, 41)
    n_pages = (1 << 32) // page_bytes + 64
    meta.page_table += n_pages - meta.n_pages
    meta.rows = [[p + n_pages - meta.n_pages for p in r] for r in meta.rows]
    meta.n_pages = n_pages
    assert int(meta.page_table.min()) * page_bytes > 1 << 32
    pool = fill(meta, kv, nkv, hd, poison=False)
    out = attend(meta, pool, q, nh, nkv, hd, new, None, None, None)
    assert bool(((out.cpu().double() - want).abs() <= attention_tolerance(hd, BF, want, mag, span)).all())
    k, v = (torch.empty(3, nkv, hd, dtype=F32, device=DEV) for _ in range(2))
    lib.kv4_load(pool, meta, k, v, nkv, hd)
    rows = torch.cat([kv[0][0][200:], kv[1][0][65:]])
    assert torch.equal(k.cpu().double(), Q.q4(rows, 32))
    assert not bool(pool[:1000].any())                                              # (a page number cut to 32 bits of offset would have written here)


@pytest.mark.parametrize("plan", [(1, 4, 1), (1, 1, 4), (2, 2, 2)])
def test_rows_behind_the_last_sequence_stay_and_a_sequence_may_bring_nothing(plan):
    nh, nkv, hd, new, before = 4, 2, 64, [2, 0, 3], [100, 50, 7]
    meta, kv, q, _, want, mag, span = attention_case(nh, nkv, hd, BF, new, before, None, 51)
    pool = fill(meta, kv, nkv, hd)
    padded = torch.cat([q, torch.full((4, nh, hd), float("nan"), dtype=BF)])
    meta.token_seq, meta.positions = (torch.cat([t, t.new_zeros(4)]) for t in (meta.token_seq, meta.positions))
    out = torch.full((9, nh * hd), 7.0, dtype=BF, device=DEV)
    attend(meta, pool, padded, nh, nkv, hd, new, None, None, plan, out)
    assert bool(((out[:5].cpu().double() - want).abs() <= attention_tolerance(hd, BF, want, mag, span)).all())
    assert bool((out[5:] == 7).all())


def test_no_rows_at_all():
    from spissa_b200.csrc import lib
    meta = KH.paged_meta([1], [0], DEV)
    pool = lib.kv4_pool(2, 2, 64, DEV)
    meta.token_seq, meta.positions = meta.token_seq[:0], meta.positions[:0]
    lib.kv4_store(torch.empty(0, 8 * 64, device=DEV), torch.empty(0, 4 * 64, dtype=BF, device=DEV), pool, meta, None, 4, 2, 64, 0)
    lib.kv4_load(pool, meta, torch.empty(0, 2, 64, device=DEV), torch.empty(0, 2, 64, device=DEV), 2, 64)
    q = torch.empty(0, 4 * 64, dtype=BF, device=DEV)
    lib.kv4_attend(q, pool, q.clone(), meta, meta.seq_start, 0, 1, 1, 4, 2, 64, None, 0.125)
    assert not bool(pool.any())


def test_attention_on_another_stream_and_in_graphs():
    """Two graphs captured one after the other, replayed in turns, and a longer step than the captured one's positions."""
    from spissa_b200.csrc import lib
    nh, nkv, hd = 8, 2, 64
    cases = []
    for seed, before in ((61, [1500, 3]), (62, [640, 1999])):
        meta, kv, q, _, want, mag, span = attention_case(nh, nkv, hd, BF, [1, 1], before, None, seed)
        meta.total_len = [2048, 2048]                                               # the split is made for a bucket of lengths
        cases.append((meta, fill_all(kv, meta, nkv, hd, before), q.reshape(2, -1).to(DEV), want, attention_tolerance(hd, BF, want, mag, span)))
    eager = [attend(m, p, q, nh, nkv, hd, [1, 1], None, None, None) for m, p, q, _, _ in cases]
    for out, (_, _, _, want, tol) in zip(eager, cases):
        assert bool(((out.cpu().double() - want).abs() <= tol).all())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [attend(m, p, q, nh, nkv, hd, [1, 1], None, None, None) for m, p, q, _, _ in cases]
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for m, p, q, _, _ in cases:
        outs.append(torch.zeros_like(q))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            attend(m, p, q, nh, nkv, hd, [1, 1], None, None, None, outs[-1])
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(eager, other, outs):
        assert torch.equal(a, b) and torch.equal(a, c)


def fill_all(kv, meta, nkv, hd, before):
    real = SimpleNamespace(**vars(meta))
    real.total_len = [b + 1 for b in before]
    return fill(real, kv, nkv, hd)


# ------------------------------------------------------------------------------------------------------------- refusals
def test_refusals_of_the_cache():
    from spissa_b200.csrc import lib
    from spissa_b200.csrc.lib import KernelError
    nh, nkv, hd = 4, 2, 64
    meta = KH.paged_meta([1, 2], [5, 70], DEV)
    pool = lib.kv4_pool(meta.n_pages, nkv, hd, DEV)
    qkv, q = torch.zeros(3, 8 * hd, device=DEV), torch.zeros(3, nh * hd, dtype=BF, device=DEV)
    freq = torch.ones(32, device=DEV)

    def other(**changed):
        return SimpleNamespace(**{**vars(meta), **changed})

    def store(qkv=qkv, q=q, pool=pool, meta=meta, freq=freq, nh=nh, nkv=nkv, hd=hd, rd=64):
        lib.kv4_store(qkv, q, pool, meta, freq, nh, nkv, hd, rd)

    def load(k=None, v=None, pool=pool, meta=meta, nkv=nkv, hd=hd):
        lib.kv4_load(pool, meta, torch.zeros(3, 2, 64, device=DEV) if k is None else k, torch.zeros(3, 2, 64, device=DEV) if v is None else v, nkv, hd)

    def attention(q=q, pool=pool, out=None, meta=meta, start=meta.seq_start, n=2, new=2, nh=nh, nkv=nkv, hd=hd, window=None, scale=0.125, sink=None, plan=None):
        lib.kv4_attend(q, pool, torch.zeros_like(q) if out is None else out, meta, start, n, new, 72, nh, nkv, hd, window, scale, sink, plan)

    def unpack(k=None, v=None, table=None, step=None):
        k = torch.zeros(3, nkv, 64, hd, device=DEV) if k is None else k
        step = step or SimpleNamespace(seq_len=meta.seq_len, seq_start=meta.seq_start, n_seqs=2)
        lib.kv4_unpack_pages(pool, meta, k, torch.zeros_like(k) if v is None else v, torch.zeros_like(meta.page_table) if table is None else table, step, None, nkv, hd)

    for fine in (store, load, attention, unpack):
        fine()
    wide = other(page_table=meta.page_table.long())
    bad = [lambda: store(qkv=qkv.to(BF)), lambda: store(qkv=qkv[:, :-1]), lambda: store(qkv=qkv.cpu()), lambda: store(q=None), lambda: store(q=q[:2]),
           lambda: store(q=q.half()), lambda: store(pool=pool.to(torch.int8)), lambda: store(pool=pool[:, :1]), lambda: store(pool=pool[:, :, :-1]),
           lambda: store(meta=wide), lambda: store(meta=other(page_size=32)), lambda: store(meta=other(positions=meta.positions[:2])),
           lambda: store(meta=other(page_table=meta.page_table.cpu())), lambda: store(freq=None), lambda: store(freq=freq[:16]), lambda: store(freq=freq.double()),
           lambda: store(rd=36), lambda: store(rd=72), lambda: store(qkv=torch.zeros(3, 16 * hd, device=DEV)[:, ::2]),
           lambda: load(k=torch.zeros(3, 2, 32, device=DEV)), lambda: load(v=torch.zeros(3, 2, 64, device=DEV, dtype=BF)), lambda: load(k=torch.zeros(3, 2, 64)),
           lambda: load(k=torch.zeros(3, 2, 64, device=DEV, dtype=torch.float16), v=torch.zeros(3, 2, 64, device=DEV, dtype=torch.float16)),
           lambda: load(k=torch.zeros(5, 2, 64, device=DEV), v=torch.zeros(5, 2, 64, device=DEV)), lambda: load(meta=wide),
           lambda: attention(q=q.half()), lambda: attention(out=torch.zeros_like(q, dtype=F32)), lambda: attention(out=torch.zeros_like(q)[:2]),
           lambda: attention(nh=3), lambda: attention(window=-1), lambda: attention(scale=0.0), lambda: attention(scale=-1.0), lambda: attention(scale=math.nan),
           lambda: attention(sink=torch.zeros(3, device=DEV)), lambda: attention(sink=torch.zeros(4, device=DEV, dtype=BF)), lambda: attention(start=meta.seq_start[:2]),
           lambda: attention(start=meta.seq_start.long()), lambda: attention(start=None), lambda: attention(new=0), lambda: attention(plan=(3, 2, 1)),
           lambda: attention(plan=(1, 0, 1)), lambda: attention(plan=(1, 2, 0)), lambda: attention(meta=wide), lambda: attention(pool=pool.cpu()),
           lambda: unpack(k=torch.zeros(3, nkv, 32, hd, device=DEV)), lambda: unpack(table=meta.page_table.long()), lambda: unpack(table=meta.page_table[:, :1]),
           lambda: unpack(step=SimpleNamespace(seq_len=meta.seq_len.long(), seq_start=meta.seq_start, n_seqs=2)),
           lambda: unpack(step=SimpleNamespace(seq_len=meta.seq_len, seq_start=meta.seq_start[:2], n_seqs=2)),
           lambda: unpack(step=SimpleNamespace(seq_len=meta.seq_len, seq_start=meta.seq_start, n_seqs=3)),
           lambda: lib.kv4_pool(2, 2, 80, DEV), lambda: lib.kv4_pool(2, 2, 160, DEV)]
    for i, call in enumerate(bad):
        with pytest.raises(KernelError):
            call()
            pytest.fail(f"call {i} of the list was taken")
    lib.check_status(DEV)


def test_refusals_of_the_products_entry():
    from spissa_b200.csrc import lib
    from spissa_b200.csrc.lib import KernelError
    codes, scales = lib.q4_pack(numbers(64, 128, seed=1).to(DEV), 32)
    x, out = torch.zeros(4, 128, dtype=BF, device=DEV), torch.zeros(4, 64, device=DEV)
    lib.q4_tc(x, codes, scales, out, 64, 32)
    for bad in (lambda: lib.q4_tc(torch.zeros(1025, 128, dtype=BF, device=DEV), codes, scales, out, 64, 32), lambda: lib.q4_tc(x[:0], codes, scales, out, 64, 32),
                lambda: lib.q4_tc(x, codes, scales, out, 64, 48), lambda: lib.q4_tc(x, codes, scales, out, 64, 32, 32, lib.TC_STORE),
                lambda: lib.q4_tc(x, codes, scales, out, 64, 32, 0, lib.TC_SILU_MUL), lambda: lib.q4_tc(x, codes, scales, out.to(BF), 64, 32, 0, lib.TC_ACCUMULATE),
                lambda: lib.q4_gemv(torch.zeros(17, 128, dtype=BF, device=DEV), codes, scales, out, 64, 32),
                lambda: lib.q4_unpack(codes, scales, torch.zeros(64, 160, device=DEV), 32), lambda: lib.q4_unpack(codes, scales, torch.zeros(128, 64, device=DEV).T, 32)):
        with pytest.raises(KernelError):
            bad()
