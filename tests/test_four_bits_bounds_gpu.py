"""Attention over four bits within the bound of plain/q4_attention_bounds.py, which counts every rounding: float32 against what a
single float16 part would be off by, groups of columns and keys of very unlike sizes, values that are zeros."""
import math

import pytest
import torch

import kernel_harness as KH
from plain import q4_attention_bounds as B
from plain import q4_plain as Q
from test_four_bits_bounds import aligned_case
from test_four_bits_edges_gpu import attend
from test_four_bits_gpu import CASES, DEV, HEADS, fill, numbers, run_attention

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def expected(q, kv, new, before, scale, window=None, sinks=None):
    """(want, tolerance) [tokens, nh · hd] of sequences with keys and values ``kv``."""
    parts, at = [], 0
    for (k, v), n, b in zip(kv, new, before):
        parts.append(B.rows(q[at:at + n], Q.q4(k, 32), Q.q4(v, 32), B.scales(v), b, scale, window, sinks))
        at += n
    return tuple(torch.cat(x).reshape(at, -1) for x in zip(*parts))


def holds(out, want, tol, note=""):
    off = (out.cpu().double() - want).abs()
    bad = ~(off <= tol)
    assert not bool(bad.any()), (note, int(bad.sum()), float((off / tol.clamp(min=1e-300)).nan_to_num(math.inf).max()))


@pytest.mark.parametrize("kind", ["q", "p"])
@pytest.mark.parametrize("hd", [64, 128])
def test_float32_needs_both_parts(kind, hd):
    """The cases whose bound a single float16 part of the queries, or of p s, would exceed."""
    q, k, v = aligned_case(kind, hd)
    n = k.shape[0]
    for G in (1, 5):                                                 # eight columns a CTA, whatever is in them
        qs = q.expand(1, G, hd).contiguous()
        want, tol = expected(qs, [(k, v)], [1], [n - 1], 1.0 / math.sqrt(hd))
        meta = KH.paged_meta([1], [n - 1], DEV)
        holds(run_attention(meta, fill(meta, [(k, v)], 1, hd), qs, G, 1, hd, None, None, [1], [n - 1]), want, tol)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
@pytest.mark.parametrize("case", range(len(CASES) - 1))
def test_attention_within_its_bound(case, nh, nkv, hd, dtype):
    new, before = CASES[case]
    for window, sink in ((None, False), (70, True)):
        meta, seed = KH.paged_meta(new, before, DEV, seed=10 * case + hd), 10 * case + hd
        kv = [tuple(numbers(n, nkv, hd, seed=seed + 3 * b + i, spread=0.3) for i in (0, 1)) for b, n in enumerate(meta.total_len)]
        q = numbers(sum(new), nh, hd, seed=seed + 99, spread=0.2, dtype=dtype)
        sinks = numbers(1, nh, seed=seed + 7, spread=0.1)[0].contiguous() if sink else None
        want, tol = expected(q, kv, new, before, 1.0 / math.sqrt(hd), window, sinks)
        holds(run_attention(meta, fill(meta, kv, nkv, hd), q, nh, nkv, hd, window, sinks, new, before), want, tol, (window, sink))


def unlike_case(kind, n, nh, nkv, hd, dtype, seed):
    """Values whose groups of 32 columns, or keys, differ by powers of two. Every query scores key 3 higher by ``lift`` than the others."""
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn(1, nh, hd, generator=gen) * 0.3
    q[..., 0] = 4.0
    k, v = torch.randn(n, nkv, hd, generator=gen) * 0.3, torch.randn(n, nkv, hd, generator=gen)
    k[:, :, 0] = 0.0
    lift, top = {"groups": (0.0, 0), "sink": (14 * math.log(2), 10), "far sink": (8 * math.log(2), 20), "lost": (14 * math.log(2), 20),
                 "outlier": (-30 * math.log(2), 0)}[kind]
    if kind == "groups":
        v *= torch.exp2(-10.0 * torch.arange(hd // 32)).repeat_interleave(32)
    elif kind == "outlier":                                          # one key of large values that hardly counts
        v[3] *= 2.0 ** 24
    else:                                                            # a key that takes most of the weight and has no value but in the first group,
        v[:, :, 32:] *= 2.0 ** -top                                  # the others' second group small
        v[3, :, 32:] = 0.0
    k[3, :, 0] = lift * math.sqrt(hd) / 4.0
    return q.to(dtype), k, v


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kind", ["groups", "sink", "far sink", "lost", "outlier"])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 128), (8, 2, 64), (3, 1, 96)])
def test_groups_and_keys_of_unlike_sizes(nh, nkv, hd, kind, dtype):
    """A group of columns keeps its precision whatever the other groups hold, and a key's size counts by its weight."""
    n = 900
    q, k, v = unlike_case(kind, n, nh, nkv, hd, dtype, hd + n)
    want, tol = expected(q, [(k, v)], [1], [n - 1], 1.0 / math.sqrt(hd))
    meta = KH.paged_meta([1], [n - 1], DEV)
    pool = fill(meta, [(k, v)], nkv, hd)
    for plan in (None, (1, 15, 1), (2, 15, 1), (2, 4, 4)):
        holds(attend(meta, pool, q, nh, nkv, hd, [1], None, None, plan), want, tol, plan)


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


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hd", [64, 128])
def test_a_keys_large_entry_that_a_query_does_not_see_leaves_its_score_alone(hd, dtype):
    """One channel of the keys is large and the queries are zero there; the others of its group stand for zeros, so every key's score comes
    from the other groups."""
    n, nh, nkv = 500, 4, 2
    gen = torch.Generator().manual_seed(hd + 1)
    q, k, v = (torch.randn(s, h, hd, generator=gen) for s, h in ((1, nh), (n, nkv), (n, nkv)))
    k[..., 5] = 2.0 ** 17 * (1 + torch.rand(n, nkv, generator=gen))
    k[..., 9] = -2.0 ** 16 * (1 + torch.rand(n, nkv, generator=gen))
    q[..., 5] = q[..., 9] = 0.0
    q = q.to(dtype)
    want, tol = expected(q, [(k, v)], [1], [n - 1], 1.0 / math.sqrt(hd))
    meta = KH.paged_meta([1], [n - 1], DEV)
    pool = fill(meta, [(k, v)], nkv, hd)
    for plan in (None, (1, 8, 1), (2, 8, 1)):
        holds(attend(meta, pool, q, nh, nkv, hd, [1], None, None, plan), want, tol, plan)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_value_that_is_not_finite_counts_however_little_its_weight(dtype):
    """Zero times NaN is NaN: a key of vanishing weight, in a chunk, a warp and a page of its own or among others."""
    n, nh, nkv, hd = 400, 4, 2, 64
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(s, h, hd, generator=gen) for s, h in ((1, nh), (n, nkv), (n, nkv)))
    q[..., 0], k[:, :, 0], k[0:64, :, 0] = 8.0, 0.0, -300.0          # the first page's scores are 300 below the others'
    v[5, 0, 40] = float("inf")
    q = q.to(dtype)
    meta = KH.paged_meta([1], [n - 1], DEV)
    pool = fill(meta, [(k, v)], nkv, hd)
    for plan in (None, (1, 7, 1), (1, 1, 7), (2, 3, 3)):
        out = attend(meta, pool, q, nh, nkv, hd, [1], None, None, plan).view(nh, hd).cpu()
        assert bool(out[:2, 32:].isnan().all()) and bool(out[:2, :32].isfinite().all()) and bool(out[2:].isfinite().all()), plan


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_sequence_longer_than_its_split_keeps_its_newest_keys(dtype):
    """``longest`` shapes the split; a sequence that has more keys than it says is read to its end."""
    from spissa_b200.csrc import lib
    n, nh, nkv, hd = 700, 4, 2, 64
    gen = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(s, h, hd, generator=gen) for s, h in ((1, nh), (n, nkv), (n, nkv)))
    q = q.to(dtype)
    want, tol = expected(q, [(k, v)], [1], [n - 1], 1.0 / math.sqrt(hd))
    meta = KH.paged_meta([1], [n - 1], DEV)
    pool, rows = fill(meta, [(k, v)], nkv, hd), q.to(DEV).reshape(1, -1)
    for longest in (1, 64, 300, 699):
        for window in (None, 650):
            out = torch.empty_like(rows)
            lib.kv4_attend(rows, pool, out, meta, None, 1, 1, longest, nh, nkv, hd, window, 1.0 / math.sqrt(hd))
            if window is None:
                holds(out, want, tol, longest)
            else:
                holds(out, *expected(q, [(k, v)], [1], [n - 1], 1.0 / math.sqrt(hd), window), (longest, window))


def test_what_a_split_and_the_rows_of_the_table_have_to_cover():
    from types import SimpleNamespace

    from spissa_b200.csrc import lib
    nh, nkv, hd = 4, 2, 64
    meta = KH.paged_meta([1, 1], [300, 20], DEV)
    pool, q = lib.kv4_pool(meta.n_pages, nkv, hd, DEV), torch.zeros(2, nh * hd, dtype=BF, device=DEV)

    def call(meta=meta, window=None, plan=None):
        lib.kv4_attend(q, pool, torch.empty_like(q), meta, None, 2, 1, 301, nh, nkv, hd, window, 0.125, None, plan)
    for plan in (None, (1, 5, 1), (2, 1, 5), (1, 2, 3)):
        call(plan=plan)
    call(window=60, plan=(1, 1, 2))
    for bad in (lambda: call(plan=(1, 4, 1)), lambda: call(plan=(1, 1, 4)), lambda: call(plan=(2, 2, 2)), lambda: call(window=60, plan=(1, 1, 1)),
                lambda: call(meta=SimpleNamespace(**{**vars(meta), "seq_slot": meta.seq_slot[:1]}))):
        with pytest.raises(lib.KernelError):
            bad()
    lib.check_status(DEV)
