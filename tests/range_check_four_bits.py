"""Run with SPISSA_B200_RANGE_CHECK=1 (tests/test_four_bits_range_check_gpu.py does): the kernels of the four-bit cache report a
page, a row or a position beyond what the host DECLARED and leave the access out. Pools and tables are larger than declared, so
every index lies inside allocated memory whether or not a check fires."""
import sys
from types import SimpleNamespace

import torch

import kernel_harness as KH
from range_check_cases import code_of
from spissa_b200.csrc import lib as K

DEV = "cuda:0"


def main() -> int:
    nh, nkv, hd = 8, 2, 64
    meta = KH.paged_meta([1, 1], [199, 69], DEV, seed=3, spare_pages=4)
    pool = K.kv4_pool(meta.n_pages, nkv, hd, DEV)
    qkv = torch.randn(2, (nh + 2 * nkv) * hd, device=DEV)
    q = torch.empty(2, nh * hd, dtype=torch.bfloat16, device=DEV)
    out, rows = torch.empty_like(q), [torch.empty(2, nkv, hd, device=DEV) for _ in range(2)]
    pages = [torch.empty(6, nkv, 64, hd, device=DEV) for _ in range(2)]
    step = SimpleNamespace(seq_len=meta.seq_len, seq_start=meta.seq_start, n_seqs=2)
    calls = {"store": lambda: K.kv4_store(qkv, q, pool, meta, None, nh, nkv, hd, 0),
             "load": lambda: K.kv4_load(pool, meta, *rows, nkv, hd),
             "unpack": lambda: K.kv4_unpack_pages(pool, meta, *pages, torch.empty_like(meta.page_table), step, None, nkv, hd),
             "attend": lambda: K.kv4_attend(q, pool, out, meta, None, 2, 1, 200, nh, nkv, hd, None, 0.125)}
    for name, call in calls.items():
        assert code_of(call) == 0, name
    for module in ("kv4", "kv4_attention"):
        assert K.range_checked(module), f"{module} is not the debug build"
    for name, call in calls.items():
        meta.declared_pages = int(meta.page_table.max())              # the highest page in the table lies beyond the bound
        before = pool.clone()
        top = code_of(call)
        # (the highest page may be one that a store of the newest tokens does not touch)
        touched = [int(meta.page_table[0, 199 // 64]), int(meta.page_table[1, 69 // 64])]
        assert top == (401 if name in ("unpack", "attend") or meta.declared_pages in touched else 0), (name, top)
        assert torch.equal(pool[meta.declared_pages], before[meta.declared_pages]), name
        meta.declared_pages = None
        meta.declared_rows = 1                                        # the second sequence's row lies beyond it
        assert code_of(call) == 402, name
        meta.declared_rows = None
    print("four-bit range check cases ok")
    return 0


if __name__ == "__main__":
    sys.exit(main())
