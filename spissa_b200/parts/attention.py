"""Causal grouped-query attention over the cache, as a mixer.

q = x·Wqᵀ, k = x·Wkᵀ, v = x·Wvᵀ (no bias); positions are applied to q and k; k and v
go to the cache at the token's position; each query head h attends, through kv head
h // (heads / kv_heads), to the visible keys of its own sequence with scores scaled by
1/√head_dim and a 32-bit softmax; the heads are projected back with Wo.
crates/spissa-runtime/src/models/llama/generate.rs:274-450,
crates/spissa-runtime/src/rotary.rs:335-415.

The three projections run as one matrix product over the stacked weight
[Wq; Wk; Wv]. With ``window`` = w a query at position p sees keys p−w+1 … p.
A run that shares another run's cache (``cache.writes`` False) computes q only and
reads the keys the other run stored; a layer built with ``shares_kv`` has no k/v
projections at all and can only run that way.
"""
from __future__ import annotations

import math

import torch

from ..cache.views import KVLayerView
from ..csrc import lib as K
from .base import KVCacheRequest, Mixer, WeightSpec
from .linear import GEMV_TOKENS, held_linear
from .registry import build_part, register_part
from ..phases import phase


def length_bucket(max_len: int, page_size: int) -> int:
    """Powers of two up to 8 pages, then steps of 8 pages, steps that double while they are under a sixteenth of
    the length: the bucket fixes how the keys are split, and a split made for a much longer bucket leaves most
    chunks empty; a capture costs tens of milliseconds, so it should not come more often than every few hundred
    steps either."""
    b = 4 * page_size
    while b < max_len and b < 8 * page_size:
        b *= 2
    if max_len <= b:
        return b
    step = 8 * page_size
    while step * 16 < max_len:
        step *= 2
    return -(-max_len // step) * step


FLASH_TC_TOKENS = 256      # bfloat16 prompt steps of at least so many tokens take the tcgen05 attention
SPLIT4_COLUMNS = 256       # bfloat16 prompt steps of up to so many query columns (tokens x heads of a kv head) of a sequence read a four-bit cache as it lies
TILED_TOKENS = 32          # 32-bit prompt steps of at least so many tokens take the attention kernel of 64-query tiles


@register_part("mixer", "attention")
class GQAAttention(Mixer):
    graph_safe = True
    four_bit_weights = four_bit_cache = True

    def __init__(self, hidden_size: int, num_heads: int, num_kv_heads: int, head_dim: int,
                 position=None, window=None, shares_kv: bool = False, prefix: str = "", names: dict | None = None):
        super().__init__(prefix)
        if num_heads % num_kv_heads:
            raise ValueError(f"{num_heads} heads are no multiple of {num_kv_heads} kv heads")
        self.hidden_size, self.num_heads = int(hidden_size), int(num_heads)
        self.num_kv_heads, self.head_dim = int(num_kv_heads), int(head_dim)
        self.window = int(window) if window else None
        self.shares_kv = bool(shares_kv)         # this layer has no k/v projections: it reads another run's cache
        self.scale = 1.0 / math.sqrt(self.head_dim)
        n = dict(q="q_proj.weight", k="k_proj.weight", v="v_proj.weight", o="o_proj.weight")
        n.update(names or {})
        self.names = {k: prefix + v for k, v in n.items()}
        self.sink = None                         # float32 [heads]: per head a score in the softmax's denominator (subclasses)
        self.position = build_part("position", position) if position is not None else None
        if getattr(self.position, "pairing", "half") != "half":
            raise ValueError(f"{prefix}: this mixer's kernels rotate dim i with dim i + rotary_dim/2 only")
        self.qkv = self.o = None

    def children(self):
        return [self.position] if self.position is not None else []

    def weight_specs(self):
        H, nh, nkv, hd = self.hidden_size, self.num_heads, self.num_kv_heads, self.head_dim
        own = [WeightSpec(self.names["q"], (nh * hd, H)), WeightSpec(self.names["o"], (H, nh * hd))]
        if self.shares_kv:
            return own
        return own + [WeightSpec(self.names["k"], (nkv * hd, H)), WeightSpec(self.names["v"], (nkv * hd, H))]

    def cache_request(self):
        bits = self.rt.cache_bits if self.rt is not None else 16
        if bits == 4 and (self.head_dim not in K.KV4_HEAD_SIZES or self._rotated() % 8):
            raise ValueError(f"{self.prefix}: a four-bit cache takes heads of {', '.join(map(str, K.KV4_HEAD_SIZES))} of which a multiple of 8 "
                             f"dims is rotated, got {self.head_dim} and {self._rotated()}")
        return KVCacheRequest(self.num_kv_heads, self.head_dim, self.window, bits=bits)

    def _rotated(self) -> int:
        return self.position.rotary_dim if self.position is not None and hasattr(self.position, "rotary") else 0

    def bind(self, tensors, rt):
        super().bind(tensors, rt)
        q = tensors[self.names["q"]]
        shared = rt.weight_bits == 4 and not self.shares_kv and q.shape[0] % 16 == 0        # q's rows are whole tiles of the packed q, k, v
        self.q_only = None if shared else held_linear(q, rt)
        if not self.shares_kv:
            k, v = tensors[self.names["k"]], tensors[self.names["v"]]
            if not (q.dtype == k.dtype == v.dtype):
                raise ValueError(f"{self.prefix}: q, k and v projections must share a storage type")
            self.qkv = held_linear(torch.cat([q, k, v], dim=0), rt)
            if shared:
                self.q_only = self.qkv.first_rows(q.shape[0])
        self.o = held_linear(tensors[self.names["o"]], rt)
        # arrival counters of the split-key decode attention; the kernel returns them to zero
        self.counters = torch.zeros(4096, dtype=torch.int32, device=rt.device)

    def fused_fields(self):
        rotary = self.position is not None and hasattr(self.position, "rotary")
        if self.shares_kv or self.window or not rotary or self.qkv is None or self.rt.weight_bits != 16 or self.rt.cache_bits != 16:
            return None
        inv_freq, rd = self.position.rotary()
        if rd != self.head_dim or self.qkv.weight.dtype != torch.bfloat16 or self.o.weight.dtype != torch.bfloat16:
            return None
        return dict(kind="gqa_rotary", qkv=self.qkv.weight, o=self.o.weight, inv_freq=inv_freq, scale=self.scale,
                    inv_freq_host=getattr(self.position, "inv_freq_host", None),
                    hidden_size=self.hidden_size, num_heads=self.num_heads, num_kv_heads=self.num_kv_heads,
                    head_dim=self.head_dim)

    def forward(self, x, step, cache, residual):
        nh, nkv, hd = self.num_heads, self.num_kv_heads, self.head_dim
        T = x.shape[0]
        writes = cache.writes
        if writes and self.shares_kv:
            raise ValueError(f"{self.prefix}: a layer without k/v projections cannot be the writer of a cache")
        rd, inv_freq = 0, None
        rotary = self.position is not None and hasattr(self.position, "rotary")
        if rotary:
            inv_freq, rd = self.position.rotary()
        q = torch.empty(T, nh * hd, dtype=self.rt.act_dtype, device=x.device)
        w = self.qkv.weight if writes and self.rt.weight_bits == 16 else None
        if (w is not None and rotary and rd == hd and hd % 16 == 0 and T <= GEMV_TOKENS and q.dtype == torch.bfloat16
                and cache.k_pool.dtype == torch.bfloat16 and K.gemv_supported(x, w)):
            # a few tokens: one kernel does the QKV product, the rotation and the cache write
            with phase("qkv_projection+rotary+kv_append_ms"):
                K.gemv_qkv_rope(x, w, q, cache.k_pool, cache.v_pool, cache, inv_freq, nh, nkv, hd)
        else:
            with phase("qkv_projection_ms"):
                proj = self.qkv if writes else self.q_only
                qkv = proj(x, out_dtype=torch.float32)             # rotation reads unrounded products
                if not writes:
                    pad = torch.empty(T, (nh + 2 * nkv) * hd, dtype=torch.float32, device=x.device)
                    pad[:, :nh * hd] = qkv
                    qkv = pad
            with phase("rotary+kv_append_ms"):
                if self.position is not None and not rotary:
                    self.position.apply(qkv, step, nh, nkv, hd)
                if getattr(cache, "bits", 16) == 4:
                    K.kv4_store(qkv, q, cache.k_pool, cache, inv_freq, nh, nkv, hd, rd, write_kv=writes)
                else:
                    K.rope_kv_write(qkv, q, cache.k_pool, cache.v_pool, cache, inv_freq, nh, nkv, hd, rd, write_kv=writes)
        with phase("attention_ms"):
            ctx = self.attend(q, step, cache)
        with phase("o_projection+attention_residual_ms"):
            self.o(ctx, out=residual, accumulate=True)

    def attend(self, q, step, cache):
        """The heads' outputs [T, heads·head_dim] for queries ``q`` (positions applied) over the keys and values that
        the cache holds for each token's sequence, the step's own tokens included."""
        return attend_paged(q, step, cache, self.num_heads, self.num_kv_heads, self.head_dim, self.window, self.scale,
                            self.sink, self.counters)


def attention_modules(hd: int, vd: int) -> tuple:
    """The kernel libraries that ``attend_paged`` needs for bfloat16 key rows of ``hd`` and value rows of ``vd`` entries."""
    if hd == vd and hd % 16 == 0 and hd <= 128:
        return ("attention",)
    if hd % 8 or vd % 8 or max(hd, vd) > 128:
        return ()
    return ("attention_kv", "flash_tc") if hd > 32 else ("attention_kv",)


def attend_paged(q, step, cache, nh, nkv, hd, window, scale, sink=None, counters=None, dist_bias=None, vd=None):
    """Softmax attention of the step's queries ``q`` [T, nh·hd] over the paged keys and values of ``cache`` (a
    ``KVLayerView``): the tensor-core kernels where they take the sizes, else the generic one. ``vd``: the size of a value
    row where it differs from a key row's. ``sink``: float32 [nh] or None. ``dist_bias``: float32 [nh, distances] or None,
    a score added by the distance between query and key. ``counters``: the arrival counters of the split-key decode
    kernel."""
    T = q.shape[0]
    if vd == hd:
        vd = None
    if getattr(cache, "bits", 16) == 4:
        if vd is not None or dist_bias is not None:
            raise K.KernelError("attention over a four-bit cache takes key and value rows of one size and no scores by distance")
        return attend_four_bits(q, step, cache, nh, nkv, hd, window, scale, sink)
    ctx = torch.empty_like(q) if vd is None else torch.empty(T, nh * vd, dtype=q.dtype, device=q.device)
    if vd is None and K.flash_supported(q, cache.k_pool, nh, nkv, hd, cache.page_size):
        flash = {}
    elif q.dtype == torch.bfloat16 and K.flash_kv_supported(q, cache.k_pool, nh, nkv, hd, vd or hd, cache.page_size):
        flash = dict(vd=vd or hd)              # sizes of their own, or one that the kernels for one size are not built for
    elif (not step.all_single and T >= TILED_TOKENS
          and K.attention_tile_f32_supported(q, cache.k_pool, cache.v_pool, step.n_seqs, nh, nkv, hd, vd or hd)):
        K.attention_tile_f32(q, cache.k_pool, cache.v_pool, ctx, cache, step.seq_start, step.n_seqs, step.max_new, nh, nkv, hd, window,
                             scale, vd=vd, sink=sink, dist_bias=dist_bias)
        return ctx
    else:
        # (a decode step by its length's bucket, as below: run directly and replayed from a graph it takes the same way)
        longest = length_bucket(step.max_len, cache.page_size) if step.all_single else step.max_len
        K.attention_generic(q, cache.k_pool, cache.v_pool, ctx, cache, nh, nkv, hd, window, scale, vd=vd, sink=sink,
                            dist_bias=dist_bias, longest=longest)
        return ctx
    if step.all_single:
        # the split is made for the length's bucket, not the length: a step run directly and the same step
        # replayed from a graph (captured for the bucket) then add up in the same order, bit for bit
        chunk_tiles, n_chunks = K.flash_decode_plan(T, nkv, length_bucket(step.max_len, cache.page_size),
                                                    cache.page_size)
        need = K.flash_decode_scratch_floats(T, nh, vd or hd, n_chunks)
        scratch = torch.empty(need, dtype=torch.float32, device=q.device)
        K.flash_decode(q, cache.k_pool, cache.v_pool, ctx, cache, step.seq_len, nh, nkv, hd, window,
                       scale, chunk_tiles, n_chunks, scratch,
                       counters if counters is not None and T * nkv <= counters.numel() else None, sink=sink,
                       dist_bias=dist_bias, **flash)
    elif T >= FLASH_TC_TOKENS and K.flash_tc_supported(q, cache.k_pool, nh, nkv, hd, cache.page_size, window, vd=vd):
        # long prompts: 128-token tiles on the tcgen05 tensor cores (S, P and O in tensor memory)
        tiles = K.query_tiles(step.host["new_counts"], K.flash_tc_query_tile())
        K.flash_prefill_tc(q, cache.k_pool, cache.v_pool, ctx, cache, step.seq_start, step.n_seqs, tiles,
                           nh, nkv, hd, window, scale, sink=sink, dist_bias=dist_bias, vd=vd)
    else:
        tiles = K.query_tiles(step.host["new_counts"], K.flash_query_tile())
        K.flash_prefill(q, cache.k_pool, cache.v_pool, ctx, cache, step.seq_start, step.n_seqs,
                        tiles, nh, nkv, hd, window, scale, sink=sink, dist_bias=dist_bias, **flash)
    return ctx


def reads_codes(q, cols: int, nkv: int, hd: int = 128, n_seqs: int = 1) -> bool:
    """Whether a prompt step's attention works on the codes of a four-bit cache, or on its pages unpacked first. ``cols``: the most
    query columns of a sequence. On the codes every 16 columns take a page apart again; unpacked, steps meet the tile kernels, which take
    a sequence's keys one after another, in a time that hardly depends on the tokens while all tiles run at once. So the codes win while
    THEIR tiles find room on the SMs at once (``lib.kv4_room``). Measured, us (codes / unpacked first), bfloat16, one sequence:
      32 heads on 8 of 128, behind 2,000: 64 tokens 32/75, 128 50/76, 192 81/78, 256 95/58, 1,024 365/75; behind 100,000: 128 1,748/3,102, 256 3,478/2,364;
      32 on 8 of 64, behind 2,000: 192 41/47, 256 65/36;    32 on 8 of 96: 192 77/57, 512 161/62;    32 on 8 of 32: 192 31/33, 512 66/44;
      9 on 3 of 96, behind 2,000: 256 29/55, 512 46/60, 1,024 96/69; behind 100,000: 256 748/2,316;    12 on 12 of 96: 384 45/61, 512 82/64;
      16 on 1 of 128, behind 2,000: 256 50/53, 512 100/57;    6 on 2 of 32: 512 24/36, 1,024 40/42; behind 100,000: 512 548/1,129;
    1,024 tokens of 64 sequences behind 1,000 (32 on 8 of 128): 180/283; float32: 512 tokens behind nothing 63/146, behind 2,000 254/960."""
    if q.dtype == torch.float32:
        return nkv * -(-cols // 16) < 1 << 16            # (tiles of columns are a grid's second dimension)
    return q.shape[0] < FLASH_TC_TOKENS or cols <= SPLIT4_COLUMNS or n_seqs * nkv * -(-cols // 16) <= K.kv4_room(hd)


def attend_four_bits(q, step, cache, nh, nkv, hd, window, scale, sink=None):
    """``attend_paged`` over pages of four bits."""
    T = q.shape[0]
    if q.dtype not in (torch.bfloat16, torch.float32) or tuple(q.shape) != (T, nh * hd) or nh % nkv:
        raise K.KernelError(f"attention: queries are [tokens, {nh} x {hd}], bfloat16 or float32, of heads in equal groups")
    if not scale > 0:
        raise K.KernelError(f"attention over a four-bit cache takes a positive scale, got {scale}")
    if step.all_single or reads_codes(q, step.max_new * (nh // nkv), nkv, hd, step.n_seqs):
        out = torch.empty_like(q)
        # (a decode step by its length's bucket, as below: run directly and replayed from a graph it adds up in the same order)
        longest = length_bucket(step.max_len, cache.page_size) if step.all_single else step.max_len
        K.kv4_attend(q, cache.k_pool, out, cache, None if step.all_single else step.seq_start, step.n_seqs, step.max_new, longest, nh, nkv, hd,
                     window, scale, sink)
        return out
    lens = step.host.get("seq_len") or step.seq_len.tolist()
    n_pages = sum(-(-n // cache.page_size) for n in lens)
    k = torch.empty(n_pages, nkv, cache.page_size, hd, dtype=q.dtype, device=q.device)
    v = torch.empty_like(k)
    table = torch.empty_like(cache.page_table)
    K.kv4_unpack_pages(cache.k_pool, cache, k, v, table, step, window, nkv, hd)
    rows = torch.arange(step.n_seqs, dtype=torch.int32, device=q.device)
    plain = KVLayerView(k, v, table, cache.page_size, cache.token_seq, cache.positions, rows, cache.window, False)
    return attend_paged(q, step, plain, nh, nkv, hd, window, scale, sink)
