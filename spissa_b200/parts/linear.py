"""y = x · Wᵀ with W stored [out, in] (crates/spissa-runtime/src/ops.rs:62-105).

``Linear`` holds one weight matrix and picks the kernel for a call by the operands'
storage types and sizes: bfloat16 activations on a bfloat16 weight go to the weight-streaming
kernel for a few tokens (decoding), to the tcgen05 kernel with the weight's rows as the instruction's M for some dozens
to some hundreds of tokens, and to the tcgen05 tile kernel otherwise, when the rows are multiples of 16 bytes;
32-bit products of more than ``GEMV_TOKENS`` rows go to the tcgen05 kernel that multiplies float32 in bfloat16 parts;
everything else goes to the FFMA kernels.

``Linear4`` and ``GatedLinear4`` hold their weights in four bits with a scale for every ``group`` columns (not in the
reference; csrc/q4.cuh states the format): the numbers that stand in their place are exactly bfloat16, and all their
products multiply those.
"""
from __future__ import annotations

import torch

from ..csrc import lib as K

_SM_COUNT: dict = {}


def sm_count(device=None) -> int:
    """Streaming multiprocessors of ``device`` (the current CUDA device when None), asked once per device."""
    index = torch.cuda.current_device() if device is None else (torch.device(device).index or 0)
    if index not in _SM_COUNT:
        _SM_COUNT[index] = int(torch.cuda.get_device_properties(index).multi_processor_count)
    return _SM_COUNT[index]
GEMV_TOKENS = 16          # up to this many tokens the weight-streaming kernel runs instead of 128-row tiles
GATED_GEMV_TOKENS = 16    # the same for the gate/up product
MID_TOKENS = 1023         # from there up to this many tokens the weight's rows are the instruction's M and the tokens its N
#                           (tc_mid.cu). Per layer of the 1B shape (QKV + output + gate/up + down, us) against what ran before
#                           (tc_stream.cu up to 64 tokens, tc_gemm.cu's tiles of 128 tokens beyond): 33 tokens 44 / 47, 64: 47 / 50,
#                           100: 53 / 92, 301: 67 / 122, 512: 83 / 108, 1,000: 138 / 201; of the 8B shape 100: 110 / 149,
#                           301: 171 / 254, 700: 321 / 416, 1,000: 430 / 435. Gated products, and from 1,024 tokens on all, go by the
#                           estimates of sp_tc_mid_or_pairs: tc_gemm.cu's pairs of CTAs read half as much per product where they have
#                           enough tiles
F32_PARTS_K = 128         # 32-bit products with sums at least so long go to tc_f32.cu. Relative error against 64 bits there / in order
#                           on FFMA: K = 8 1.0e-7 / 5e-8, 72: 1.2e-7 / 1.5e-7, 128: 1.3e-7 / 2.0e-7, 2,048: 1.6e-7 / 8.1e-7
STREAM_TOKENS = 64        # what tc_mid.cu does not take (gate and up rows in blocks of 64): tc_stream.cu up to this many tokens


PAIR_TOKENS = 1024        # from here on tc_gemm.cu computes all its tiles, of 256 rows, by pairs of CTAs
MOST_MID_TOKENS = 2048    # the most that tc_mid.cu is built for


def mid_takes(mode, x: torch.Tensor, w: torch.Tensor) -> bool:
    """Whether tc_mid.cu is the faster one for a product that tc_gemm.cu's tiles could take as well."""
    return (x.shape[0] <= MID_TOKENS and mode != K.TC_SILU_MUL) or not K.tc_mid_or_pairs(mode, x.shape[0], w.shape[0], w.shape[1], 1, x.device.index)


def tile_width(M: int, N: int, sms: int | None = None) -> int:
    """256-wide tiles (half the shared-memory traffic per FLOP) when they still occupy most SMs, else 128-wide;
    192-wide when that saves a round of tiles: 2,048 tokens x 3,072 outputs are 96 pair tiles of 256 columns, two
    rounds on 74 pairs of which the second is a third full, but 128 tiles of 192 columns, two rounds of shorter tiles.
    The rounds are counted as the kernel walks them, by pairs of row tiles from ``PAIR_TOKENS`` on: 6,000 tokens x 4,096 of
    the 8B shape are 6 rounds of 256 columns or 8 of 192, and a 192-wide tile costs an eighth more per column: the output
    product 213 us at 192, 160 at 256, the down product 675 and 566."""
    SM_COUNT = sms if sms else sm_count()
    paired = M >= PAIR_TOKENS
    m_tiles, walkers = ((M + 255) // 256, SM_COUNT // 2) if paired else ((M + 127) // 128, SM_COUNT)
    tiles_256 = m_tiles * ((N + 255) // 256)
    if tiles_256 < (walkers * 2) // 3:
        return 128
    if M > 128:
        cost_256 = -(-tiles_256 // walkers) * 256
        cost_192 = -(-(m_tiles * ((N + 191) // 192)) // walkers) * 192
        if cost_192 * (9 if paired else 10) <= cost_256 * (8 if paired else 9):
            return 192
    return 256


class Linear:
    def __init__(self, weight: torch.Tensor):
        if weight.dim() != 2:
            raise ValueError("a linear weight is a matrix [out, in]")
        self.weight = weight.contiguous()
        self.out_features, self.in_features = weight.shape

    def __call__(self, x: torch.Tensor, out: torch.Tensor | None = None, out_dtype=None,
                 accumulate: bool = False) -> torch.Tensor:
        """``accumulate`` adds the product into ``out`` (float32) instead of overwriting it."""
        if out is None:
            if accumulate:
                raise ValueError("accumulation needs the tensor to add into")
            out = torch.empty(x.shape[0], self.out_features, dtype=out_dtype or x.dtype, device=x.device)
        mode = K.TC_ACCUMULATE if accumulate else K.TC_STORE
        bf16 = x.dtype == torch.bfloat16                     # (a float32 model asks for no library of the bfloat16 kernels)
        if x.shape[0] <= GEMV_TOKENS and K.gemv_supported(x, self.weight):
            K.gemv(x, self.weight, out, mode)
        elif bf16 and x.shape[0] <= MOST_MID_TOKENS and mid_takes(mode, x, self.weight) and K.tc_mid_supported(x, self.weight, out, mode):
            K.tc_mid(x, self.weight, out, mode)
        elif x.shape[0] <= STREAM_TOKENS and K.tc_stream_supported(x, self.weight, mode):
            K.tc_stream(x, self.weight, out, mode)
        elif K.tc_gemm_supported(x, self.weight):
            width = x.shape[0] >= PAIR_TOKENS and K.tc_mid_or_pairs(mode, x.shape[0], self.out_features, self.in_features, 1, x.device.index)
            K.tc_gemm(x, self.weight, out, mode, width or tile_width(x.shape[0], self.out_features, sm_count(x.device)))
        elif x.shape[0] > GEMV_TOKENS and x.shape[1] >= F32_PARTS_K and K.tc_f32_supported(x, self.weight, out):
            K.tc_f32(x, self.weight, out, accumulate=accumulate)
        else:
            K.gemm_generic(x, self.weight, out, accumulate=accumulate)
        return out


class GatedLinear:
    """act(x·Wgᵀ) ⊙ (x·Wuᵀ) · mult as one product over the stacked weight (``act``: K.ACT_SILU or K.ACT_GELU; K.ACT_CLAMPED with
    its ``limit`` and ``slope``: g·sigmoid(slope·g)·(u + 1), g = min(x·Wgᵀ, limit), u = clamp(x·Wuᵀ, ±limit)).

    When the sizes allow, gate and up rows are interleaved in blocks (``block`` gate rows, then
    the ``block`` up rows of the same outputs) so that one tile of the tensor-core kernel holds
    both halves and applies act·up in its epilogue.
    """

    def __init__(self, gate: torch.Tensor, up: torch.Tensor, act: int = K.ACT_SILU, mult: float = 1.0, limit: float = 0.0,
                 slope: float = 0.0):
        I = gate.shape[0]
        self.act, self.mult = act, float(mult)
        self.limit, self.slope = float(limit), float(slope)
        if act == K.ACT_CLAMPED and self.mult != 1.0:
            raise ValueError("the clamped unit takes no factor")
        self.intermediate = I
        self.block = 128 if I % 128 == 0 else 64 if I % 64 == 0 else 0
        fused = self.block and gate.dtype == torch.bfloat16 and gate.shape[1] % 8 == 0
        if act == K.ACT_CLAMPED and not self.limit > 0:
            fused = 0                                    # the epilogues are built for positive limits
        if fused:
            h = self.block
            g = gate.reshape(I // h, h, -1)
            u = up.reshape(I // h, h, -1)
            self.weight = torch.stack([g, u], dim=1).reshape(2 * I, -1).contiguous()
        else:
            self.block = 0
            self.weight = torch.cat([gate, up], dim=0).contiguous()
        self.plain = Linear(self.weight)

    def __call__(self, x: torch.Tensor, act_dtype) -> torch.Tensor:
        out = torch.empty(x.shape[0], self.intermediate, dtype=act_dtype, device=x.device)
        kw = dict(act=self.act, mult=self.mult, limit=self.limit, slope=self.slope)
        if self.block and x.shape[0] <= GATED_GEMV_TOKENS and K.gemv_supported(x, self.weight):
            K.gemv(x, self.weight, out, K.TC_SILU_MUL, self.block, **kw)
        elif (self.block and x.shape[0] <= MOST_MID_TOKENS and mid_takes(K.TC_SILU_MUL, x, self.weight)
              and K.tc_mid_supported(x, self.weight, out, K.TC_SILU_MUL, self.block)):
            K.tc_mid(x, self.weight, out, K.TC_SILU_MUL, self.block, **kw)
        elif self.block and x.shape[0] <= STREAM_TOKENS and K.tc_stream_supported(x, self.weight, K.TC_SILU_MUL, self.block):
            K.tc_stream(x, self.weight, out, K.TC_SILU_MUL, self.block, **kw)
        elif self.block and K.tc_gemm_supported(x, self.weight):
            K.tc_gemm(x, self.weight, out, K.TC_SILU_MUL, 2 * self.block, **kw)
        elif self.act == K.ACT_CLAMPED:
            K.clamped_glu(self.plain(x, out_dtype=torch.float32), out, self.limit, self.slope)     # the clamps read unrounded products
        else:
            gu = self.plain(x, out_dtype=act_dtype)
            K.gated_mul(gu, out, self.act, self.mult)
        return out


class Linear4:
    """y = x · Ŵᵀ, Ŵ the numbers that ``weight`` [out, in] becomes in four bits, in groups of ``group`` (32, 64 or 128) columns;
    in a multiple of the group. Called as ``Linear``: x bfloat16 or float32. Up to 16 rows stream the codes (from 9 bfloat16 rows on only
    of small weights), up to 1,024 bfloat16 rows multiply with them on the tcgen05 cores where that is estimated to be the faster way
    (``product4``), more, and float32 ones from 17 on, unpack the weight first."""

    def __init__(self, weight: torch.Tensor, group: int = 64):
        if weight.dim() != 2:
            raise ValueError("a linear weight is a matrix [out, in]")
        self.out_features, self.in_features = weight.shape
        self.group = int(group)
        self.codes, self.scales = K.q4_pack(weight.contiguous(), self.group)

    def first_rows(self, n: int) -> "Linear4":
        """The product with the first ``n`` rows of the weight (a multiple of 16: the codes of whole tiles), sharing its codes."""
        if n <= 0 or n % 16 or n > self.out_features:
            raise ValueError(f"rows of a four-bit weight are taken in tiles of 16, got {n} of {self.out_features}")
        part = Linear4.__new__(Linear4)
        part.out_features, part.in_features, part.group = n, self.in_features, self.group
        part.codes, part.scales = self.codes[:n // 16], self.scales[:n // 16]
        return part

    def unpacked(self, dtype=torch.bfloat16) -> torch.Tensor:
        w = torch.empty(self.out_features, self.in_features, dtype=dtype, device=self.codes.device)
        K.q4_unpack(self.codes, self.scales, w, self.group)
        return w

    def __call__(self, x: torch.Tensor, out: torch.Tensor | None = None, out_dtype=None,
                 accumulate: bool = False) -> torch.Tensor:
        """``accumulate`` adds the product into ``out`` (float32) instead of overwriting it."""
        if out is None:
            if accumulate:
                raise ValueError("accumulation needs the tensor to add into")
            out = x.new_empty((x.shape[0], self.out_features), dtype=out_dtype)
        M = check4(self, x, out, self.out_features, accumulate)
        if M == 0:
            return out
        way, mode = product4(self, x, self.out_features), K.TC_ACCUMULATE if accumulate else K.TC_STORE
        if way == "unpack":
            return Linear(self.unpacked(x.dtype))(on_boundaries(x, 8), out=out, accumulate=accumulate)
        (K.q4_gemv if way == "gemv" else K.q4_tc)(on_boundaries(x), self.codes, self.scales, out, self.out_features, self.group, 0, mode)
        return out


class GatedLinear4:
    """act(x·Ŵgᵀ) ⊙ (x·Ŵuᵀ) · mult with gate and up weights in four bits (``act``: K.ACT_SILU or K.ACT_GELU)."""

    def __init__(self, gate: torch.Tensor, up: torch.Tensor, act: int = K.ACT_SILU, mult: float = 1.0, group: int = 64):
        if gate.dim() != 2 or gate.shape != up.shape or gate.dtype != up.dtype:
            raise ValueError("gate and up weights are two matrices [out, in] of one type")
        if act not in (K.ACT_SILU, K.ACT_GELU):
            raise ValueError("gated products of four-bit weights are built for silu and gelu")
        self.act, self.mult, self.group = act, float(mult), int(group)
        self.intermediate, self.in_features = gate.shape
        self.codes, self.scales = K.q4_pack(torch.cat([gate, up], dim=0), self.group, half=self.intermediate)

    def unpacked(self, dtype=torch.bfloat16) -> GatedLinear:
        """The product over the numbers the codes stand for."""
        plain = GatedLinear.__new__(GatedLinear)
        I = self.intermediate
        plain.act, plain.mult, plain.limit, plain.slope, plain.intermediate = self.act, self.mult, 0.0, 0.0, I
        plain.block = 0 if dtype != torch.bfloat16 else 128 if I % 128 == 0 else 64 if I % 64 == 0 else 0
        plain.weight = torch.empty(2 * I, self.in_features, dtype=dtype, device=self.codes.device)
        K.q4_unpack(self.codes, self.scales, plain.weight, self.group, half=I, block=plain.block)
        plain.plain = Linear(plain.weight)
        return plain

    def __call__(self, x: torch.Tensor, act_dtype) -> torch.Tensor:
        out = x.new_empty((x.shape[0], self.intermediate), dtype=act_dtype)
        M = check4(self, x, out, self.intermediate, False)
        if M == 0:
            return out
        way = product4(self, x, 2 * self.intermediate, self.intermediate)
        if way == "unpack":
            return self.unpacked(x.dtype)(on_boundaries(x, 8), act_dtype)
        (K.q4_gemv if way == "gemv" else K.q4_tc)(on_boundaries(x), self.codes, self.scales, out, 2 * self.intermediate, self.group,
                                                  self.intermediate, K.TC_SILU_MUL, self.act, self.mult)
        return out


def product4(lin, x, rows: int, half: int = 0) -> str:
    """The way of a product of four-bit weights (``rows`` of them): "gemv" streams the codes (q4_kernels.cu), "tc" multiplies with
    them on the tcgen05 cores (q4_tc.cu), "unpack" takes the weight apart in memory. Measured, us:
      9 to 16 rows of x, weight 14336 x 4096 gate and up: gemv 51, tc 32; 4096 x 4096: 11, 9.6; 2048 x 2048: 6.4, 7.7;
      256 rows, gate and up: tc 73, unpack 111; 4096 x 4096: 17, 25 (more sizes: q4_tc.cu).
    Beyond 256 rows tc takes each code apart more than once, unpack writes and reads 2 bytes a number once: an estimate of each
    decides, unpack's as 2,300 numbers a nanosecond and a product of 1.5 PFLOP/s that starts in 9 us."""
    M, numbers = x.shape[0], rows * lin.in_features
    if M <= 8 or (M <= K.Q4_GEMV_ROWS and (numbers < 1 << 23 or x.dtype != torch.bfloat16)):
        return "gemv"
    if x.dtype != torch.bfloat16 or M > K.Q4_TC_ROWS:
        return "unpack"
    if M <= 256 or K.q4_tc_estimate(M, rows, lin.in_features, lin.group, half) < numbers / 2300 + 9000 + M * numbers * 2 / 1.5e6:
        return "tc"
    return "unpack"


def held_linear(weight: torch.Tensor, rt):
    """A linear operator that holds its weight in as many bits as the runtime asks for."""
    return Linear4(weight, group_of(weight)) if rt.weight_bits == 4 else Linear(weight)


def held_gated(gate: torch.Tensor, up: torch.Tensor, act: int, mult: float, rt):
    return GatedLinear4(gate, up, act, mult, group_of(gate)) if rt.weight_bits == 4 else GatedLinear(gate, up, act, mult)


def group_of(weight: torch.Tensor) -> int:
    """Columns that share a scale: 64 (4.25 bits a number), 32 where the rows are no multiple of that."""
    return 64 if weight.shape[1] % 64 == 0 else 32


_ROWS = (torch.bfloat16, torch.float32)


def check4(lin, x, out, out_features: int, accumulate: bool) -> int:
    """Refuses what the products of four-bit weights do not take; the number of rows."""
    if x.dtype not in _ROWS or out.dtype not in _ROWS or (accumulate and out.dtype != torch.float32):
        raise K.KernelError(f"products of four-bit weights take bfloat16 or float32 rows, are stored as either and added into float32; got "
                            f"{x.dtype} rows and a {out.dtype} output")
    if x.dim() != 2 or x.shape[1] != lin.in_features or out.shape != (x.shape[0], out_features):
        raise K.KernelError(f"shapes do not match: x {tuple(x.shape)}, weight [{out_features}, {lin.in_features}], out {tuple(out.shape)}")
    if x.stride(1) != 1 or out.stride(1) != 1:
        raise K.KernelError("product operands must have unit stride in their last dimension")
    if x.shape[0] > 1 and out.stride(0) < out_features:
        raise K.KernelError("the rows of a product's output may not overlap")
    if not (x.get_device() == out.get_device() == lin.codes.get_device() == torch._C._cuda_getDevice()):
        raise K.KernelError(f"the weight (on {lin.codes.device}), its rows and its output live on the current device, got {x.device} and {out.device}")
    return x.shape[0]


def on_boundaries(x, entries: int = 0):
    """``x``, or a copy of it where its rows do not start on boundaries of 16 bytes, or of ``entries`` numbers where those are more
    (columns of wider rows, an odd offset), or overlap (one row for all): the tensor-core kernels take no such rows (the 32-bit one wants
    8 numbers), and what does is the FFMA product (2,048 bfloat16 rows of 4096 x 4096, us: 3,100, with the copy 86; 200 float32
    ones 590 and 92)."""
    size = max(16, entries * x.element_size())
    if (x.data_ptr() | x.stride(0) * x.element_size()) % size == 0 and x.stride(0) >= x.shape[1]:
        return x
    return x.clone(memory_format=torch.contiguous_format)
