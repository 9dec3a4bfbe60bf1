"""Timed operators: four bits a number for weights and for cached keys and values.

One format serves both. A group of neighbouring numbers x (32 along a head of the cache; 32, 64 or 128 along a weight's row)
has a scale s with four significant bits, a zero z and a code c a number, both in 0..15; the number it stands for is
s · (c − z), which is exactly a bfloat16:

    lo = min(0, min x), hi = max(0, max x)
    s = (hi − lo) / 15, rounded up to four significant bits       (hi − lo < 2^-100: s = z = c = 0)
    z = round(−lo / s),  c = clamp(round(x / s) + z, 0, 15)       (quotients rounded to nearest, ties to even)

Products: y = x · Wᵀ for W held so, and act(x · Wgᵀ) ⊙ (x · Wuᵀ). Store: q and k of the QKV product are rotated, k and v
quantised into the pages of the cache and read back as the values they stand for. Attention: of one token a sequence, of a few
behind a long cache and of whole prompts, over pages held so.

With ``own`` false everything runs in elementary tensor operations in 32 bits; ``exact`` states the same in 64.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
F64 = torch.float64
GROUP = 32                       # of the cache
PAGE = 64
THETA = 500000.0

HEADS_1B = dict(nh=32, nkv=8, hd=64)
HEADS_8B = dict(nh=32, nkv=8, hd=128)


# ---------------------------------------------------------------------------------------------------------- the cases
def linear(name, M, N, K, group, dtype="bfloat16"):
    return dict(name=name, kind="linear", M=M, N=N, K=K, group=group, dtype=dtype)


def gated(name, M, N, K, group, dtype="bfloat16"):
    return dict(name=name, kind="gated", M=M, N=N, K=K, group=group, dtype=dtype)


def store(name, tokens, seqs, cached, heads, rd, dtype="bfloat16"):
    return dict(name=name, kind="store", tokens=tokens, seqs=seqs, cached=cached, rd=rd, dtype=dtype, **heads)


def attend(name, tokens, seqs, cached, heads, window=0, dtype="bfloat16"):
    return dict(name=name, kind="attend", tokens=tokens, seqs=seqs, cached=cached, window=window, dtype=dtype, **heads)


def listed():
    return [
        # one user's decode step at the 8B layer sizes, the down product: the smallest call a server makes of it
        linear("linear_1", 1, 4096, 14336, 64),
        # gate and up of a decode step of eight users, 8B sizes
        gated("gated_8", 8, 14336, 4096, 128),
        # the true 32-bit mode: the down product of the 1B sizes for four users
        linear("linear_fp32_4", 4, 2048, 8192, 32, "float32"),
        # gate and up of three requests that arrive together, some hundred tokens, 1B sizes
        gated("gated_prompt_301", 301, 8192, 2048, 64),
        # a document-sized prompt through the output product, 8B sizes
        linear("linear_prompt_2048", 2048, 4096, 4096, 64),
        # the keys and values of a decode step of eight users behind long contexts
        store("store_decode_8", 8, 8, 60000, HEADS_8B, 128),
        # the same of three prompts of unequal length
        store("store_prompt_2000", 2000, 3, 0, HEADS_8B, 128),
        # one user's decode step behind a prompt of 2,048 tokens, 1B sizes
        attend("attend_decode_1", 1, 1, 2048, HEADS_1B),
        # a full server, 8B sizes
        attend("attend_decode_64", 64, 64, 2048, HEADS_8B),
        # three users with book-sized contexts: what a cache of four bits makes room for
        attend("attend_decode_long", 3, 3, 60000, HEADS_8B),
        # a chat turn of some dozen tokens behind a long conversation
        attend("attend_turn_40", 40, 1, 6000, HEADS_8B),
        # prompts of unequal length that arrive together
        attend("attend_prompt_2000", 2000, 3, 0, HEADS_8B),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


DRAWN_HEADS = [HEADS_1B, HEADS_8B, dict(nh=32, nkv=8, hd=128), dict(nh=16, nkv=2, hd=64), dict(nh=9, nkv=3, hd=96),
               dict(nh=8, nkv=8, hd=64), dict(nh=20, nkv=2, hd=128), dict(nh=6, nkv=2, hd=32)]


def draw(rng):
    kind = rng.choice(["linear", "linear", "gated", "store", "decode", "decode", "decode", "turn", "prompt"])
    dtype = "float32" if rng.random() < 0.2 else "bfloat16"
    if kind in ("linear", "gated"):
        group = rng.choice([32, 64, 128])
        if rng.random() < 0.5:
            N, K = rng.choice([(4096, 4096), (2048, 8192), (4096, 14336), (2048, 2048)] if kind == "linear"
                              else [(8192, 2048), (14336, 4096)])
        else:                                                        # odd sizes
            N, K = _log(rng, 100, 8192), group * max(1, _log(rng, 256, 8192) // group)
        M = _log(rng, 1, 16) if rng.random() < 0.5 else _log(rng, 1, 1024 if dtype == "bfloat16" else 200)
        c = (linear if kind == "linear" else gated)("", M, N, K, group, dtype)
    elif kind == "store":
        heads = rng.choice(DRAWN_HEADS)
        tokens = _log(rng, 1, 2000)
        c = store("", tokens, rng.randint(1, min(8, tokens)), _log(rng, 1, 100000), heads,
                  rng.choice([heads["hd"], heads["hd"], heads["hd"] // 2, 0]), dtype)
    elif kind == "decode":
        seqs = _log(rng, 1, 64)
        c = attend("", seqs, seqs, _log(rng, 1, 150000 // seqs), rng.choice(DRAWN_HEADS),
                   rng.choice([0, 0, 0, _log(rng, 1, 4096)]), dtype)
    elif kind == "turn":
        tokens = _log(rng, 2, 60)
        c = attend("", tokens, rng.randint(1, min(3, tokens)), _log(rng, 1, 8000), rng.choice(DRAWN_HEADS),
                   rng.choice([0, 0, 0, _log(rng, 1, 2048)]), dtype)
    else:
        tokens = _log(rng, 20, 2000)
        c = attend("", tokens, rng.randint(1, 4), rng.choice([0, 0, _log(rng, 1, 1000)]), rng.choice(DRAWN_HEADS),
                   rng.choice([0, 0, 0, _log(rng, 1, 2048)]), dtype)
    c.pop("name")
    return c


# ------------------------------------------------------------------------------------------------------------- inputs
def torch_dtype(case):
    return getattr(torch, case["dtype"])


class Source:
    """Random tensors from one seed."""

    def __init__(self, seed):
        self.gen = torch.Generator(device=DEV)
        self.gen.manual_seed(1000003 * int(seed) + 41)
        self.host = random.Random(1000003 * int(seed) + 43)

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        return torch.empty(shape, dtype=torch.float32, device=DEV).normal_(0.0, std, generator=self.gen).to(dtype)


def counts_of(case):
    """(cached, new) tokens of every sequence: unequal, each with at least one new token."""
    r = random.Random(case["tokens"] * 131 + case["seqs"] * 17 + case["cached"])
    n, total = case["seqs"], case["tokens"]
    if n == total:
        new = [1] * n
    else:
        w = [r.uniform(0.3, 1.0) for _ in range(n)]
        new = [1 + int((total - n) * x / sum(w)) for x in w]
        new[0] += total - sum(new)
    cached = [case["cached"]] if n == 1 else [int(case["cached"] * r.uniform(0.6, 1.0)) for _ in range(n)]
    return list(zip(cached, new))


def inv_freq(rd):
    return (1.0 / THETA ** (torch.arange(0, rd, 2, dtype=F64) / rd)).float().to(DEV) if rd else None


def weight_inputs(case, seed):
    src, dt = Source(seed), torch_dtype(case)
    parts = [src.normal(case["N"], case["K"], std=0.02, dtype=torch.bfloat16) for _ in range(2 if case["kind"] == "gated" else 1)]
    return src.normal(case["M"], case["K"], dtype=dt), parts


def qkv_input(case, seed):
    """The rows [q | k | v] that the QKV product leaves: channels of unlike size, as keys have them."""
    src = Source(seed)
    heads = case["nh"] + 2 * case["nkv"]
    size = torch.exp(0.5 * src.normal(heads, case["hd"]))
    return (src.normal(case["tokens"], heads, case["hd"]) * size).reshape(case["tokens"], -1)


def cached_inputs(case, seed):
    """q [T, nh, hd] and, one part of a sequence at a time, (sequence, first position, k, v [n, nkv, hd])."""
    src = Source(seed)
    size = torch.exp(0.5 * src.normal(2, case["nkv"], case["hd"]))
    q = src.normal(case["tokens"], case["nh"], case["hd"]).to(torch_dtype(case))

    def parts():
        for b, (cached, new) in enumerate(counts_of(case)):
            for at in range(0, cached + new, 16384):
                n = min(16384, cached + new - at)
                k, v = (src.normal(n, case["nkv"], case["hd"]) * size[i] for i in range(2))
                yield b, at, k, v
    return q, parts()


# --------------------------------------------------------------------------------------------------------- plain forms
def quantise(x, group):
    """(codes uint8 as x, s, z float32 [..., groups]) of float32 values."""
    g = x.to(F64).unflatten(-1, (-1, group))
    lo, hi = g.amin(-1).clamp(max=0.0), g.amax(-1).clamp(min=0.0)
    m, e = torch.frexp((hi - lo) / torch.full((), 15.0, dtype=F64, device=x.device))
    s = torch.ldexp(torch.ceil(m * 16.0) / 16.0, e)
    s = torch.where(hi - lo < 2.0 ** -100, torch.zeros_like(s), s)
    d = torch.where(s > 0, s, torch.ones_like(s))
    z = torch.round(-lo / d)
    c = (torch.round(g / d.unsqueeze(-1)) + z.unsqueeze(-1)).clamp(0.0, 15.0)
    c = torch.where(s.unsqueeze(-1) > 0, c, torch.zeros_like(c))
    z = torch.where(s > 0, z, torch.zeros_like(z))
    return c.flatten(-2).to(torch.uint8), s.float(), z.float()


def values(codes, s, z):
    g = codes.float().unflatten(-1, (s.shape[-1], -1))
    return (s.unsqueeze(-1) * (g - z.unsqueeze(-1))).flatten(-2)


def rotate(x, positions, freq):
    """x [T, heads, hd] with the first 2·len(freq) dims of every head turned, rounded once to 32 bits."""
    if freq is None:
        return x
    h = freq.numel()
    angle = positions.to(F64)[:, None] * freq.to(F64)
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = x[..., :h].to(F64), x[..., h:2 * h].to(F64)
    return torch.cat([(a * c - b * s).float(), (b * c + a * s).float(), x[..., 2 * h:]], -1)


def plain_linear(state):
    x = state["x"].float()
    y = [x @ values(*w).T for w in state["weights"]]
    if state["case"]["kind"] == "gated":
        y = [y[0] / (1.0 + torch.exp(-y[0])) * y[1]]
    return y[0].to(state["x"].dtype)


def plain_store(state):
    case, dt = state["case"], torch_dtype(state["case"])
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    rows = state["qkv"].view(-1, nh + 2 * nkv, hd)
    qk = rotate(rows[:, :nh + nkv], state["positions"], state["freq"])
    kv = torch.cat([qk[:, nh:], rows[:, nh + nkv:]], 1)
    back = values(*quantise(kv, GROUP)).to(dt)
    return [qk[:, :nh].reshape(-1, nh * hd).to(dt), back[:, :nkv].contiguous(), back[:, nkv:].contiguous()]


def plain_attend(state):
    case, out = state["case"], []
    nh, nkv, hd, window = case["nh"], case["nkv"], case["hd"], case["window"]
    G = nh // nkv
    first = 0
    for (cached, new), (k, v) in zip(counts_of(case), state["cache"]):
        q = state["q"][first:first + new].float().view(new, nkv, G, hd)
        first += new
        key = torch.arange(cached + new, device=DEV)
        pos = cached + torch.arange(new, device=DEV)
        seen = key[None] <= pos[:, None]
        if window:
            seen &= key[None] > pos[:, None] - window
        K, V = values(*k), values(*v)
        o = torch.empty(new, nkv, G, hd, device=DEV)
        for h in range(nkv):
            score = (q[:, h].reshape(new * G, hd) @ K[:, h].T).view(new, G, -1) * (1.0 / math.sqrt(hd))
            score = torch.where(seen[:, None], score, torch.full((), -math.inf, device=DEV))
            p = torch.exp(score - score.amax(-1, keepdim=True))
            o[:, h] = ((p / p.sum(-1, keepdim=True)).view(new * G, -1) @ V[:, h]).view(new, G, hd)
        out.append(o.reshape(new, nh * hd))
    return torch.cat(out).to(torch_dtype(case))


# ------------------------------------------------------------------------------------------------------------ running
def pages_of(case, seed):
    """Every sequence's pages, in an order of their own."""
    need = [-(-(cached + new) // PAGE) for cached, new in counts_of(case)]
    order = list(range(sum(need) + 3))
    random.Random(seed).shuffle(order)
    it = iter(order)
    return len(order), [[next(it) for _ in range(n)] for n in need]


def view_of(pool, tables, entries, before):
    """The step's arrays and the view of the cache that a layer gets, as the engine makes them."""
    from spissa_b200.cache.views import KVLayerView
    from spissa_b200.engine import pack_step
    step = pack_step(entries, before, {"kv": tables}, torch.device(DEV))
    return step, KVLayerView(pool, pool, step.page_tables["kv"], PAGE, step.token_seq, step.positions, step.seq_row, None, True, bits=4)


def prepare(case, seed):
    state = dict(case=case, own=own)
    if case["kind"] in ("linear", "gated"):
        state["x"], parts = weight_inputs(case, seed)
        if not own:
            state["weights"] = [quantise(w.float(), case["group"]) for w in parts]
            return state
        from spissa_b200.parts.linear import GatedLinear4, Linear4
        state["product"] = GatedLinear4(*parts, group=case["group"]) if case["kind"] == "gated" else Linear4(*parts, group=case["group"])
        return state
    counts = counts_of(case)
    if case["kind"] == "store":
        state["qkv"], state["freq"] = qkv_input(case, seed), inv_freq(case["rd"])
        state["positions"] = torch.cat([torch.arange(c, c + n) for c, n in counts]).to(DEV)
        if own:
            from spissa_b200.csrc import lib as K
            n_pages, tables = pages_of(case, seed)
            pool = K.kv4_pool(n_pages, case["nkv"], case["hd"], torch.device(DEV))
            state["step"], state["view"] = view_of(pool, tables, [(b, [0] * n, []) for b, (_, n) in enumerate(counts)], [c for c, _ in counts])
        return state
    state["q"], parts = cached_inputs(case, seed)
    if not own:
        held = [[] for _ in counts]
        for b, _, k, v in parts:
            held[b].append((quantise(k, GROUP), quantise(v, GROUP)))
        state["cache"] = [tuple(tuple(torch.cat([part[i][j] for part in h]) for j in range(3)) for i in range(2)) for h in held]
        return state
    from spissa_b200.csrc import lib as K
    n_pages, tables = pages_of(case, seed)
    pool = K.kv4_pool(n_pages, case["nkv"], case["hd"], torch.device(DEV))
    for b, at, k, v in parts:
        _, view = view_of(pool, [tables[b]], [(b, [0] * k.shape[0], [])], [at])
        K.kv4_store(torch.cat([k, v], 1).reshape(k.shape[0], -1), None, pool, view, None, 0, case["nkv"], case["hd"], 0)
    state["step"], state["view"] = view_of(pool, tables, [(b, [0] * n, []) for b, (_, n) in enumerate(counts)], [c for c, _ in counts])
    state["q"] = state["q"].view(case["tokens"], -1)
    return state


def run(state):
    case = state["case"]
    if not state["own"]:
        return dict(linear=plain_linear, gated=plain_linear, store=plain_store, attend=plain_attend)[case["kind"]](state)
    if case["kind"] == "linear":
        return state["product"](state["x"])
    if case["kind"] == "gated":
        return state["product"](state["x"], state["x"].dtype)
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    if case["kind"] == "store":
        from spissa_b200.csrc import lib as K
        T, view, dt = case["tokens"], state["view"], torch_dtype(case)
        q = torch.empty(T, nh * hd, dtype=dt, device=DEV)
        k, v = (torch.empty(T, nkv, hd, dtype=dt, device=DEV) for _ in range(2))
        K.kv4_store(state["qkv"], q, view.k_pool, view, state["freq"], nh, nkv, hd, case["rd"])
        K.kv4_load(view.k_pool, view, k, v, nkv, hd)
        return [q, k, v]
    from spissa_b200.parts.attention import attend_paged
    return attend_paged(state["q"], state["step"], state["view"], nh, nkv, hd, case["window"] or None, 1.0 / math.sqrt(hd))


# --------------------------------------------------------------------------------------------- the least work of a pass
def work(case):
    eb = 2 if case["dtype"] == "bfloat16" else 4
    if case["kind"] in ("linear", "gated"):
        M, N, K, n = case["M"], case["N"], case["K"], 2 if case["kind"] == "gated" else 1
        return dict(bytes=n * N * K * (0.5 + 2.0 / case["group"]) + eb * M * (K + N),
                    flops=2.0 * n * M * N * K)
    nh, nkv, hd, T = case["nh"], case["nkv"], case["hd"], case["tokens"]
    row = 2 * nkv * hd * (0.5 + 2.0 / GROUP)                          # a position's key and value
    if case["kind"] == "store":
        # the rows of the QKV product in, q and the pages' rows out, and those rows read back
        return dict(bytes=T * ((nh + 2 * nkv) * hd * 4 + nh * hd * eb + 2 * row + 2 * nkv * hd * eb),
                    flops=T * (3.0 * (nh + nkv) * case["rd"] + 8.0 * 2 * nkv * hd))
    keys = pairs = 0
    for cached, new in counts_of(case):
        lowest = max(0, cached + 1 - case["window"]) if case["window"] else 0
        keys += cached + new - lowest
        pairs += sum(min(case["window"] or p + 1, p + 1) for p in range(cached, cached + new))
    return dict(bytes=keys * row + 2 * T * nh * hd * eb, flops=4.0 * pairs * nh * hd)


# ------------------------------------------------------------------------------------------------- the definition again
def nearest_even(d):
    low = torch.floor(d)
    rest = d - low
    odd = torch.remainder(low, 2.0) == 1.0
    return low + ((rest > 0.5) | ((rest == 0.5) & odd)).to(F64)


def stands_for(x, group):
    """What a tensor's numbers become when they are held in four bits, in 64 bits."""
    x = x.to(F64)
    shape = x.shape
    x = x.reshape(-1, group)
    zero = torch.zeros(x.shape[0], 1, dtype=F64, device=x.device)
    low = torch.cat([x, zero], 1).min(1, keepdim=True).values
    span = torch.cat([x, zero], 1).max(1, keepdim=True).values - low
    step = torch.div(span, zero + 15.0)
    unit = torch.exp2(torch.floor(torch.log2(step.clamp(min=2.0 ** -200))) - 3.0)
    s = torch.ceil(step / unit) * unit
    z = nearest_even(-low / s)
    c = torch.minimum(torch.maximum(nearest_even(x / s) + z, zero), zero + 15.0)
    return torch.where(span >= 2.0 ** -100, s * (c - z), zero).reshape(shape)


def exact(case, seed):
    if case["kind"] in ("linear", "gated"):
        x, parts = weight_inputs(case, seed)
        y = [torch.einsum("mk,nk->mn", x.to(F64), stands_for(w, case["group"])) for w in parts]
        return y[0] if len(y) == 1 else y[0] * torch.sigmoid(y[0]) * y[1]
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    if case["kind"] == "store":
        rows = qkv_input(case, seed).view(-1, nh + 2 * nkv, hd).to(F64)
        if case["rd"]:
            half = case["rd"] // 2
            pos = torch.tensor([p for c, n in counts_of(case) for p in range(c, c + n)], dtype=F64, device=DEV)
            angle = torch.outer(pos, inv_freq(case["rd"]).to(F64))
            turned = torch.complex(rows[:, :nh + nkv, :half].contiguous(), rows[:, :nh + nkv, half:2 * half].contiguous()) \
                * torch.polar(torch.ones_like(angle), angle)[:, None]
            rows[:, :nh + nkv, :half], rows[:, :nh + nkv, half:2 * half] = turned.real, turned.imag
        # the rotated keys are 32-bit numbers before they are quantised
        return [rows[:, :nh].reshape(-1, nh * hd), stands_for(rows[:, nh:nh + nkv].float(), GROUP), stands_for(rows[:, nh + nkv:], GROUP)]
    q, parts = cached_inputs(case, seed)
    held = [([], []) for _ in counts_of(case)]
    for b, _, k, v in parts:
        held[b][0].append(stands_for(k, GROUP))
        held[b][1].append(stands_for(v, GROUP))
    out, at = [], 0
    for (cached, new), (k, v) in zip(counts_of(case), held):
        k, v = torch.cat(k), torch.cat(v)
        dist = torch.arange(cached, cached + new, device=DEV)[:, None] - torch.arange(cached + new, device=DEV)[None]
        hidden = dist < 0
        if case["window"]:
            hidden |= dist >= case["window"]
        rows = torch.empty(new, nh, hd, dtype=F64, device=DEV)
        for h in range(nh):
            score = torch.einsum("td,jd->tj", q[at:at + new, h].to(F64), k[:, h * nkv // nh]) / hd ** 0.5
            rows[:, h] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v[:, h * nkv // nh]
        out.append(rows.reshape(new, nh * hd))
        at += new
    return torch.cat(out)
