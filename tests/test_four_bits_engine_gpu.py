"""A Llama with weights and cache of four bits, through the engine: against plain 64-bit arithmetic over the same numbers, whole
prompts against prompts in pieces and single tokens, captured decode steps against direct ones."""
import json

import pytest
import torch

from plain import llama_plain as P
from plain import q4_plain as Q

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

SMALL = dict(architectures=["LlamaForCausalLM"], model_type="llama", num_hidden_layers=2, hidden_size=192, num_attention_heads=6,
             num_key_value_heads=2, head_dim=64, intermediate_size=320, vocab_size=500, rope_theta=10000.0, rope_scaling=None,
             tie_word_embeddings=True, rms_norm_eps=1e-5, max_position_embeddings=2048)
WIDE = dict(SMALL, hidden_size=160, num_attention_heads=10, num_key_value_heads=1, head_dim=128, intermediate_size=96, num_hidden_layers=1,
            tie_word_embeddings=False)


def weights_of(cfg, seed):
    gen = torch.Generator().manual_seed(seed)
    H, I, hd, nh, nkv = (cfg[k] for k in ("hidden_size", "intermediate_size", "head_dim", "num_attention_heads", "num_key_value_heads"))
    def mat(*s):
        return (torch.randn(*s, generator=gen) * 0.08).to(torch.bfloat16)
    t = {"model.embed_tokens.weight": mat(cfg["vocab_size"], H), "model.norm.weight": 1 + mat(H)}
    for i in range(cfg["num_hidden_layers"]):
        p = f"model.layers.{i}."
        for name, shape in (("self_attn.q_proj", (nh * hd, H)), ("self_attn.k_proj", (nkv * hd, H)), ("self_attn.v_proj", (nkv * hd, H)),
                            ("self_attn.o_proj", (H, nh * hd)), ("mlp.gate_proj", (I, H)), ("mlp.up_proj", (I, H)), ("mlp.down_proj", (H, I))):
            t[p + name + ".weight"] = mat(*shape)
        for name in ("input_layernorm", "post_attention_layernorm"):
            t[p + name + ".weight"] = 1 + mat(H)
    if not cfg["tie_word_embeddings"]:
        t["lm_head.weight"] = mat(cfg["vocab_size"], H)
    return t


def held(weights):
    """What the layers' matrices become in four bits."""
    return {k: Q.q4(v, 64 if v.shape[1] % 64 == 0 else 32) if "_proj" in k else v for k, v in weights.items()}


def engine_of(cfg, weights, dtype, weight_bits, cache_bits, **kw):
    from spissa_b200 import Engine, LlamaConfig
    t = {k: v.to(DEV).to(torch.float32 if dtype == "float32" else v.dtype) for k, v in weights.items()}
    return Engine(LlamaConfig.from_dict(cfg), t, dtype, 4096, 8, DEV, weight_bits=weight_bits, cache_bits=cache_bits, **kw)


def tokens(n, seed, vocab=500):
    return [(seed * 7919 + i * i * 31 + i * 17) % vocab for i in range(n)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("cfg", [SMALL, WIDE], ids=["small", "wide"])
def test_weights_of_four_bits_give_the_plain_models_logits(cfg, dtype):
    weights = weights_of(cfg, 5)
    engine = engine_of(cfg, weights, dtype, 4, 16)
    for n in (3, 20, 90):
        ids = tokens(n, n)
        want = P.model_logits(cfg, held(weights), ids)
        slot = engine.acquire()
        got = engine.step([(slot, ids[:-1], list(range(n - 1)))])
        last = engine.step([(slot, ids[-1:], [0])])
        engine.release(slot)
        # float32: sums of up to 320 terms off by 2^-23 each, through 2 layers; bfloat16: the tolerance of the 16-bit model's tests
        tol = (2e-4 if dtype == "float32" else 3e-2) * float(want.abs().max())
        assert float((torch.cat([got, last]).cpu().double() - want).abs().max()) <= tol


def cached(engine, slot, n, cache_id):
    """What the pages hold of a sequence's first ``n`` positions: k, v [n, kv heads, head size] float64."""
    from spissa_b200.csrc import lib as K
    from spissa_b200.engine import pack_step
    g = engine.cache.kv_groups[engine.cache.cache_group[cache_id]]
    step = pack_step([(slot, [0] * n, [])], [0], {g.name: [engine.cache.seqs[slot].pages[g.name]]}, torch.device(DEV))
    view = engine.cache.view(cache_id, step, False)
    assert view.bits == 4
    nkv, hd = g.request.num_kv_heads, g.request.head_dim
    k, v = (torch.empty(n, nkv, hd, device=DEV) for _ in range(2))
    K.kv4_load(view.k_pool, view, k, v, nkv, hd)
    return k.cpu().double(), v.cpu().double()


def plain_logits(cfg, weights, ids, caches):
    """The plain model over keys and values taken from ``caches`` [layer] -> (k, v); and the keys and values it would have stored."""
    n = P.config_numbers(cfg)
    w = {k: v.double() for k, v in weights.items()}
    freq = P.rope_inv_freq(n["theta"], n["hd"], n["scaling"], dtype=torch.float32)
    nh, nkv, hd = cfg["num_attention_heads"], cfg["num_key_value_heads"], cfg["head_dim"]
    h, pos, stored = P.embedding(w["model.embed_tokens.weight"], ids), torch.arange(len(ids)), []
    for i in range(n["L"]):
        p = f"model.layers.{i}."
        x = P.rms_norm(h, w[p + "input_layernorm.weight"], n["eps"])
        q, k, v = (P.linear(x, w[p + f"self_attn.{c}_proj.weight"]).reshape(len(ids), -1, hd) for c in "qkv")
        angle = pos.double()[:, None] * freq.double()
        c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
        def turn(t):
            a, b = t[..., :hd // 2], t[..., hd // 2:]
            return torch.cat([a * c - b * s, b * c + a * s], -1)
        q, k = turn(q), turn(k)
        stored.append((k, v))
        kh, vh = caches[i]
        o = Q.attention(q, kh, vh, 0, hd ** -0.5).reshape(len(ids), nh * hd)
        h = h + P.linear(o, w[p + "self_attn.o_proj.weight"])
        h = h + P.swiglu(P.rms_norm(h, w[p + "post_attention_layernorm.weight"], n["eps"]), w, p + "mlp.")
    h = P.rms_norm(h, w["model.norm.weight"], n["eps"])
    return P.linear(h, w["lm_head.weight"] if "lm_head.weight" in w else w["model.embed_tokens.weight"]), stored


@pytest.mark.parametrize("weight_bits", [16, 4])
@pytest.mark.parametrize("cfg", [SMALL, WIDE], ids=["small", "wide"])
def test_a_cache_of_four_bits_holds_the_plain_models_keys_and_values_and_is_read_as_it_is(cfg, weight_bits):
    weights = weights_of(cfg, 9)
    engine = engine_of(cfg, weights, "float32", weight_bits, 4)
    pw = held(weights) if weight_bits == 4 else weights
    for n, cut in ((6, 5), (150, 149), (150, 100)):
        ids = tokens(n, n + 1)
        slot = engine.acquire()
        got = torch.cat([engine.step([(slot, ids[:cut], list(range(cut)))])] +
                        [engine.step([(slot, part, list(range(len(part))))]) for part in ([ids[cut:]] if n - cut < 8 else [ids[cut:cut + 40], ids[cut + 40:]])])
        caches = [cached(engine, slot, n, i) for i in range(cfg["num_hidden_layers"])]
        engine.release(slot)
        want, stored = plain_logits(cfg, pw, ids, caches)
        assert float((got.cpu().double() - want).abs().max()) <= 2e-4 * float(want.abs().max())
        for (k, v), (pk, pv) in zip(caches, stored):
            for have, real in ((k, pk), (v, pv)):
                g = real.reshape(-1, 32)
                step = (g.amax(1).clamp(min=0) - g.amin(1).clamp(max=0)) / 15 * 9 / 8
                # half a step of its own, half of the zero's, and the products' own error
                assert bool(((have.reshape(-1, 32) - g).abs().amax(1) <= 1.001 * step + 1e-4 * float(real.abs().max())).all())


@pytest.mark.parametrize("weight_bits,cache_bits", [(4, 4), (16, 4), (4, 16)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generation_is_the_same_with_graphs_without_and_one_by_one(dtype, weight_bits, cache_bits):
    from spissa_b200 import SamplingParams
    weights = weights_of(SMALL, 21)
    prompts = [tokens(n, n) for n in (1, 7, 70, 130)]
    runs = []
    for graphs in (True, False):
        engine = engine_of(SMALL, weights, dtype, weight_bits, cache_bits, use_graphs=graphs)
        runs.append([r.tokens for r in engine.generate(prompts, 24, SamplingParams(), stop_ids=[])[0]])
        engine.cache.check()
    assert runs[0] == runs[1] and all(len(t) == 24 for t in runs[0])
    again = [r.tokens for r in engine.generate(prompts, 24, SamplingParams(), stop_ids=[])[0]]
    assert again == runs[0]


def test_a_window_over_four_bits_returns_its_pages_and_sees_the_same_keys():
    """A windowed layer of the same part: long sequences hand pages back, and what is left gives the same outputs as pages of a fresh cache."""
    from spissa_b200.cache import CacheManager
    from spissa_b200.csrc import lib as K
    from spissa_b200.engine import pack_step
    from spissa_b200.parts.attention import attend_paged
    from spissa_b200.parts.base import KVCacheRequest
    nh, nkv, hd, window, n = 4, 2, 64, 100, 400
    m = CacheManager({0: KVCacheRequest(nkv, hd, window, bits=4)}, 64 * 12, 2, 64, torch.bfloat16, torch.device(DEV))
    gen = torch.Generator(device=DEV).manual_seed(1)
    rows = torch.randn(n, (nh + 2 * nkv) * hd, device=DEV, generator=gen)
    slot, outs = m.acquire(), []
    for a in range(0, n, 50):
        res = m.reserve([(slot, 50)])
        step = pack_step([(slot, [0] * 50, [])], [a], res.tables, torch.device(DEV))
        view = m.view(0, step, True)
        q = torch.empty(50, nh * hd, dtype=torch.bfloat16, device=DEV)
        K.kv4_store(rows[a:a + 50], q, view.k_pool, view, None, nh, nkv, hd, 0)
        outs.append(attend_paged(q, step, view, nh, nkv, hd, window, 0.125))
        m.commit(res)
    m.check()
    assert m.kv_groups[m.cache_group[0]].pages.free_count >= 12 - 4
    k, v = (Q.q4(rows.cpu()[:, (nh + i * nkv) * hd:(nh + (i + 1) * nkv) * hd].reshape(n, nkv, hd), 32) for i in range(2))
    want = Q.attention(rows.cpu()[:, :nh * hd].to(torch.bfloat16).reshape(n, nh, hd), k, v, 0, 0.125, window).reshape(n, -1)
    mag = Q.attention(rows.cpu()[:, :nh * hd].to(torch.bfloat16).reshape(n, nh, hd), k, v.abs(), 0, 0.125, window).reshape(n, -1)
    # probabilities and outputs rounded to bfloat16, 2^-8 each; scores in 32 bits
    assert bool(((torch.cat(outs).cpu().double() - want).abs() <= 2.0 ** -8 * (mag + want.abs()) + 1e-3 * mag).all())


def test_sizes_the_engine_refuses():
    weights = weights_of(SMALL, 1)
    from spissa_b200.csrc.lib import KernelError
    with pytest.raises(ValueError, match="4, got 8"):
        engine_of(SMALL, weights, "bfloat16", 8, 16)
    odd = dict(SMALL, hidden_size=200)
    with pytest.raises(KernelError, match="multiple of 32"):
        engine_of(odd, weights_of(odd, 1), "bfloat16", 4, 16)
    small = dict(SMALL, head_dim=16)
    with pytest.raises(ValueError, match="heads of 32"):
        engine_of(small, weights_of(small, 1), "bfloat16", 16, 4)


def test_the_command_generates_with_four_bits(tmp_path, capsys):
    from spissa_b200 import cli
    cfg = tmp_path / "config.json"
    cfg.write_text(json.dumps(SMALL))
    assert cli.main(["generate", "--random", str(cfg), "--token-ids", "1,2,3", "--token-ids", "9", "--max-new-tokens", "5", "--ctx", "128",
                     "--weight-bits", "4", "--cache-bits", "4"]) == 0
    lines = [json.loads(x) for x in capsys.readouterr().out.splitlines() if x.startswith("{")]
    assert [len(x["tokens"]) for x in lines] == [5, 5]
