"""Four bits without a GPU: what is refused, what a cache of four bits asks for, the command line's options."""
import pytest
import torch

from plain import q4_plain as Q
from tiny import TINY_A, TINY_D, TINY_E


def model_of(cfg):
    from spissa_b200 import LlamaConfig
    from spissa_b200.engine.model import Model
    return Model(LlamaConfig.from_dict(cfg).to_spec())


def test_bits_are_4_or_16():
    model = model_of(TINY_E)
    for w, c in ((16, 16), (4, 16), (16, 4), (4, 4)):
        model.check_bits(w, c)
    for w, c in ((8, 16), (16, 3), (0, 4)):
        with pytest.raises(ValueError, match="16 .* or 4"):
            model.check_bits(w, c)


def test_models_with_parts_that_have_no_such_form_are_refused():
    from lazulix_models import CONFIGS
    from spissa_b200.config import config_from_dict
    from spissa_b200.engine.model import Model
    model = Model(config_from_dict(CONFIGS["a"]).to_spec())
    model.check_bits(16, 16)
    for w, c in ((4, 16), (16, 4)):
        with pytest.raises(ValueError, match="no form with"):
            model.check_bits(w, c)


def test_a_subclass_does_not_inherit_the_form():
    from spissa_b200.parts.attention import GQAAttention

    class Other(GQAAttention):
        pass
    model = model_of(TINY_E)
    mixer = model.layers[0].mixer
    mixer.__class__ = Other
    with pytest.raises(ValueError, match="Other has no form with a cache"):
        model.check_bits(16, 4)


def test_head_sizes_and_rotations_a_cache_refuses():
    from spissa_b200.parts import Runtime
    rt = Runtime(torch.device("cpu"), torch.bfloat16, 64, 16, 4)
    for cfg, ok in ((TINY_E, True), (TINY_A, False), (TINY_D, False)):
        mixer = model_of(cfg).layers[0].mixer
        mixer.rt = rt
        if ok:
            assert mixer.cache_request().bits == 4
        else:
            with pytest.raises(ValueError, match="heads of 32, 64, 96, 128"):
                mixer.cache_request()
    mixer = model_of(TINY_E).layers[0].mixer
    mixer.rt = rt
    mixer.position.rotary_dim = 20
    with pytest.raises(ValueError, match="multiple of 8"):
        mixer.cache_request()


def test_pages_of_four_bits():
    from spissa_b200.cache import CacheManager
    from spissa_b200.parts.base import KVCacheRequest
    four, plain = KVCacheRequest(2, 128, bits=4), KVCacheRequest(2, 128)
    m = CacheManager({0: four, 1: plain, 2: four}, 200, 3, 64, torch.bfloat16, "cpu")
    g = m.kv_groups[m.cache_group[0]]
    assert g.k.shape == (2, 4, 2, 64 * (128 + 16)) and g.k.dtype == torch.uint8 and g.v is g.k
    assert g.bytes() == 2 * 4 * 2 * 64 * 144
    assert m.kv_groups[m.cache_group[1]].bytes() == 4 * 2 * 64 * 128 * 2 * 2
    for bad in (dict(bits=8), dict(bits=4, keys_only=True), dict(bits=4, v_head_dim=64)):
        with pytest.raises(ValueError):
            CacheManager({0: KVCacheRequest(2, 128, **bad)}, 200, 3, 64, torch.bfloat16, "cpu")
    with pytest.raises(ValueError):
        CacheManager({0: four}, 200, 3, 32, torch.bfloat16, "cpu")


def test_the_command_line_takes_bits():
    from spissa_b200 import cli
    seen = {}

    def engine(args, n):
        seen.update(weight=args.weight_bits, cache=args.cache_bits)
        raise SystemExit(0)
    old, cli._engine = cli._engine, engine
    try:
        with pytest.raises(SystemExit):
            cli.main(["generate", "nowhere", "--token-ids", "1,2", "--weight-bits", "4", "--cache-bits", "4"])
        assert seen == dict(weight=4, cache=4)
        with pytest.raises(SystemExit):
            cli.main(["generate", "nowhere", "--token-ids", "1,2"])
        assert seen == dict(weight=16, cache=16)
        with pytest.raises(SystemExit):
            cli.main(["generate", "nowhere", "--token-ids", "1,2", "--weight-bits", "8"])
    finally:
        cli._engine = old


def test_packed_shapes_refuse_what_has_no_layout():
    from spissa_b200.csrc.lib import KernelError, kv4_tile_bytes, q4_shapes
    assert q4_shapes(17, 160, 32) == ((2, 2, 1024), (2, 2, 8, 4, 2))
    assert q4_shapes(40, 128, 128, 20) == ((4, 1, 1024), (4, 1, 8, 1, 2))
    for bad in ((16, 100, 32), (16, 96, 64), (16, 64, 16), (0, 64, 64), (16, 64, 64, 7)):
        with pytest.raises(KernelError):
            q4_shapes(*bad)
    assert kv4_tile_bytes(64) == 64 * 72
    for hd in (16, 48, 160, 256):
        with pytest.raises(KernelError):
            kv4_tile_bytes(hd)


def test_the_plain_statement_of_the_format():
    """Properties that follow from the definition: every number is a bfloat16, s covers the range with at most an eighth to spare,
    so a number is off by at most half a step, half the range / 15 · 9/8."""
    x = torch.randn(64, 32, generator=torch.Generator().manual_seed(3)) * torch.exp(torch.randn(64, 1, generator=torch.Generator().manual_seed(4)) * 3)
    y = Q.q4(x, 32)
    assert torch.equal(y, y.to(torch.bfloat16).double())
    reach = x.double().amax(1).clamp(min=0) - x.double().amin(1).clamp(max=0)
    # z is rounded too, so an end of the range may be cut by half a step on top of the half step of its code
    assert bool(((y - x.double()).abs().amax(1) <= reach / 15 * 9 / 8).all())


def test_a_split_of_the_keys_covers_them():
    from spissa_b200.csrc.lib import kv4_attend_plan
    for n_seqs, nkv, hd, cols in ((1, 8, 64, 4), (64, 8, 128, 4), (3, 8, 128, 4), (1, 8, 128, 160), (200, 2, 96, 3), (5, 1, 32, 33)):
        for pages in (1, 2, 5, 33, 64, 641, 2000):
            nt, each, n = kv4_attend_plan(n_seqs, nkv, hd, cols, pages)
            assert nt in (1, 2) and n >= 1 and each * n >= pages > each * (n - 1)


@pytest.mark.parametrize("weight_bits,cache_bits,more", [(16, 16, set()), (4, 16, {"q4", "q4_tc"}), (16, 4, {"kv4", "kv4_attention"}),
                                                         (4, 4, {"q4", "q4_tc", "kv4", "kv4_attention"})])
def test_the_libraries_are_asked_for_before_the_weights_are_read(weight_bits, cache_bits, more, monkeypatch, tmp_path):
    import json

    from spissa_b200.engine import engine as E
    (tmp_path / "config.json").write_text(json.dumps(TINY_E))
    asked = []
    monkeypatch.setattr(E, "_require_gpu", lambda device: torch.device("cpu"))
    monkeypatch.setattr(E.kernel_build, "prefetch", lambda names: asked.append(set(names)))

    def read(*args):
        raise InterruptedError
    monkeypatch.setattr(E, "load_tensors", read)
    with pytest.raises(InterruptedError):
        E.Engine.from_folder(tmp_path, weight_bits=weight_bits, cache_bits=cache_bits)
    assert len(asked) == 1 and asked[0] & {"q4", "q4_tc", "kv4", "kv4_attention"} == more and "generic" in asked[0]


def test_which_prompt_steps_read_the_codes():
    """Those whose tiles of sixteen query columns find room at once, whatever the head's size; and short ones."""
    from spissa_b200.csrc.lib import kv4_room
    from spissa_b200.parts.attention import reads_codes

    def takes(T, n_seqs, max_new, nh, nkv, hd):
        return reads_codes(torch.empty(T, 1, dtype=torch.bfloat16), max_new * (nh // nkv), nkv, hd, n_seqs)
    assert kv4_room(32) == kv4_room(64) > kv4_room(96) == kv4_room(128)
    for T, nh, nkv, hd, want in ((255, 32, 8, 128, True), (256, 32, 8, 128, False), (256, 16, 1, 128, True), (512, 16, 1, 128, False),
                                 (512, 9, 3, 96, True), (1024, 9, 3, 96, False), (384, 12, 12, 96, True), (512, 12, 12, 96, False),
                                 (1024, 6, 2, 32, True), (384, 16, 4, 32, True), (512, 16, 4, 32, False), (256, 32, 8, 64, False)):
        assert takes(T, 1, T, nh, nkv, hd) is want, (T, nh, nkv, hd)
    assert takes(1024, 64, 24, 32, 8, 128) and not takes(2048, 16, 128, 32, 8, 128) and not takes(2000, 3, 900, 32, 8, 128)


def test_rows_are_copied_only_where_a_kernel_does_not_take_them():
    from spissa_b200.parts.linear import on_boundaries
    for dtype, entries, kept in ((torch.bfloat16, 8, (0, 8, 16)), (torch.bfloat16, 0, (0, 8, 16)), (torch.float32, 8, (0, 8, 16)), (torch.float32, 0, (0, 4, 8, 12))):
        wide = torch.zeros(5, 96, dtype=dtype)
        wide = wide[:, (-wide.data_ptr() // wide.element_size()) % 16:][:, :80]
        for at in range(17):
            rows = wide[:, at:at + 64]
            assert (on_boundaries(rows, entries) is rows) == (at in kept or at % 16 == 0), (dtype, entries, at)
    row = torch.zeros(1, 64)
    assert on_boundaries(row.expand(5, 64)).is_contiguous() and on_boundaries(row) is row
