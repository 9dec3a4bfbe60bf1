"""A step over a cache of four bits is a transaction too: it fails on the host (a status word is written, a forward pass raises), is
repeated, and leaves the pages and logits of a run that nothing disturbed."""
import pytest
import torch

from spissa_b200.csrc import lib as K
from spissa_b200.csrc.lib import KernelError
from test_four_bits_engine_gpu import DEV, SMALL, cached, engine_of, tokens, weights_of

pytestmark = pytest.mark.gpu


def books(engine):
    return ({s: (q.length, {n: list(p) for n, p in q.pages.items()}) for s, q in engine.cache.seqs.items()},
            {n: g.pages.free_count for n, g in engine.cache.kv_groups.items()}, engine.cache.slots.free_count)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_failed_step_is_undone_and_its_repetition_is_the_undisturbed_run(dtype, monkeypatch):
    weights, ids = weights_of(SMALL, 33), tokens(140, 4)
    parts = [ids[:60], ids[60:66], ids[66:139], ids[139:]]           # within a page, across its end, over two pages, a decode step
    calm, engine = (engine_of(SMALL, weights, dtype, 4, 4) for _ in range(2))
    slot, other = calm.acquire(), engine.acquire()
    want = [calm.step([(slot, p, list(range(len(p))))]) for p in parts]
    for i, part in enumerate(parts):
        before = books(engine)
        K.status_word(DEV).fill_(172)                                # as if a kernel had given up a wait
        with pytest.raises(KernelError, match="code 172: kv4_attention"):
            engine.step([(other, part, [0])])
        assert books(engine) == before
        engine.cache.check()
        down = engine.model.layers[1].ffn

        def fails(*args, **kw):
            raise InterruptedError("in the middle of a step")
        if len(part) > 1:                                            # (a decode step is a graph: no host code runs within it)
            with monkeypatch.context() as m:
                m.setattr(type(down), "forward", fails)
                with pytest.raises(InterruptedError):
                    engine.step([(other, part, [0])])
            assert books(engine) == before
            engine.cache.check()
        got = engine.step([(other, part, list(range(len(part))))])
        assert torch.equal(got, want[i])
    for layer in range(SMALL["num_hidden_layers"]):
        for a, b in zip(cached(calm, slot, 140, layer), cached(engine, other, 140, layer)):
            assert torch.equal(a, b)
    engine.release(other)
    engine.cache.check()
