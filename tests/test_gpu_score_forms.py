"""Engine.score() over every form of the engine: the caches, either prefill, both arrangements of
the weights, generation after it, and alternatives that grow from call to call."""
import numpy as np
import pytest

import limited
import synth
import w4format
from gpu_util import bits
from test_gpu_logprob import check

pytestmark = pytest.mark.gpu


def engine(**kw):
    cfg = w4format.Config(synth.tiny_arch())
    kw.setdefault("fused", kw.get("kv_dtype") != "q8")
    return limited.Engine(config=cfg, tensors=synth.iter_tensors(cfg, 8), quiet=True,
                          max_context=320, **kw)


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
def test_score_does_not_depend_on_the_engines_form(hv, kv):
    """The same bits with either prefill, weight arrangement and step; over the f32 and binary16
    caches against log softmax of the engine's own logits, which are the same in any run."""
    want = None
    forms = [dict(prefill=p, gemv_layout=g) for p in ("batched", "steps") for g in ("pp", "dq")]
    if kv != "q8":
        forms.append(dict(fused=False, prefill="steps"))
    for form in forms:
        e = engine(kv_dtype=kv, **form)
        try:
            ids = synth.prompt_ids(e.cfg, 8, 290)
            before = e.generate(ids[:40], 20, stop_on_eos=False)[0]
            got = e.score(ids, top=3)
            if want is None:
                want = got
            for key in want:
                assert np.array_equal(bits(got[key]), bits(want[key])), (form, key)
            if kv != "q8":
                for i in (0, 100, 288):
                    row = [got[k][i:i + 1] for k in ("logprob", "entropy", "top_ids",
                                                     "top_logprobs")]
                    check(row, e.logits(ids[:i + 1])[None], np.array([ids[i + 1]]), 3)
            assert e.generate(ids[:40], 20, stop_on_eos=False)[0] == before
            graph = e.generate(ids[:40], 20, stop_on_eos=False, use_graph=True)[0]
            e.score(ids[:10])
            assert e.generate(ids[:40], 20, stop_on_eos=False, use_graph=True)[0] == graph == before
        finally:
            e.free()


def test_alternatives_that_grow_take_no_further_memory(hv):
    e = engine(prefill="batched")
    try:
        ids = synth.prompt_ids(e.cfg, 9, 270)
        first = e.score(ids, top=2)
        held = len(e._buffers)
        whole = e.score(ids, top=32)
        for top in (0, 3, 7, 32, 1):
            got = e.score(ids, top=top)
            assert np.array_equal(got["top_ids"], whole["top_ids"][:, :top])
            assert np.array_equal(bits(got["top_logprobs"]), bits(whole["top_logprobs"][:, :top].copy()))
            assert np.array_equal(bits(got["logprob"]), bits(first["logprob"]))
        assert len(e._buffers) == held
    finally:
        e.free()
