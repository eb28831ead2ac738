"""The greedy choice over logits that are not numbers."""
import numpy as np
import pytest

from gpu_util import Dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", ["one", "two", "all", "behind", "infinities", "lowest"])
def test_argmax_of_logits_that_are_not_numbers(hv, case):
    """np.argmax's order: the first NaN, whatever else there is; a token in any case, whose row the
    next step reads."""
    n = 5003
    x = np.random.default_rng(3).standard_normal(n).astype(np.float32)
    if case == "one":
        x[1234] = np.nan
    if case == "two":
        x[[40, 4999]] = np.nan
    if case == "all":
        x[:] = np.nan
    if case == "behind":
        x[17], x[-1] = np.inf, np.nan
    if case == "infinities":
        x[:] = -np.inf
        x[[7, 9]] = np.inf
    if case == "lowest":
        x[:] = -np.inf
    pv, pi = Dev(nbytes=128 * 4), Dev(nbytes=128 * 4)
    tok, step, pos, gen = (Dev(np.zeros(4, np.int32)) for _ in range(4))
    hv.argmax_partial(Dev(x), pv, pi, n, 128)
    hv.argmax_final(pv, pi, tok, gen, step, pos, 128)
    assert tok.get(np.int32)[0] == gen.get(np.int32)[0] == np.argmax(x)


@pytest.mark.parametrize("fused,kv", [(True, "f32"), (True, "f16"), (False, "f32"), (False, "q8")])
def test_engine_whose_logits_are_not_numbers(hv, fused, kv):
    """Token 0 at every step, and an engine that goes on (the next step reads the token's row)."""
    import limited
    import synth
    import w4format
    cfg = w4format.Config(synth.tiny_arch())

    def tensors():
        for name, x in synth.iter_tensors(cfg, 8):
            yield name, np.full_like(x, np.nan) if name == "model.norm.weight" else x
    e = limited.Engine(config=cfg, tensors=tensors(), quiet=True, max_context=64, kv_dtype=kv,
                       fused=fused)
    try:
        ids = synth.prompt_ids(cfg, 8, 9)
        assert np.isnan(e.logits(ids)).all()
        for graph in (False, True):
            assert e.generate(ids, 6, stop_on_eos=False, use_graph=graph)[0] == [0] * 6
    finally:
        e.free()
