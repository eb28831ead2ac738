"""Many continuations of one prompt: what a call gives does not depend on the calls before it."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_results_do_not_depend_on_larger_calls_before(hv):
    import limited
    import synth
    import w4format
    cfg = w4format.Config(synth.tiny_arch(hidden=512, n_head=8, n_kv=2))
    make = lambda: limited.Engine(config=cfg, tensors=synth.iter_tensors(cfg, 8), quiet=True,  # noqa: E731
                                  max_context=3000, kv_dtype="f16")
    a, b = make(), make()
    try:
        ids = synth.prompt_ids(cfg, 8, 700)
        g = np.random.default_rng(8)
        text = lambda n: g.integers(0, cfg.vocab, n).tolist()  # noqa: E731
        few, long, many = [text(n) for n in (9, 4, 1, 8)], [text(2000), text(3)], [text(5)] * 200
        hidden = lambda e, m: e._download(e._pf["h"], (m, cfg.hidden), np.uint32)  # noqa: E731

        def short(e):
            s = e.score_many(ids, few)
            h = hidden(e, sum(map(len, few)))
            toks = e.generate_many(ids, few, 6, stop_on_eos=False)
            return [x[k].view(np.uint32) for x in s for k in ("logprob", "entropy")] + [h, hidden(e, 4)], toks
        want, toks = short(a)
        for before in (long, many, long + many[:3]):
            b.score_many(ids, before)
            got, t = short(b)
            assert t == toks
            assert all(np.array_equal(x, y) for x, y in zip(got, want))
    finally:
        a.free()
        b.free()
