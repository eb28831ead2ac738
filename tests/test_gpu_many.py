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


def means(q, pk, pv, plen, tk, tv, rows, tails, scale):
    """Contexts of rows [sum(rows), nq, 128] in 64 bits, a sequence's rows of a head together."""
    out = np.empty(q.shape)
    nkv, group, r0 = tk.shape[1], q.shape[1] // tk.shape[1], 0
    for s, (r, t) in enumerate(zip(rows, tails)):
        hidden = plen + np.arange(t)[None] > plen + t - r + np.arange(r)[:, None]
        hidden = np.concatenate([np.zeros((r, plen), bool), hidden], 1)
        for h in range(q.shape[1]):
            k, v = (np.concatenate([a[h // group, :plen], b[s, h // group, :t]]).astype(np.float64)
                    for a, b in ((pk, tk), (pv, tv)))
            x = np.where(hidden, -np.inf, (q[r0:r0 + r, h].astype(np.float64) @ k.T) * scale)
            w = np.exp(x - x.max(1, keepdims=True))
            out[r0:r0 + r, h] = (w @ v) / w.sum(1, keepdims=True)
        r0 += r
    return out


@pytest.mark.parametrize("pcap,nkv,group,rows,tails", [
    # chunks of a whole tail: many places for a prefix leave one, and many rows do
    (1 << 20, 1, 1, [1] * 8, [30000, 1, 29999, 4097, 1, 63, 16000, 30000]),
    (1 << 20, 1, 4, [1] * 8, [30000, 1, 29999, 4097, 1, 63, 16000, 30000]),
    (64, 8, 1, [100, 90], [12000, 11000]),
    (64, 1, 1, [1], [30000]), (64, 1, 8, [1, 1], [30000, 29000])])
def test_long_tails(hv, pcap, nkv, group, rows, tails):
    """Values of one sign under weights that hardly differ: sums that grow at every step. Their errors,
    with u = 2^-24: a step's products are summed by the tensor pipe, which may cut (4 u); weights
    and their terms are rounded, and so is every addition to what the steps before gave, so that
    over the values of a long tail those have no direction: sqrt(steps) u of a value, less than u
    of the mean of a hundred and more. 16 u covers the mean; sums that are cut at every one of
    some hundred steps are off by about as many u, all one way."""
    import span_ref as R
    from test_gpu_shared import run_shared, near, SCALE
    g = np.random.default_rng(len(rows))
    f16 = lambda n, a: (a + g.random((n, 128), np.float32) if a else g.standard_normal((n, 128), np.float32))  # noqa: E731
    nseq, tcap, plen = len(rows), max(tails), 40
    pk, pv = np.zeros((2, nkv, pcap, 128), np.float16)
    tk = np.zeros((nseq, nkv, tcap, 128), np.float16)
    tv = np.zeros_like(tk)
    for h in range(nkv):
        pk[h, :plen], pv[h, :plen] = f16(plen, 0), f16(plen, 1)
        for s, n in enumerate(tails):
            tk[s, h, :n], tv[s, h, :n] = f16(n, 0), f16(n, 1)
    q = (0.2 * g.standard_normal((sum(rows), nkv * group, 128))).astype(np.float32)
    row0 = np.concatenate([[0], np.cumsum(rows)])
    got = run_shared(hv, q, pk, pv, plen, tk, tv, row0, tails)
    want = means(q, pk, pv, plen, tk, tv, rows, tails, SCALE)
    off = (got - want) / want
    for s in np.flatnonzero(np.array(tails) > 10000):
        mean = off[row0[s]:row0[s + 1]].mean()
        print(tails[s], "positions: mean error", mean, "largest", np.abs(off[row0[s]:row0[s + 1]]).max())
        assert abs(mean) <= 16 * R.U
    n = max(tails) + plen
    big = SCALE * (np.abs(q).max() * np.abs(tk).max(initial=0).astype(np.float64)) * 128     # over any score
    near(got, want, (96 * R.U * big + (n / 8 + 64) * R.U) * want)
