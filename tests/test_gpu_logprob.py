"""Scoring on a B200: hv_logprob_rows against 64-bit log softmax, and Engine.score()."""
import numpy as np
import pytest

import synth
import w4format
from gpu_util import Dev, bits

pytestmark = pytest.mark.gpu
F32 = np.float32
U = 2.0 ** -24


def call(hv, x, tok, top, ld=None, scratch=None):
    rows, n = x.shape
    ld = n if ld is None else ld
    wide = np.full((rows, ld), np.nan, F32)
    wide[:, :n] = x
    lp, ent = Dev(nbytes=rows * 4), Dev(nbytes=rows * 4)
    ids = Dev(np.full((rows, max(top, 1)), -7, np.int32))
    alt = Dev(nbytes=rows * max(top, 1) * 4)
    s = scratch or Dev(nbytes=hv.logprob_scratch(rows, n, top))
    hv.logprob_rows(Dev(wide), ld, rows, n, Dev(np.asarray(tok, np.int32)), top, lp, ent, ids,
                    alt, s)
    return (lp.get(F32), ent.get(F32), ids.get(np.int32)[:rows * top].reshape(rows, top),
            alt.get(F32)[:rows * top].reshape(rows, top))


def reference(x, tok, top):
    """64 bits. The sum of the weights other than the largest, S, and each log p, entropy."""
    z = x.astype(np.float64)
    a = z.argmax(1)
    z = z - z.max(1, keepdims=True)
    e = np.exp(z)
    rest = e.copy()
    rest[np.arange(len(x)), a] = 0
    S = rest.sum(1)
    ls = np.log1p(S)
    with np.errstate(invalid="ignore"):
        T = np.where(e > 0, -z * e, 0).sum(1)
    logp = z - ls[:, None]
    order = np.argsort(-np.where(x == 0, 0, x), axis=1, kind="stable")[:, :top]
    return (logp[np.arange(len(x)), tok], ls + T / (1 + S), order,
            np.take_along_axis(logp, order, 1), S)


def check(got, x, tok, top):
    """z = x - m is rounded once (u |z|). A weight 2^(z log2 e): the exponent is off by 2u of
    itself, so the weight by 1.4 * 2u |z| + 8u; weights count for |z| < 104, and those with
    |z| > 30 are below 1e-13 of the largest, so 100u covers them. A running sum of n weights
    in chains of n / 256 and their joining: (n / 256 + 64) u. log1p: 4u. A weight below f32's
    normal range has no relative precision and may count as 0: each of the n is then off by at
    most 2^-126, and its term of the entropy by |z| < 128 times that."""
    lp, ent, order, alt, S = reference(x, tok, top)
    rel = (x.shape[1] / 256 + 164) * U
    tiny = x.shape[1] * 2.0 ** -126
    near = rel * S / (1 + S) + 4 * U * np.log1p(S) + tiny
    with np.errstate(invalid="ignore"):
        for g, w, t in ((got[0], lp, near + 4 * U * np.abs(lp)),
                        (got[1], ent, 2 * (rel + 8 * U) * ent + 129 * tiny),
                        (got[3], alt, near[:, None] + 4 * U * np.abs(alt))):
            ok = (np.abs(g.astype(np.float64) - w) <= t) | (g == w)
            assert ok.all(), (g[~ok][:4], np.broadcast_to(w, g.shape)[~ok][:4])
    assert np.array_equal(got[2], order)


@pytest.mark.parametrize("rows,n,top,ld", [
    (1, 1, 1, 1), (2, 2, 0, 2), (3, 5, 5, 9), (1, 31, 20, 31), (7, 33, 32, 40), (4, 1000, 1, 1000),
    (2, 1023, 20, 1025), (5, 4097, 32, 4097), (1, 151936, 20, 151936), (300, 2049, 3, 2052),
    (9, 151936, 5, 151937), (2, 70001, 32, 70001)])
def test_rows_of_logits(hv, rows, n, top, ld):
    g = np.random.default_rng(n + rows)
    x = (g.standard_normal((rows, n)) * g.choice([0.01, 2.5, 20.0], (rows, 1))).astype(F32)
    tok = g.integers(0, n, rows)
    tok[0] = x[0].argmax()
    check(call(hv, x, tok, top, ld), x, tok, top)


def test_ties_go_to_the_lower_id(hv):
    g = np.random.default_rng(1)
    x = g.integers(-3, 3, (6, 5000)).astype(F32)              # thousands of equal values
    x[1] = 2.0
    x[2, ::2] = -0.0
    x[2, 1::2] = 0.0
    x[3] = np.sort(x[3])
    x[4] = np.sort(x[4])[::-1]
    check(call(hv, x, [0] * 6, 32), x, np.zeros(6, int), 32)


def test_nearly_certain_rows_keep_their_precision(hv):
    x = np.full((4, 3001), -40, F32)
    x[0, 17], x[1, 0], x[2, 3000] = 0, 60, 20
    x[3] = -30
    x[3, 1500] = -5
    tok = [17, 5, 3000, 1500]
    check(call(hv, x, tok, 3), x, np.array(tok), 3)


def test_tokens_that_cannot_occur(hv):
    g = np.random.default_rng(2)
    x = g.standard_normal((4, 2000)).astype(F32)
    x[0, 100:] = -np.inf
    x[1, 1:] = -np.inf                                        # certain: entropy 0
    x[2, :1999] = -np.inf
    x[3, ::2] = np.finfo(F32).min
    tok = np.array([50, 0, 1999, 1])
    got = call(hv, x, tok, 20)
    check(got, x, tok, 20)
    assert got[0][1] == 0 and got[1][1] == 0 and got[1][2] == 0
    assert call(hv, x, [500, 1, 2, 3], 0)[0][0] == -np.inf


def test_rows_without_a_distribution(hv):
    g = np.random.default_rng(3)
    x = g.standard_normal((5, 1500)).astype(F32)
    x[0, 700] = np.nan
    x[1, 3] = np.inf
    x[2] = -np.inf
    x[3, [9, 1400]] = np.nan
    lp, ent, ids, alt = call(hv, x, [1, 2, 3, 4, 5], 4)
    assert np.isnan(lp[:4]).all() and np.isnan(ent[:4]).all() and np.isnan(alt[:4]).all()
    assert np.isfinite(lp[4]) and np.isfinite(ent[4]) and np.isfinite(alt[4]).all()
    assert ids[0, 0] == 700 and ids[1, 0] == 3 and ids[3, :2].tolist() == [9, 1400]
    assert ids[2].tolist() == [0, 1, 2, 3]
    assert ids[0, 1] == np.nanargmax(x[0])


def test_given_tokens_outside_the_vocabulary(hv):
    x = np.random.default_rng(4).standard_normal((4, 100)).astype(F32)
    lp, ent, _, _ = call(hv, x, [-1, 100, 1 << 30, 99], 0)
    assert np.isnan(lp[:3]).all() and np.isfinite(lp[3]) and np.isfinite(ent).all()


def test_scratch_is_ready_for_the_next_call_and_bits_repeat(hv):
    g = np.random.default_rng(5)
    x = g.standard_normal((3, 60000)).astype(F32)
    s = Dev(nbytes=hv.logprob_scratch(3, 60000, 20))
    a = call(hv, x, [1, 2, 3], 20, scratch=s)
    call(hv, -x[:2], [1, 2], 7, scratch=s)                      # a smaller call between
    b = call(hv, x, [1, 2, 3], 20, scratch=s)
    for p, q in zip(a, b):
        assert np.array_equal(bits(p), bits(q))


def test_captured_scoring(hv):
    g = np.random.default_rng(6)
    x, y = (g.standard_normal((2, 40000)).astype(F32) for _ in range(2))
    want = call(hv, y, [7, 8], 5)
    d, tok, s = Dev(x), Dev(np.array([7, 8], np.int32)), Dev(nbytes=hv.logprob_scratch(2, 40000, 5))
    lp, ent, ids, alt = (Dev(nbytes=n) for n in (8, 8, 40, 40))
    st = hv.stream_create()
    hv.capture_begin(st)
    hv.logprob_rows(d, 40000, 2, 40000, tok, 5, lp, ent, ids, alt, s, st)
    graph = hv.capture_end(st)
    ex = hv.graph_instantiate(graph)
    for z in (x, y):
        d.put(z)
        hv.synchronize()
        hv.graph_launch(ex, st)
        hv.stream_synchronize(st)
    for p, q in zip((lp.get(F32), ent.get(F32), ids.get(np.int32), alt.get(F32)), want):
        assert np.array_equal(bits(p), bits(q.ravel()))
    hv.graph_destroy(graph, ex)
    hv.stream_destroy(st)


@pytest.mark.parametrize("kv", ["f32", "q8"])
def test_engine_score(hv, kv):
    """score() against log softmax of the engine's own logits. Over the f32 cache every
    prefix's logits are the same bits in any run; over the 8-bit cache the last row's are."""
    import limited
    cfg = w4format.Config(synth.tiny_arch())
    e = limited.Engine(config=cfg, tensors=synth.iter_tensors(cfg, 8), quiet=True,
                       max_context=320, prefill="batched", kv_dtype=kv, fused=kv == "f32")
    try:
        ids = synth.prompt_ids(cfg, 8, 300)
        got = e.score(ids, top=4)
        assert got["logprob"].shape == (299,) and got["top_ids"].shape == (299, 4)
        for i in ((0, 1, 31, 255, 256, 298) if kv == "f32" else (298,)):
            x = e.logits(ids[:i + 1])[None]
            row = [got["logprob"][i:i + 1], got["entropy"][i:i + 1], got["top_ids"][i:i + 1],
                   got["top_logprobs"][i:i + 1]]
            check(row, x, np.array([ids[i + 1]]), 4)
        again = e.score(ids)
        assert np.array_equal(bits(again["logprob"]), bits(got["logprob"]))
        assert again["top_ids"].shape == (299, 0)
        for bad in ([1], [1, -1], [1, cfg.vocab], list(range(322)), [1.0, 2.0],
                    np.array([1, (1 << 32) + 1])):
            with pytest.raises(ValueError):
                e.score(bad)
        with pytest.raises(ValueError):
            e.score(ids, top=33)
    finally:
        e.free()


def test_one_scratch_for_calls_of_different_sizes(hv):
    """The scratch of the largest call serves any smaller one in any order."""
    g = np.random.default_rng(9)
    s = Dev(nbytes=max(hv.logprob_scratch(r, 30000, 32) for r in (1, 2, 100, 290)))
    for rows in (100, 2, 290, 1, 100, 290):
        x = g.standard_normal((rows, 30000)).astype(F32)
        tok = g.integers(0, 30000, rows)
        check(call(hv, x, tok, 32, scratch=s), x, tok, 32)


def test_scratch_does_for_every_smaller_call(hv):
    """Fewer rows are cut into more pieces: one scratch, of the largest call, for all."""
    for n in (1, 4096, 70001, 151936):
        for top in (0, 5):
            sizes = [hv.logprob_scratch(r, n, top) for r in range(1, 1400)]
            assert sizes == sorted(sizes)
    rows, n, top = 256, 40000, 32
    need = hv.logprob_scratch(rows, n, top)
    room = np.full(need + 65536, 0x5A, np.uint8)
    room[:need] = 0
    s = Dev(room)
    x = (np.random.default_rng(31).standard_normal((rows, n)) * 3).astype(F32)
    for r, t in ((256, 32), (148, 32), (98, 5), (1, 32), (74, 0), (30, 32), (147, 1), (256, 2)):
        tok = np.arange(r) * 7
        check(call(hv, x[:r], tok, t, scratch=s), x[:r], tok, t)
        assert (s.get(np.uint8)[need:] == 0x5A).all(), (r, t)


@pytest.mark.parametrize("order", ["up", "down", "saw", "late"])
def test_orders_that_keep_bringing_larger_logits(hv, order):
    n = 50000
    x = np.linspace(-30, 30, n).astype(F32)[None].repeat(2, 0)
    if order == "down":
        x = x[:, ::-1].copy()
    if order == "saw":
        x = x + 20 * (np.arange(n) % 4096 / 4096).astype(F32)
    if order == "late":
        x[:, :-40] = 0
    check(call(hv, x, [5, n - 1], 32), x, np.array([5, n - 1]), 32)


@pytest.mark.parametrize("rows", [2, 300])
@pytest.mark.parametrize("n", [40, 257, 4096, 4097, 9001, 33000])
@pytest.mark.parametrize("top", [1, 5, 32])
def test_alternatives_in_order_whatever_comes_first(hv, n, rows, top):
    """The order of np.argmax, rows whole and cut: equal logits, few values, NaN and infinities
    among the first logits or the last, all that counts in one lane."""
    g = np.random.default_rng(n + top)
    x = g.standard_normal((rows, n)).astype(F32)
    x[0] = 1.5
    x[1] = g.integers(0, 3, n)
    if rows > 2:
        x[2, :7] = np.nan
        x[3, -3:] = np.nan
        x[4, :4], x[4, -2:] = np.inf, np.nan
        x[5, 9:] = -np.inf
        x[6, :-5] = -np.inf
        x[7, 4:8] += 90
        x[8, ::512] += 50
        x[9] = np.linspace(3, -3, n)
        x[10] = -np.inf
    ids = call(hv, x, np.zeros(rows, int), top)[2]
    key = np.where(np.isnan(x), np.inf, np.where(x == 0, 0, x))
    for r in range(min(rows, 20)):
        want = np.lexsort((np.arange(n), -key[r], ~np.isnan(x[r])))[:top]
        assert np.array_equal(ids[r], want), r
