"""Attention over a shared prefix, the write of a batch's rows, attention that adds up its weights
and eviction on a B200, against the 64-bit plain forms of span_ref.py."""
import numpy as np
import pytest

import span_ref as R
from gpu_util import Dev, bits

pytestmark = pytest.mark.gpu
F32, F16, HD = np.float32, np.float16, 128
SCALE = float(F32(1.0 / np.sqrt(HD)))


def cache(g, *shape):
    """K and V in binary16, some dims of K larger than others."""
    k = g.standard_normal((*shape, HD)) * np.exp(0.5 * g.standard_normal(HD))
    return k.astype(F16), g.standard_normal((*shape, HD)).astype(F16)


def queries(g, rows, nq, scale=1.0):
    return (scale * g.standard_normal((rows, nq, HD)) * np.exp(0.5 * g.standard_normal(HD))).astype(F32)


def i32(x):
    return Dev(np.atleast_1d(np.array(x, np.int32)))


def scratch(n):
    return Dev(nbytes=n)


def near(got, want, tol):
    off = np.abs(got.astype(np.float64) - want)
    assert np.isfinite(got).all()
    assert (off <= tol).all(), float((off / tol).max())


# ---- attention over a shared prefix ----------------------------------------------------

def run_shared(hv, q, pk, pv, plen, tk, tv, row0, tlen, scale=SCALE, fill=7.0, s=None, stream=0):
    nrow, nq, _ = q.shape
    nseq, nkv, tcap, _ = tk.shape
    pcap, group = pk.shape[1], nq // nkv
    s = s or scratch(hv.attn_shared_scratch(nq, group, pcap, tcap, nseq, nrow))
    ctx = Dev(np.full(q.shape, fill, F32))
    dev = [Dev(x) for x in (q, tk, tv)] + [Dev(pk) if pcap else 0, Dev(pv) if pcap else 0]
    dr = 0 if row0 is None else i32(row0)
    dt, dp, ds = i32(tlen), i32(plen), Dev(np.array([scale], F32))
    hv.attn_shared(dev[0], dev[3], dev[4], pcap, dp if pcap else 0, dev[1], dev[2], tcap, dr, dt, ctx,
                   ds, nq, HD, group, nseq, nrow, s, stream)
    return ctx.get(F32, q.shape)


def check_shared(hv, g, nkv, group, plen, pcap, rows, tlen, tcap, extra=0, stale=np.nan, one=False):
    nseq, nrow = len(rows), sum(rows) + extra
    pk, pv = cache(g, nkv, pcap)
    tk, tv = cache(g, nseq, nkv, tcap)
    pk[:, plen:], pv[:, plen:] = stale, stale            # nothing there may count
    for s, n in enumerate(tlen):
        tk[s, :, n:], tv[s, :, n:] = stale, stale
    q = queries(g, nrow, nkv * group)
    row0 = None if one else np.concatenate([[0], np.cumsum(rows)])
    got = run_shared(hv, q, pk, pv, plen, tk, tv, row0, tlen)
    want, tol = R.shared(q, pk, pv, plen, tk, tv, row0, tlen, SCALE)
    m = sum(rows)
    near(got[:m], want[:m], tol[:m])
    assert (got[m:] == 7).all()


@pytest.mark.parametrize("nkv,group,plen,tails", [
    (1, 1, 0, [1]), (2, 1, 1, [1]), (8, 2, 45, [3, 9]), (2, 4, 31, [0, 1, 2]), (1, 8, 32, [5] * 9),
    (3, 5, 33, [64, 1, 65, 17]), (2, 3, 127, [2] * 33), (1, 7, 128, [1, 16, 130]),
    (2, 6, 129, [7] * 20), (8, 4, 300, list(range(1, 17))), (2, 8, 1000, [40] * 16),
    (1, 4, 4096, [3, 200] * 16), (2, 2, 4225, [9] * 64), (1, 1, 5000, [1, 2, 3])])
def test_one_row_a_sequence(hv, nkv, group, plen, tails):
    g = np.random.default_rng(plen + group)
    check_shared(hv, g, nkv, group, plen, plen + 5, [1] * len(tails), tails, max(tails) + 2, one=True)


@pytest.mark.parametrize("nkv,group,plen,rows,tails", [
    (2, 4, 0, [3], [3]), (1, 2, 10, [1, 0, 5], [4, 9, 5]), (2, 8, 100, [17, 3, 0, 12], [17, 3, 4, 40]),
    (8, 4, 200, [9, 31, 33, 1], [9, 31, 64, 300]), (1, 5, 700, [40, 2, 65], [41, 2, 65]),
    (2, 3, 64, [150], [150]), (1, 8, 2000, [3, 17, 8, 8, 9, 2] * 3, [3, 20, 8, 30, 9, 2] * 3),
    (2, 1, 300, [128, 64], [130, 64]), (1, 4, 20, [0, 0, 2], [5, 0, 2]),
    (2, 4, 2000, [1, 2, 3] * 10, [1, 2, 9] * 10), (1, 8, 1111, [0, 4, 1] * 9, [7, 30, 1] * 9)])
def test_runs_of_rows(hv, nkv, group, plen, rows, tails):
    g = np.random.default_rng(plen + len(rows))
    check_shared(hv, g, nkv, group, plen, plen + 3, rows, tails, max(tails) + 1, extra=2)


@pytest.mark.parametrize("nkv,group,nseq,plen", [
    (1, 1, 129, 2100), (2, 3, 50, 2500), (1, 5, 70, 1024), (8, 4, 64, 1100), (3, 7, 40, 1500),
    (1, 8, 64, 4097), (1, 2, 65, 2176), (1, 4, 40, 12800), (8, 8, 64, 2100), (8, 4, 33, 8190),
    (1, 1, 600, 2100), (2, 3, 100, 2500), (1, 2, 300, 2176), (1, 5, 250, 1024)])
def test_many_rows_over_a_long_prefix(hv, nkv, group, nseq, plen):
    g = np.random.default_rng(plen)
    check_shared(hv, g, nkv, group, plen, plen + 130, [1] * nseq, [1 + i % 7 for i in range(nseq)], 9, one=True)


@pytest.mark.parametrize("nseq", [3, 70, 160])
@pytest.mark.parametrize("way", ["rising", "falling", "steps", "peaks", "far"])
def test_scores_that_change_along_the_prefix(hv, nseq, way):
    """The largest score so far is passed often, seldom, by a little and by far."""
    g = np.random.default_rng(13)
    plen, nkv, group = 2300, 1, 4
    pk, pv = cache(g, nkv, plen)
    tk, tv = cache(g, nseq, nkv, 4)
    q = queries(g, nseq, nkv * group)
    u = g.standard_normal(HD)
    u /= np.sqrt(HD)
    t = np.arange(plen)
    size = {"rising": 0.05 * t, "falling": -0.05 * t, "steps": 12.0 * (t // 100), "peaks": 150.0 * (t % 331 == 330) * (t / plen),
            "far": np.where(t == 1777, 4000.0, -0.02 * t)}[way]
    pk = (pk * 0.2 + size[None, :, None] * u).astype(F16)
    q += (u * np.sqrt(HD) * 0.9).astype(F32)
    got = run_shared(hv, q, pk, pv, plen, tk, tv, None, [4] * nseq)
    near(got, *R.shared(q, pk, pv, plen, tk, tv, None, [4] * nseq, SCALE))


@pytest.mark.parametrize("nkv,group,rows,longest", [
    (8, 1, [1] * 40, 31), (8, 4, [2, 9, 17] * 6, 30), (8, 8, [16, 0, 3, 5] * 5, 30), (2, 4, [40, 33, 65] * 3, 66),
    (8, 3, [5, 6, 1] * 12, 120), (8, 8, [7, 2] * 20, 250), (4, 2, [1] * 100, 257), (8, 4, [3, 12] * 9, 400),
    (8, 8, [30, 2] * 12, 300), (1, 7, [8] * 5, 1100)])
def test_tails_of_many_rows_after_a_long_prefix(hv, nkv, group, rows, longest):
    """Tails from the shortest to the longest in one call, their chunks ending inside a block."""
    g = np.random.default_rng(longest + group)
    tails = [max(r, min(longest, 1 + (i * 37) % longest)) for i, r in enumerate(rows)]
    tails[-1] = longest
    plen = -(-2 ** 20 // (nkv * group * (sum(rows) + 3)))  # just enough for tiles
    check_shared(hv, g, nkv, group, plen, plen, rows, tails, longest + 1, extra=3)


@pytest.mark.parametrize("nkv,group,plen,rows,tails", [
    (8, 8, 50, [40] * 4, [40, 300, 129, 64]), (8, 4, 0, [30, 50, 80, 1], [400, 300, 80, 270]),
    (8, 4, 45, [1] * 64, [1 + 37 * s % 290 for s in range(64)]), (8, 8, 3, [2] * 40, [2 + 7 * s for s in range(40)]),
    (8, 2, 200, [9] * 8, [60 - s for s in range(8)]), (2, 8, 90, [70, 3, 90], [70, 600, 95])])
def test_tails_of_many_rows_after_a_short_prefix(hv, nkv, group, plen, rows, tails):
    g = np.random.default_rng(plen + group)
    check_shared(hv, g, nkv, group, plen, plen + 2, rows, tails, max(tails) + 1, extra=1)


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad", [np.nan, -np.inf])
@pytest.mark.parametrize("longest", [30, 200, 300])
def test_tails_of_many_rows_and_what_is_not_finite(hv, which, bad, longest):
    """As below, for sequences of many rows after a prefix of whole tiles."""
    g = np.random.default_rng(longest)
    nseq, n = 24, 20
    plen = -(-2 ** 17 // (2 * nseq * n))
    pk, pv = cache(g, 8, plen)
    tk, tv = cache(g, nseq, 8, longest)
    q = queries(g, nseq * n, 16)
    row0, tails = np.arange(nseq + 1) * n, [longest - s % 3 for s in range(nseq)]
    want, tol = R.shared(q, pk, pv, plen, tk, tv, row0, tails, SCALE)
    at = tails[5] - n + 11                                # row 11 of sequence 5 is the first to see it
    (tk if which == "k" else tv)[5, 3, at, :] = bad
    got = run_shared(hv, q, pk, pv, plen, tk, tv, row0, tails)
    hit = np.zeros((nseq * n, 16), bool)
    hit[5 * n + 11:6 * n, 6:8] = True
    near(got[~hit], want[~hit], tol[~hit])
    if which == "v" or np.isnan(bad):
        assert not np.isfinite(got[hit]).all(-1).any()


def test_a_prefix_of_full_capacity_and_none_at_all(hv):
    g = np.random.default_rng(5)
    check_shared(hv, g, 2, 4, 256, 256, [1] * 20, [8] * 20, 8, one=True)
    check_shared(hv, g, 2, 4, 0, 0, [2, 1], [2, 6], 6)
    check_shared(hv, g, 2, 2, 0, 40, [2, 1], [2, 6], 6)
    check_shared(hv, g, 2, 4, 0, 5000, [1] * 40, [i % 5 for i in range(40)], 5, one=True)
    check_shared(hv, g, 1, 4, 1024, 1024, [1] * 40, [5] * 40, 5, one=True)
    check_shared(hv, g, 2, 8, 1024, 1024, [1] * 70, [5] * 70, 5, one=True)


def test_rows_that_see_nothing_are_zero(hv):
    """A row of a sequence whose tail is shorter than its rows, without a prefix."""
    g = np.random.default_rng(6)
    check_shared(hv, g, 2, 4, 0, 8, [3, 1, 2], [1, 0, 2], 4)
    check_shared(hv, g, 1, 8, 40, 64, [5, 1], [2, 0], 4)


@pytest.mark.parametrize("rows,plen", [([1] * 4, 200), ([1] * 40, 600), ([6, 4], 300), ([1] * 40, 2000), ([1] * 100, 2000)])
def test_lengths_out_of_range_leave_nan(hv, rows, plen):
    g = np.random.default_rng(7)
    nseq = len(rows)
    pk, pv = cache(g, 2, plen)
    tk, tv = cache(g, nseq, 2, 16)
    q = queries(g, sum(rows), 8)
    row0 = np.concatenate([[0], np.cumsum(rows)])
    tlen = np.full(nseq, 9)
    tlen[1] = 17
    got = run_shared(hv, q, pk, pv, plen, tk, tv, row0, tlen)
    bad = np.arange(row0[1], row0[2])
    assert np.isnan(got[bad]).all()
    ok = np.setdiff1d(np.arange(sum(rows)), bad)
    want, tol = R.shared(q, pk, pv, plen, tk, tv, row0, np.minimum(tlen, 16), SCALE)
    near(got[ok], want[ok], tol[ok])
    for n in (-1, plen + 1, 2 ** 31 - 1):
        assert np.isnan(run_shared(hv, q, pk, pv, n, tk, tv, row0, np.full(nseq, 9))).all()
    tlen[1] = -1
    assert np.isnan(run_shared(hv, q, pk, pv, plen, tk, tv, row0, tlen)[bad]).all()


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_a_row_does_not_see_does_not_count(hv, which, bad):
    """An infinity or a NaN in a tail reaches the rows behind it of that sequence only."""
    g = np.random.default_rng(8)
    rows, tails = [20, 9, 3], [20, 30, 3]
    pk, pv = cache(g, 2, 150)
    tk, tv = cache(g, 3, 2, 32)
    q = queries(g, 32, 8)
    row0 = np.concatenate([[0], np.cumsum(rows)])
    want, tol = R.shared(q, pk, pv, 150, tk, tv, row0, tails, SCALE)
    (tk if which == "k" else tv)[0, 1, 11, 5] = bad
    (tk if which == "k" else tv)[1, 1, 26, :] = bad
    got = run_shared(hv, q, pk, pv, 150, tk, tv, row0, tails)
    hit = np.zeros((32, 8), bool)
    hit[11:20, 4:] = True
    hit[20 + 5:29, 4:] = True
    near(got[~hit], want[~hit], tol[~hit])
    assert not np.isfinite(got[25:29, 4:]).all(-1).any()
    if which == "v" or np.isnan(bad):
        assert not np.isfinite(got[11:20, 4:]).all(-1).any()


@pytest.mark.parametrize("scale,qs,ks", [(SCALE, 1e-20, 1.0), (SCALE, 30.0, 20.0), (-SCALE, 1.0, 1.0),
                                         (0.0, 1.0, 1.0), (1.0, 2e4, 1e-3), (1e-30, 3e34, 1.0)])
def test_queries_and_scales_of_any_size(hv, scale, qs, ks):
    g = np.random.default_rng(9)
    for nseq, plen in ((3, 300), (40, 300), (40, 2000), (150, 2000)):
        pk, pv = cache(g, 1, plen)
        tk, tv = cache(g, nseq, 1, 40)
        pk, tk = (pk * F16(ks)).astype(F16), (tk * F16(ks)).astype(F16)
        pv[:, ::3], tv[:, :, ::3] = F16(6e4), F16(-6e4)
        q = queries(g, nseq, 4, qs)
        q[0, 0] = 0
        q[1, 1, 5:] *= F32(1e-9)
        tl = [33] * nseq
        got = run_shared(hv, q, pk, pv, plen, tk, tv, None, tl, scale)
        want, tol = R.shared(q, pk, pv, plen, tk, tv, None, tl, float(F32(scale)))
        near(got, want, tol)


def test_repeats_are_equal(hv):
    """The same call gives the same bits."""
    g = np.random.default_rng(10)
    pk, pv = cache(g, 2, 500)
    tk, tv = cache(g, 12, 2, 20)
    q = queries(g, 12, 8)
    a = run_shared(hv, q, pk, pv, 500, tk, tv, None, [20] * 12)
    b = run_shared(hv, q, pk, pv, 500, tk, tv, None, [20] * 12)
    assert np.array_equal(bits(a), bits(b))


def test_one_scratch_serves_calls_of_every_size(hv):
    """The scratch of the largest call, used by others in turn on a stream of its own."""
    g = np.random.default_rng(11)
    s = scratch(hv.attn_shared_scratch(16, 8, 3000, 100, 40, 60))
    st = hv.stream_create()
    try:
        for nseq, plen, tcap in ((40, 3000, 5), (1, 3, 100), (17, 900, 33), (40, 2999, 100), (2, 0, 4)):
            pk, pv = cache(g, 2, 3000)
            tk, tv = cache(g, nseq, 2, tcap)
            q = queries(g, nseq, 16)
            nq, ctx = 16, Dev(np.zeros(q.shape, F32))
            dev = [Dev(x) for x in (q, pk, pv, tk, tv)]
            dp, dt, ds = i32(plen), i32([tcap] * nseq), Dev(np.array([SCALE], F32))
            hv.synchronize()
            hv.attn_shared(dev[0], dev[1], dev[2], 3000, dp, dev[3], dev[4], tcap, 0, dt, ctx, ds, nq,
                           HD, 8, nseq, nseq, s, st)
            hv.stream_synchronize(st)
            near(ctx.get(F32, q.shape), *R.shared(q, pk, pv, plen, tk, tv, None, [tcap] * nseq, SCALE))
    finally:
        hv.stream_destroy(st)


def test_two_captured_graphs_follow_device_lengths(hv):
    """Write and attention captured twice, each with a scratch of its own, replayed in turn as the
    lengths on the device grow."""
    g = np.random.default_rng(12)
    nkv, group, nseq, tcap, plen, cap = 2, 4, 5, 24, 130, 200
    nq = nkv * group
    ang = np.arange(cap)[:, None] * (1e4 ** (-np.arange(64) / 64.0))[None]
    cos, sin = Dev(np.cos(ang).astype(F32)), Dev(np.sin(ang).astype(F32))
    gains = [Dev((1 + 0.1 * g.standard_normal(HD)).astype(F32)) for _ in range(2)]
    lanes = []
    for _ in range(2):
        pk, pv = cache(g, nkv, plen)
        qkv = g.standard_normal((nseq, (nq + 2 * nkv) * HD)).astype(F32)
        L = dict(pk=pk, pv=pv, qkv=Dev(qkv), dpk=Dev(pk), dpv=Dev(pv),
                 tk=Dev(nbytes=nseq * nkv * tcap * 256), tv=Dev(nbytes=nseq * nkv * tcap * 256),
                 q=Dev(nbytes=nseq * nq * 512), ctx=Dev(nbytes=nseq * nq * 512), st=hv.stream_create(),
                 s=scratch(hv.attn_shared_scratch(nq, group, plen, tcap, nseq, nseq)),
                 pl=i32(plen), tl=i32([0] * nseq), sc=Dev(np.array([SCALE], F32)))
        hv.synchronize()
        hv.capture_begin(L["st"])
        hv.qk_shared(L["qkv"], *gains, cos, sin, cap, L["pl"], 0, L["tl"], L["q"], L["tk"], L["tv"], nq,
                     nkv, HD, tcap, 1e-5, nseq, nseq, L["st"])
        hv.attn_shared(L["q"], L["dpk"], L["dpv"], plen, L["pl"], L["tk"], L["tv"], tcap, 0, L["tl"],
                       L["ctx"], L["sc"], nq, HD, group, nseq, nseq, L["s"], L["st"])
        L["graph"] = hv.capture_end(L["st"])
        L["exec"] = hv.graph_instantiate(L["graph"])
        lanes.append(L)
    for step in range(1, 4):
        tlen = np.array([step, step + 3, step, 2 * step, step + 10], np.int32)
        for L in lanes:
            L["tl"].put(tlen)
            L["qkv"].put(g.standard_normal((nseq, (nq + 2 * nkv) * HD)).astype(F32))
        hv.synchronize()
        for L in lanes:
            hv.graph_launch(L["exec"], L["st"])
        for L in lanes:
            hv.stream_synchronize(L["st"])
            tk, tv = (L[x].get(F16, (nseq, nkv, tcap, HD)) for x in ("tk", "tv"))
            q = L["q"].get(F32, (nseq, nq, HD))
            near(L["ctx"].get(F32, q.shape), *R.shared(q, L["pk"], L["pv"], plen, tk, tv, None, tlen, SCALE))
    for L in lanes:
        hv.graph_destroy(L["graph"], L["exec"])
        hv.stream_destroy(L["st"])


@pytest.mark.parametrize("nseq,plen", [(40, 1500), (70, 5000)])
def test_captured_call_over_a_long_prefix(hv, nseq, plen):
    """Several kernels in a call: replayed back to back over changing inputs."""
    g = np.random.default_rng(plen)
    nkv, group, tcap = 2, 4, 40
    nq = nkv * group
    pk, pv = cache(g, nkv, plen)
    tk, tv = cache(g, nseq, nkv, tcap)
    d = [Dev(x) for x in (pk, pv, tk, tv)]
    tlen = g.integers(0, tcap + 1, nseq)
    pl, tl, sc = i32(plen), i32(tlen), Dev(np.array([SCALE], F32))
    q, ctx = Dev(nbytes=nseq * nq * 512), Dev(nbytes=nseq * nq * 512)
    s = scratch(hv.attn_shared_scratch(nq, group, plen, tcap, nseq, nseq))
    st = hv.stream_create()
    hv.synchronize()
    hv.capture_begin(st)
    hv.attn_shared(q, d[0], d[1], plen, pl, d[2], d[3], tcap, 0, tl, ctx, sc, nq, HD, group, nseq, nseq, s, st)
    gr = hv.capture_end(st)
    ex = hv.graph_instantiate(gr)
    for rep in range(3):
        rows = queries(g, nseq, nq)
        q.put(rows)
        hv.synchronize()
        for _ in range(1 + 5 * rep):
            hv.graph_launch(ex, st)
        hv.stream_synchronize(st)
        near(ctx.get(F32, rows.shape), *R.shared(rows, pk, pv, plen, tk, tv, None, tlen, SCALE))
    hv.graph_destroy(gr, ex)
    hv.stream_destroy(st)


# ---- the write of a batch's rows -------------------------------------------------------

@pytest.mark.parametrize("nkv,group,rows,tails,base", [
    (1, 1, [1], [1], 0), (2, 4, [1, 1, 1], [1, 7, 20], 33), (8, 8, [5, 0, 17, 3], [9, 4, 17, 20], 100),
    (3, 5, [2, 40], [2, 40], 7)])
def test_rows_are_written_as_runs_are(hv, nkv, group, rows, tails, base):
    """Bit for bit what qk_rows writes for each sequence's run at its positions."""
    g = np.random.default_rng(base)
    nq, nrow, tcap, cap = nkv * group, sum(rows) + 1, 44, 160
    ang = np.arange(cap)[:, None] * (1e6 ** (-np.arange(64) / 64.0))[None]
    cos, sin = np.cos(ang).astype(F32), np.sin(ang).astype(F32)
    dc, dsn = Dev(cos), Dev(sin)
    qn, kn = (Dev((1 + 0.1 * g.standard_normal(HD)).astype(F32)) for _ in range(2))
    qkv = g.standard_normal((nrow, (nq + 2 * nkv) * HD)).astype(F32)
    row0 = np.concatenate([[0], np.cumsum(rows)])
    old = g.standard_normal((2, len(rows), nkv, tcap, HD)).astype(F16)
    tk, tv, qo = Dev(old[0]), Dev(old[1]), Dev(np.full((nrow, nq, HD), 7, F32))
    dq, dbase, dr, dt = Dev(qkv), i32(base), i32(row0), i32(tails)
    hv.qk_shared(dq, qn, kn, dc, dsn, cap, dbase, dr, dt, qo, tk, tv, nq, nkv, HD, tcap, 1e-5, len(rows),
                 nrow)
    want_q = np.full((nrow, nq, HD), 7, F32)
    want = old.copy()
    for s, (r, t) in enumerate(zip(rows, tails)):
        if not r:
            continue
        kc, vc, q2 = Dev(nbytes=nkv * cap * 256), Dev(nbytes=nkv * cap * 256), Dev(nbytes=r * nq * 512)
        run = Dev(qkv[row0[s]:row0[s + 1]])
        hv.qk_rows(run, qn, kn, dc, dsn, base + t - r, q2, kc, vc, nq, nkv, HD, cap, 1e-5, r, f16=True)
        want_q[row0[s]:row0[s + 1]] = q2.get(F32, (r, nq, HD))
        for i, c in enumerate((kc, vc)):
            want[i, s, :, t - r:t] = c.get(F16, (nkv, cap, HD))[:, base + t - r:base + t]
    assert np.array_equal(bits(qo.get(F32, want_q.shape)), bits(want_q))
    for i, c in enumerate((tk, tv)):
        assert np.array_equal(c.get(np.uint16), want[i].view(np.uint16).ravel())


def test_rows_outside_are_not_written(hv):
    """Slots before 0, tails longer than their room, positions past the tables."""
    g = np.random.default_rng(3)
    nq = nkv = 2
    rows, tails, tcap, cap, base = [3, 1, 2, 1], [2, 9, 6, -3], 8, 40, 35
    row0 = np.concatenate([[0], np.cumsum(rows)])
    ones, tab = Dev(np.ones(HD, F32)), Dev(np.ones((cap, 64), F32))
    old = g.standard_normal((4, nkv, tcap, HD)).astype(F16)
    tk, tv, qo = Dev(old), Dev(old), Dev(np.full((7, nq, HD), 7, F32))
    dq = Dev(g.standard_normal((7, 6 * HD)).astype(F32))
    db, dr, dt = i32(base), i32(row0), i32(tails)
    hv.qk_shared(dq, ones, ones, tab, tab, cap, db, dr, dt, qo, tk, tv, nq, nkv, HD, tcap, 1e-5, 4, 7)
    q = qo.get(F32, (7, nq, HD))
    assert np.isnan(q).all((1, 2)).tolist() == [True, False, False, True, False, True, True]
    new = tk.get(F16, old.shape)
    changed = (new != old).any((1, 3))
    want = np.zeros((4, tcap), bool)
    want[0, 0] = want[0, 1] = want[2, 4] = True
    assert np.array_equal(changed, want)


# ---- attention that adds up its weights -------------------------------------------------

def run_mass(hv, q, k, v, pos0, mass_in, decode, apart=True, stream=0, s=None, scale=SCALE):
    """-> context, mass_out (what was in it before: 5)."""
    ntok, nq, _ = q.shape
    nkv, cap, _ = k.shape
    group = nq // nkv
    dq, dk, dv, ds = Dev(q), Dev(k), Dev(v), Dev(np.array([scale], F32))
    ctx = Dev(np.full(q.shape, 7, F32))
    out = Dev(np.full((nkv, cap), 5, F32))
    src = 0
    if mass_in is not None:
        src = Dev(mass_in)
        out = out if apart else src
    s = s or scratch(hv.attn_mass_scratch(nq, group, cap, ntok))
    if decode:
        dp = i32(pos0)
        hv.attn_decode_mass(dq, dk, dv, ctx, src, out, ds, dp, nq, HD, group, cap, s, stream)
    else:
        hv.attn_rows_mass(dq, dk, dv, ctx, src, out, ds, pos0, nq, HD, group, cap, ntok, s, stream)
    return ctx.get(F32, q.shape), out.get(F32, (nkv, cap))


def check_mass(hv, g, nkv, group, pos0, ntok, cap, decode, form):
    n = pos0 + ntok
    k, v = cache(g, nkv, cap)
    k[:, n:], v[:, n:] = np.nan, np.nan
    q = queries(g, ntok, nkv * group)
    mi = None if form == "none" else np.abs(g.standard_normal((nkv, cap))).astype(F32)
    ctx, m = run_mass(hv, q, k, v, pos0, mi, decode, form == "apart")
    want, tol, wm, mt = R.mass(q, k, v, pos0, mi, SCALE)
    near(ctx, want, tol)
    near(m[:, :n], wm, mt)
    assert np.array_equal(m[:, n:], mi[:, n:] if form == "same" else np.full((nkv, cap - n), 5, F32))


@pytest.mark.parametrize("form", ["same", "apart", "none"])
@pytest.mark.parametrize("nkv,group,n", [(1, 1, 1), (2, 4, 2), (8, 2, 31), (3, 5, 64), (2, 8, 129),
                                         (8, 4, 1000), (1, 7, 4225), (2, 3, 9001)])
def test_decode_with_mass(hv, nkv, group, n, form):
    check_mass(hv, np.random.default_rng(n), nkv, group, n - 1, 1, n + 3 * (form != "apart"), True, form)


@pytest.mark.parametrize("nkv,group,pos0,ntok", [
    (1, 1, 0, 1), (2, 4, 0, 5), (8, 2, 256, 44), (1, 8, 100, 17), (2, 5, 63, 65), (1, 3, 1000, 31),
    (2, 4, 128, 128), (1, 8, 700, 256), (2, 1, 0, 300), (1, 2, 2048, 200), (1, 7, 4000, 3),
    (1, 1, 900, 290), (2, 5, 500, 120), (1, 3, 0, 700), (8, 8, 2100, 64), (8, 4, 1000, 200),
    (8, 4, 2400, 2), (8, 4, 1200, 4), (8, 4, 600, 4), (1, 2, 0, 2500)])
def test_run_with_mass(hv, nkv, group, pos0, ntok):
    g = np.random.default_rng(pos0 + ntok)
    check_mass(hv, g, nkv, group, pos0, ntok, pos0 + ntok + 2, False, "apart")
    check_mass(hv, g, nkv, group, pos0, ntok, pos0 + ntok, False, "same")


def test_mass_adds_up_over_calls(hv):
    """A run, then single rows: every weight once. Each row's weights are 1 in all."""
    g = np.random.default_rng(20)
    nkv, group, cap, ntok = 2, 4, 80, 60
    k, v = cache(g, nkv, cap)
    q = queries(g, cap, nkv * group)
    _, m = run_mass(hv, q[:ntok], k, v, 0, np.zeros((nkv, cap), F32), False, False)
    for t in range(ntok, cap):
        _, m = run_mass(hv, q[t:t + 1], k, v, t, m, True, False)
    _, _, want, tol = R.mass(q, k, v, 0, None, SCALE)
    near(m, want, 4 * tol + 32 * R.U * want)
    assert np.allclose(m.sum(1), cap * group, rtol=1e-4)


def test_decode_with_mass_outside_the_cache(hv):
    g = np.random.default_rng(21)
    k, v = cache(g, 2, 40)
    q = queries(g, 1, 4)
    for pos in (-1, 40, 2 ** 31 - 1, -2 ** 31):
        ctx, m = run_mass(hv, q, k, v, pos, np.ones((2, 40), F32), True)
        assert np.isnan(ctx).all() and (m == 5).all()


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_mass_of_rows_before_a_bad_position(hv, bad):
    g = np.random.default_rng(22)
    for group, ntok, cap in ((4, 30, 200), (8, 100, 200), (8, 100, 2000)):
        k, v = cache(g, 1, cap)
        q = queries(g, ntok, group)
        want, tol, _, _ = R.mass(q, k, v, 60, None, SCALE)
        v[0, 60 + 11] = bad
        ctx, m = run_mass(hv, q, k, v, 60, None, False)
        near(ctx[:11], want[:11], tol[:11])
        assert not np.isfinite(ctx[11:]).any()


def test_captured_decode_with_mass(hv):
    """Replayed as *pos moves, in place, one scratch."""
    g = np.random.default_rng(23)
    nkv, group, cap = 2, 4, 300
    k, v = cache(g, nkv, cap)
    q = queries(g, 1, nkv * group)
    dq, dk, dv, ds = Dev(q), Dev(k), Dev(v), Dev(np.array([SCALE], F32))
    ctx, m, pos = Dev(nbytes=q.nbytes), Dev(nbytes=nkv * cap * 4), i32(0)
    s = scratch(hv.attn_mass_scratch(nkv * group, group, cap, 1))
    st = hv.stream_create()
    hv.synchronize()
    hv.capture_begin(st)
    hv.attn_decode_mass(dq, dk, dv, ctx, m, m, ds, pos, nkv * group, HD, group, cap, s, st)
    gr = hv.capture_end(st)
    ex = hv.graph_instantiate(gr)
    total, tol = np.zeros((nkv, cap)), np.zeros((nkv, cap))
    for p in (0, 1, 31, 32, 200, 299):
        pos.put(np.array([p], np.int32))
        hv.synchronize()
        hv.graph_launch(ex, st)
        hv.stream_synchronize(st)
        want, ct, w, wt = R.mass(q, k, v, p, None, SCALE)
        near(ctx.get(F32, q.shape), want, ct)
        total[:, :p + 1] += w
        tol[:, :p + 1] += wt + 8 * R.U * total[:, :p + 1]
    near(m.get(F32, (nkv, cap)), total, tol)
    hv.graph_destroy(gr, ex)
    hv.stream_destroy(st)


# ---- eviction ----------------------------------------------------------------------------

def run_evict(hv, k, v, mass, n, added, limit, keep, recent, dcap=None, stream=0, want_kept=True):
    """k, v [nset, nkv, cap, 128]; dcap None: in place, the sets' K and V side by side as an engine
    has them. -> k, v, mass, kept, length."""
    nset, nkv, cap, _ = k.shape
    one = nkv * cap * HD
    both = Dev(np.stack([k, v], 1))                       # [set][K, V]
    dm, dl, s = Dev(mass), i32(n - added), scratch(hv.kv_evict_scratch(nkv, cap, nset))
    d = cap if dcap is None else dcap
    kept = Dev(np.full((nset, nkv, d), -7, np.int32))
    if dcap is None:
        out, om, step = both, dm, 2 * one
    else:
        out = Dev(np.full((nset, 2, nkv, d, HD), 3, F16))
        om, step = Dev(np.full((nset, nkv, d), 5, F32)), 2 * nkv * d * HD
    hv.kv_evict(both.ptr, both.ptr + 2 * one, 2 * one, dm, cap, dl, added, out.ptr,
                out.ptr + 2 * nkv * d * HD, step, om, d, dl, kept if want_kept else 0, limit, keep, recent,
                nkv, HD, nset, s, stream)
    o = out.get(np.uint16, (nset, 2, nkv, d, HD))
    return o[:, 0], o[:, 1], om.get(F32, (nset, nkv, d)), kept.get(np.int32, (nset, nkv, d)), dl.get(np.int32)[0]


def check_evict(hv, k, v, mass, n, added, limit, keep, recent, dcap):
    nset, nkv, cap, _ = k.shape
    ko, vo, mo, kept, left = run_evict(hv, k, v, mass, n, added, limit, keep, recent, dcap)
    moved = n > limit
    assert left == (keep if moved else n)
    for i in range(nset):
        for h in range(nkv):
            idx = R.evict(mass[i, h], n, limit, keep, recent)
            m = len(idx)
            if dcap is not None or moved:
                assert np.array_equal(kept[i, h, :m], idx)
                assert (kept[i, h, m:] == -7).all()
            else:
                assert (kept[i, h] == -7).all()
            assert np.array_equal(ko[i, h, :m], k[i, h, idx].view(np.uint16))
            assert np.array_equal(vo[i, h, :m], v[i, h, idx].view(np.uint16))
            assert np.array_equal(bits(mo[i, h, :m]), bits(mass[i, h, idx]))
            if dcap is not None:                           # behind them: untouched
                assert (mo[i, h, m:] == 5).all()
                assert (ko[i, h, m:] == F16(3).view(np.uint16)).all()


def some_mass(g, *shape):
    m = np.exp(2 * g.standard_normal(shape)).astype(F32)
    m[g.random(shape) < 0.2] = 0
    m[g.random(shape) < 0.1] = F32(1.5)
    return m


@pytest.mark.parametrize("nset,nkv,n,limit,keep,recent", [
    (1, 1, 1, 1, 1, 0), (1, 1, 2, 1, 1, 0), (1, 1, 2, 1, 1, 1), (2, 3, 40, 32, 32, 8), (1, 2, 300, 256, 256, 32),
    (3, 2, 300, 299, 1, 0), (1, 8, 1000, 700, 512, 512), (1, 2, 1024, 1023, 1000, 0),
    (2, 1, 1025, 1024, 1024, 1), (1, 2, 4352, 4351, 4096, 1024), (1, 1, 20000, 9000, 8192, 100),
    (1, 1, 70000, 60000, 60000, 17), (36, 2, 352, 351, 320, 64), (1, 2, 100, 100, 50, 3), (2, 2, 0, 9, 5, 2)])
@pytest.mark.parametrize("place", ["in place", "apart"])
def test_eviction(hv, nset, nkv, n, limit, keep, recent, place):
    g = np.random.default_rng(n + keep)
    cap = max(n, limit) + 3
    k, v = cache(g, nset, nkv, cap)
    mass = some_mass(g, nset, nkv, cap)
    mass[..., n:] = np.inf                                 # of no position that is held
    dcap = None if place == "in place" else max(limit, n if n <= limit else keep) + 2
    check_evict(hv, k, v, mass, n, min(n, 1), limit, keep, recent, dcap)


@pytest.mark.parametrize("fill", ["equal", "nan", "signed", "sorted", "rising", "tiny"])
def test_eviction_of_unusual_masses(hv, fill):
    g = np.random.default_rng(31)
    n = 2500
    k, v = cache(g, 1, 2, n)
    mass = {"equal": np.ones((1, 2, n)), "nan": g.standard_normal((1, 2, n)),
            "signed": g.standard_normal((1, 2, n)).round(1), "sorted": np.arange(n, 0, -1.0) * np.ones((1, 2, 1)),
            "rising": np.arange(n) * np.ones((1, 2, 1)), "tiny": g.random((1, 2, n)) * 1e-42}[fill].astype(F32)
    if fill == "nan":
        mass[:, :, ::7] = np.nan
        mass[:, :, 3::50] = np.inf
        mass[:, :, 4::50] = -np.inf
    if fill == "signed":
        mass[mass == 0] = F32(-0.0)
        mass[:, :, ::31] = 0
    for keep in (200, 400, 2400):
        for dcap in (None, keep):
            check_evict(hv, k, v, mass, n, 0, keep, keep, 100, dcap)


def test_eviction_leaves_impossible_lengths_alone(hv):
    g = np.random.default_rng(32)
    k, v = cache(g, 1, 1, 50)
    mass = some_mass(g, 1, 1, 50)
    for n in (51, -1, 2 ** 31 - 1):
        ko, vo, mo, kept, left = run_evict(hv, k, v, mass, n, 0, 40, 30, 5)
        assert left == n and (kept == -7).all()
        assert np.array_equal(ko[0, 0], k[0, 0].view(np.uint16)) and np.array_equal(bits(mo), bits(mass))
    assert run_evict(hv, k, v, mass, 50, 1, 40, 30, 5, want_kept=False)[4] == 30


def test_offsets_past_32_bits(hv):
    """Heads and caches more than 2^32 bytes apart: a few rows at the front of each."""
    g = np.random.default_rng(33)
    nkv, group, n, cap = 9, 4, 700, 1 << 21
    head = cap * HD * 2                                     # bytes
    big = [Dev(nbytes=nkv * head) for _ in range(2)]
    k, v = cache(g, nkv, n)
    for d, x in zip(big, (k, v)):
        for h in range(nkv):
            hv.upload(d.ptr + h * head, np.ascontiguousarray(x[h]).ctypes.data, n * HD * 2)
    sc = Dev(np.array([SCALE], F32))
    # one row, and a batch over it as a prefix, by tiles and without
    q = queries(g, 1, nkv * group)
    dq, ctx, m, pos = Dev(q), Dev(nbytes=q.nbytes), Dev(nbytes=nkv * cap * 4), i32(n - 1)
    s = scratch(hv.attn_mass_scratch(nkv * group, group, cap, 1))
    hv.attn_decode_mass(dq, big[0], big[1], ctx, 0, m, sc, pos, nkv * group, HD, group, cap, s)
    want, tol, wm, mt = R.mass(q, k, v, n - 1, None, SCALE)
    near(ctx.get(F32, q.shape), want, tol)
    near(m.get(F32, (nkv, cap))[:, :n], wm, mt)
    del s
    for nseq in (2, 20):
        tk, tv = cache(g, nseq, nkv, 3)
        q = queries(g, nseq, nkv * group)
        dq, ctx, dt = Dev(q), Dev(nbytes=q.nbytes), [Dev(tk), Dev(tv)]
        s = scratch(hv.attn_shared_scratch(nkv * group, group, cap, 3, nseq, nseq))
        pl, tl = i32(n), i32([3] * nseq)
        hv.attn_shared(dq, big[0], big[1], cap, pl, dt[0], dt[1], 3, 0, tl, ctx, sc, nkv * group, HD, group,
                       nseq, nseq, s)
        near(ctx.get(F32, q.shape), *R.shared(q, k, v, n, tk, tv, None, [3] * nseq, SCALE))
    # thinned in place
    mass = some_mass(g, nkv, cap)
    dm, ln, s = Dev(mass), i32(n), scratch(hv.kv_evict_scratch(nkv, cap, 1))
    hv.kv_evict(big[0], big[1], 0, dm, cap, ln, 0, big[0], big[1], 0, dm, cap, ln, 0, 500, 300, 50, nkv, HD, 1, s)
    hv.synchronize()
    for h in range(nkv):
        got = np.empty((300, HD), np.uint16)
        hv.download(got.ctypes.data, big[1].ptr + h * head, got.nbytes)
        assert np.array_equal(got, v[h, R.evict(mass[h], n, 500, 300, 50)].view(np.uint16))


# ---- a run of them together ---------------------------------------------------------------

def test_a_thinned_prompt_shared_by_a_batch(hv):
    """A prompt's rows with their weights, its cache thinned into another, and a batch over what is
    left, on one stream without a wait between them."""
    g = np.random.default_rng(40)
    nkv, group, n, keep, nseq, tcap = 2, 4, 500, 160, 6, 9
    nq = nkv * group
    k, v = cache(g, nkv, n)
    q, q2 = queries(g, n, nq), queries(g, nseq, nq)
    tk, tv = cache(g, nseq, nkv, tcap)
    st = hv.stream_create()
    d = {x: Dev(y) for x, y in dict(k=k, v=v, q=q, q2=q2, tk=tk, tv=tv, sc=np.array([SCALE], F32),
                                    n=np.array([n], np.int32), tl=np.full(nseq, tcap, np.int32)).items()}
    ctx, ctx2, m = Dev(nbytes=q.nbytes), Dev(nbytes=q2.nbytes), Dev(nbytes=nkv * n * 4)
    kd, vd, md, kept = (Dev(nbytes=nkv * keep * b) for b in (256, 256, 4, 4))
    left = i32(0)
    ss = [scratch(x) for x in (hv.attn_mass_scratch(nq, group, n, n), hv.kv_evict_scratch(nkv, n, 1),
                               hv.attn_shared_scratch(nq, group, keep, tcap, nseq, nseq))]
    hv.synchronize()
    hv.attn_rows_mass(d["q"], d["k"], d["v"], ctx, 0, m, d["sc"], 0, nq, HD, group, n, n, ss[0], st)
    hv.kv_evict(d["k"], d["v"], 0, m, n, d["n"], 0, kd, vd, 0, md, keep, left, kept, keep, keep, 16, nkv, HD,
                1, ss[1], st)
    hv.attn_shared(d["q2"], kd, vd, keep, left, d["tk"], d["tv"], tcap, 0, d["tl"], ctx2, d["sc"], nq, HD,
                   group, nseq, nseq, ss[2], st)
    hv.stream_synchronize(st)
    mass = m.get(F32, (nkv, n))
    idx = np.stack([R.evict(mass[h], n, keep, keep, 16) for h in range(nkv)])
    assert np.array_equal(kept.get(np.int32, (nkv, keep)), idx)
    pk, pv = (np.stack([x[h, idx[h]] for h in range(nkv)]) for x in (k, v))
    near(ctx2.get(F32, q2.shape), *R.shared(q2, pk, pv, keep, tk, tv, None, [tcap] * nseq, SCALE))
    hv.stream_destroy(st)


# ---- the engine -----------------------------------------------------------------------------

def engine(arch, seed, cap, **kw):
    import limited
    import synth
    import w4format
    cfg = w4format.Config(arch)
    return limited.Engine(config=cfg, tensors=synth.iter_tensors(cfg, seed), quiet=True, max_context=cap,
                          kv_dtype="f16", **kw)


def prompt(e, seed, n):
    import synth
    return synth.prompt_ids(e.cfg, seed, n)


def layer(e, l, cap):
    c = e.cfg
    return [e._download(p, (c.n_kv, cap, HD), F16) for p in (e.KC[l], e.VC[l])]


@pytest.mark.parametrize("prefill", ["steps", "batched"])
def test_engine_with_a_bounded_cache(hv, prefill):
    """The first layer's K and V do not depend on attention: what the bounded cache holds are rows
    of the whole one, in order, the latest at the end. The last layer's context is attention over
    what its cache holds. The graph-replayed decode gives the direct one's tokens."""
    import synth
    arch = synth.tiny_arch(hidden=512, n_head=8, n_kv=2)
    n, keep, recent, cap = 500, 96, 24, 600
    a = engine(arch, 3, cap, fused=False, prefill=prefill, kv_keep=keep, kv_recent=recent)
    f = engine(arch, 3, cap, fused=False, prefill="batched")
    try:
        c, slots = a.cfg, keep + a.PREFILL_BATCH
        assert a.kv_cap == slots
        assert a.kv_bytes == c.n_layer * 2 * c.n_kv * slots * HD * 2
        ids = prompt(a, 3, n)
        la = a.logits(ids)
        f.logits(ids)
        assert np.isfinite(la).all()
        held = a._get_i32(a.d_held)
        assert keep <= held < slots
        whole = layer(f, 0, cap)
        for h in range(c.n_kv):
            k, v = (x[h].view(np.uint16) for x in layer(a, 0, slots))
            kw, vw = (x[h].view(np.uint16) for x in whole)
            where = {kw[i].tobytes() + vw[i].tobytes(): i for i in range(n)}
            at = [where[k[i].tobytes() + v[i].tobytes()] for i in range(held)]
            assert at == sorted(at) and len(set(at)) == held
            late = recent + held - keep
            assert at[-late:] == list(range(n - late, n))
        m = a._download(a._mass(c.n_layer - 1), (c.n_kv, slots), F32)[:, :held]
        assert np.isfinite(m).all() and (m >= 0).all() and (m > 0).any(1).all()
        if prefill == "steps":
            q, ctx = (a._download(x, (c.n_head, HD), F32) for x in (a.d_qkv, a.d_ctx))
            end = held
        else:
            r = (n - 1) % a.PREFILL_BATCH
            q, ctx = (a._download(a._pf[x] + r * c.n_head * HD * 4, (c.n_head, HD), F32) for x in ("q", "ctx"))
            end = held
        k, v = layer(a, c.n_layer - 1, slots)
        for h in range(c.n_head):
            want, tol = R.attend(q[h], k[h // c.group, :end], v[h // c.group, :end], float(a.attn_scale))[:2]
            near(ctx[h], want, tol)
        toks, _, _ = a.generate(ids[:300], 90, stop_on_eos=False)
        assert a.generate(ids[:300], 90, stop_on_eos=False, use_graph=True)[0] == toks
        assert a.generate(ids[:300], 90)[0] == toks
        for no in (a.profile_step, lambda: a._step_fused(0)):
            with pytest.raises(ValueError, match="kv_keep"):
                no()
        assert a.step_status() == 0
        s = a.score(ids)
        assert np.isfinite(s["logprob"]).all()
    finally:
        a.free()
        f.free()


def test_bounded_engine_past_the_reference_orders_16384(hv):
    """Room for 64 + 256 positions while the text goes on past what the reference-order attention
    can hold."""
    import synth
    a = engine(synth.tiny_arch(hidden=256, n_head=10, n_kv=2), 4, 17000, fused=False, prefill="batched",
               kv_keep=64, kv_recent=64)
    try:
        ids = prompt(a, 4, 16500)
        toks, _, _ = a.generate(ids, 8, stop_on_eos=False)
        assert len(toks) == 8 and a.kv_cap == 320
    finally:
        a.free()


def check_many_state(hv, e, ids, branches, plen):
    """The first layer's tails are the rows that the whole text's cache has there; the last layer's
    contexts are attention over prefix and tails as they stand."""
    c, mb, nseq = e.cfg, e._many, len(branches)
    tcap = mb["tcap"]
    got = lambda l, which: e._download(  # noqa: E731
        mb["tails"] + (2 * l + which) * nseq * c.n_kv * tcap * HD * 2, (nseq, c.n_kv, tcap, HD), F16)
    row0, tlen = (e._download(mb[x], (k,), np.int32) for x, k in (("row0", nseq + 1), ("tlen", nseq)))
    m = row0[-1]
    q, ctx = (e._download(e._pf[x], (m, c.n_head, HD), F32) for x in ("q", "ctx"))
    pk, pv = layer(e, c.n_layer - 1, e.kv_cap)
    near(ctx, *R.shared(q, pk, pv, plen, got(c.n_layer - 1, 0), got(c.n_layer - 1, 1), row0, tlen,
                        float(e.attn_scale)))
    return got(0, 0), got(0, 1), tlen


@pytest.mark.parametrize("keep", [None, 120])
def test_many_continuations(hv, keep):
    import synth
    arch = synth.tiny_arch(hidden=512, n_head=8, n_kv=2)
    cap = 512
    kw = dict(fused=False, kv_keep=keep) if keep else {}
    e = engine(arch, 5, cap, **kw)
    f = engine(arch, 5, cap, fused=False, prefill="batched")
    try:
        ids = prompt(e, 5, 400)
        g = np.random.default_rng(5)
        branches = [g.integers(0, e.cfg.vocab, n).tolist() for n in (0, 3, 17, 1, 40, 0)]
        max_new = 6
        got = e.generate_many(ids, branches, max_new, stop_on_eos=False)
        assert [len(x) for x in got] == [max_new] * 6 and got[0] == got[5]
        held = e._held if keep else len(ids) - 1
        tk, tv, tlen = check_many_state(hv, e, ids, branches, held)
        assert tlen.tolist() == [1 + len(b) + max_new - 1 for b in branches]
        for s, b in enumerate(branches):
            text = ids + b + got[s]
            f.logits(text)
            k, v = layer(f, 0, cap)
            at = slice(len(ids) - 1, len(ids) - 1 + tlen[s])
            assert np.array_equal(tk[s, :, :tlen[s]].view(np.uint16), k[:, at].view(np.uint16))
            assert np.array_equal(tv[s, :, :tlen[s]].view(np.uint16), v[:, at].view(np.uint16))
        assert e.generate_many(ids, branches, max_new, stop_on_eos=False) == got
        # other sizes after it, and one prompt token (no prefix at all)
        assert len(e.generate_many(ids[:1], [[5, 6]] * 9, 3, stop_on_eos=False)) == 9
        e.cfg.eos = got[1][2]
        stopped = e.generate_many(ids, branches, max_new)
        for a, b in zip(stopped, got):
            n = b.index(e.cfg.eos) + 1 if e.cfg.eos in b else max_new
            assert a == b[:n]
    finally:
        e.free()
        f.free()


def test_many_texts_scored(hv):
    """Over 256 rows in all, so several runs; the log probabilities are those of the logits, and a
    branch scored twice has the same ones."""
    import synth
    e = engine(synth.tiny_arch(hidden=512, n_head=8, n_kv=2), 6, 512)
    try:
        ids = prompt(e, 6, 100)
        g = np.random.default_rng(6)
        branches = [g.integers(0, e.cfg.vocab, n).tolist() for n in (5, 130, 1, 140, 9)] + [[7, 8, 9, 3, 2]]
        out = e.score_many(ids, branches)
        for b, o in zip(branches, out):
            assert o["logprob"].shape == o["entropy"].shape == (len(b),)
            assert np.isfinite(o["logprob"]).all() and (o["logprob"] < 0).all()
        rows = sum(len(b) for b in branches) - 256                   # of the second run
        x = e._download(e._sc["logits"], (rows, e.n_head_rows), F32).astype(np.float64)
        lp = x - x.max(1, keepdims=True)
        lp -= np.log(np.exp(lp).sum(1, keepdims=True))
        last = branches[-1]
        want = [lp[rows - len(last) + i, t] for i, t in enumerate(last)]
        # logits of size |x| are in f32: a log probability is off by a few steps of the largest
        assert np.abs(out[-1]["logprob"] - want).max() <= 16 * R.U * (np.abs(x).max() + 12)
        check_many_state(hv, e, ids, branches, len(ids) - 1)
        again = e.score_many(ids, branches)
        for a, b in zip(out, again):
            assert np.array_equal(bits(a["logprob"]), bits(b["logprob"]))
    finally:
        e.free()
