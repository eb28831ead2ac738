"""Attention over the 8-bit KV cache where blocks, or rows of the open block, differ from their
neighbours by many orders: each kernel (one token, few rows, long runs) against the 64-bit model
and bound of kv_q8_ref.py."""
import numpy as np
import pytest

import kv_q8_ref as R
from gpu_util import Dev
from test_gpu_kv_q8 import SCALE, i32, near, queries, rows, scratch

pytestmark = pytest.mark.gpu
F32 = np.float32
HD = 128

# (kv heads, group, pos0, ntok): long runs as one chunk, as a cluster and as chunks of a second
# launch; few rows whole and cut; one token
LONG = [(8, 8, 30, 220), (2, 5, 4000, 71), (1, 1, 15001, 200)]
FEW = [(2, 2, 210, 40), (8, 4, 1000, 8), (1, 4, 246, 4)]
ONE = [(2, 4, 249, 1), (8, 2, 2000, 1)]


def run(hv, ref, q, pos0, group):
    """The run q [ntok, nq, 128] at pos0 over the model's contents, other bytes 0xFF."""
    ntok, nq = q.shape[:2]
    ctx = Dev(np.zeros(q.shape, F32))
    hv.attn_rows_q8(Dev(q), Dev(ref.buffer(0xFF)), ctx, Dev(np.array([SCALE])), pos0, nq, HD,
                    group, ref.cap, ntok, scratch(hv, nq, group, ref.cap, ntok))
    return ctx.get(F32, q.shape)


def some(ntok, *more):
    return sorted({0, 1, ntok // 3, ntok // 2, ntok - 2, ntok - 1, *more} & set(range(ntok)))


@pytest.mark.parametrize("size", [1.0, 1e-6, 1e-12])
@pytest.mark.parametrize("nkv,group,pos0,ntok", LONG + FEW + ONE)
def test_blocks_whose_values_are_all_zero(hv, nkv, group, pos0, ntok, size):
    """They weigh in the sum of the weights and add nothing else, however small the rest is: one
    block, a whole chunk of them, the open block."""
    n = pos0 + ntok
    for zero in (slice(64, 96), slice(0, 32 * (n // 64)), slice(n // 32 * 32, n), slice(0, n)):
        g = np.random.default_rng(51)
        k, v = rows(g, n, nkv, 0.3)
        v *= F32(size)
        v[zero] = 0
        ref = R.Cache(nkv, n + 9)
        ref.write(k, v, 0)
        q = queries(g, ref, ntok, nkv * group)
        got = run(hv, ref, q, pos0, group)
        for t in some(ntok):
            near(got[t], *R.attention(q[t], ref.val, pos0 + t, group, float(SCALE)))


@pytest.mark.parametrize("nkv,group,pos0,ntok", LONG + FEW + ONE)
def test_blocks_of_values_further_apart_than_an_exponent(hv, nkv, group, pos0, ntok):
    """V of 1e20 beside V of 1e-20, in one chunk and in different ones: the small values add next
    to nothing, but their weights count."""
    n = pos0 + ntok
    for large in (lambda p: p // 32 % 2 == 0, lambda p: p < n // 2, lambda p: p >= n // 2,
                  lambda p: p // 32 == 1, lambda p: p >= n // 32 * 32):
        g = np.random.default_rng(52)
        k, v = rows(g, n, nkv, 0.3)
        big = large(np.arange(n))
        v *= np.where(big, 1e20, 1e-20).astype(F32)[:, None, None]
        ref = R.Cache(nkv, n + 9)
        ref.write(k, v, 0)
        q = queries(g, ref, ntok, nkv * group)
        q[:, 0] = 0                                            # equal weights
        got = run(hv, ref, q, pos0, group)
        for t in some(ntok):
            near(got[t], *R.attention(q[t], ref.val, pos0 + t, group, float(SCALE)))


@pytest.mark.parametrize("which", ["k", "v", "v up", "both"])
@pytest.mark.parametrize("nkv,group,pos0,ntok", [
    (8, 8, 30, 220), (2, 5, 4001, 94), (1, 1, 15024, 200), (2, 2, 210, 40), (8, 4, 992, 28),
    (1, 4, 224, 26), (2, 4, 249, 1)])
def test_open_rows_of_very_different_sizes(hv, nkv, group, pos0, ntok, which):
    """The open block's rows are f32: one that a query does not see, however large, takes nothing
    from those that it sees, and small ones keep their precision beside it."""
    n = pos0 + ntok
    first = n // 32 * 32
    assert n - first >= 24
    g = np.random.default_rng(53)
    k, v = rows(g, n, nkv, 0.3)
    up, down = F32(1e20), F32(1e-20)
    if which != "k":
        if which == "v":
            v *= down                                          # all small, then two large rows
        v[first + 3] *= down
        v[first + 4] = 0
        v[first + 18:first + 20] *= up
    if which in ("k", "both"):
        k[first + 3] *= down
        k[first + 18] *= F32(1e12)
    ref = R.Cache(nkv, n + 9)
    ref.write(k, v, 0)
    q = queries(g, ref, ntok, nkv * group)
    q[:, 0] = 0
    if which in ("k", "both"):
        q = np.clip(q, -8, 8)                                  # look for rows, not the large one
    got = run(hv, ref, q, pos0, group)
    for t in some(ntok, *(first + i - pos0 for i in (2, 3, 4, 5, 16, 17, 18, 19, 20))):
        near(got[t], *R.attention(q[t], ref.val, pos0 + t, group, float(SCALE)))


@pytest.mark.parametrize("nkv,group,pos0,ntok", [(8, 8, 30, 220), (2, 4, 210, 40), (2, 3, 249, 1)])
def test_queries_and_open_rows_up_to_the_largest_float(hv, nkv, group, pos0, ntok):
    n, nq = pos0 + ntok, nkv * group
    g = np.random.default_rng(55)
    top = np.finfo(F32).max
    k, v = rows(g, n, nkv, 0.3)
    k *= F32(3e-38)
    q = g.standard_normal((ntok, nq, HD)).astype(F32)
    q[:, ::2] *= F32(5e37)
    q[:, ::2, 5] = top
    q[:, 1] = 0
    q[:, 1, 7] = -top
    ref = R.Cache(nkv, n + 9)
    ref.write(k, v, 0)
    got = run(hv, ref, q, pos0, group)
    for t in some(ntok):
        near(got[t], *R.attention(q[t], ref.val, pos0 + t, group, float(SCALE)))


@pytest.mark.parametrize("which,bad", [("k", np.nan), ("k", -np.inf), ("k", np.inf),
                                       ("v", np.nan), ("v", np.inf)])
@pytest.mark.parametrize("nkv,group,cap", [(8, 8, 288), (1, 4, 288), (8, 3, 288), (1, 8, 40000)])
def test_open_rows_that_are_not_finite_lose_the_whole_context(hv, nkv, group, cap, which, bad):
    """As a complete block that holds one reads NaN throughout: every head of that kv head's
    group, in all its dimensions, from that position on, in each kernel."""
    n, at = 250, 237
    g = np.random.default_rng(54)
    k, v = rows(g, n, nkv, 0.3)
    (k if which == "k" else v)[at, -1, 77] = bad
    ref = R.Cache(nkv, cap)
    ref.write(k, v, 0)
    nq = nkv * group
    q = np.abs(g.standard_normal((220, nq, HD))).astype(F32)
    lost = np.arange(nq) // group == nkv - 1
    clean = ref.val.copy()
    clean[:, -1, at] = 0
    for ntok in (220, 40, 17):
        got = run(hv, ref, q[:ntok], n - ntok, group)
        for t in some(ntok, at - 1 - n + ntok, at - n + ntok):
            pos = n - ntok + t
            gone = lost & (pos >= at)
            assert np.isnan(got[t][gone]).all()
            want, tol = R.attention(q[t], clean, pos, group, float(SCALE))
            near(got[t][~gone], want[~gone], tol[~gone])
    kv, s, ctx = Dev(ref.buffer(0xFF)), scratch(hv, nq, group, cap), Dev(nbytes=nq * HD * 4)
    for pos in (at - 1, at, n - 1):
        hv.attn_decode_q8(Dev(q[0]), kv, ctx, Dev(np.array([SCALE])), i32(pos), nq, HD, group, cap,
                          s)
        got = ctx.get(F32, (nq, HD))
        gone = lost & (pos >= at)
        assert np.isnan(got[gone]).all()
        want, tol = R.attention(q[0], clean, pos, group, float(SCALE))
        near(got[~gone], want[~gone], tol[~gone])


@pytest.mark.parametrize("nkv,group,cap", [(8, 8, 13000), (1, 5, 40000), (2, 6, 20000),
                                           (3, 7, 12321), (2, 4, 20000)])
def test_decode_over_caches_too_long_for_a_cluster(hv, nkv, group, cap):
    """The form with bulk copies, whose chunks meet in the scratch, at any length of the cache."""
    nq = nkv * group
    g = np.random.default_rng(56)
    k, v = rows(g, cap, nkv, 0.3)
    ref = R.Cache(nkv, cap)
    s, at = scratch(hv, nq, group, cap), 0
    for n in (1, 32, 45, 300, 4225, cap):
        ref.write(k[at:n], v[at:n], at)
        at = n
        kv, q, ctx = Dev(ref.buffer(0xFF)), queries(g, ref, 1, nq), Dev(nbytes=nq * HD * 4)
        for pos in sorted({n - 1, n // 2}):
            hv.attn_decode_q8(Dev(q), kv, ctx, Dev(np.array([SCALE])), i32(pos), nq, HD, group,
                              cap, s)
            near(ctx.get(F32, (nq, HD)), *R.attention(q[0], ref.val, pos, group, float(SCALE)))


def test_engine_decodes_past_16384_positions(hv):
    """A group of 5 query heads over a cache beyond the reference-order attention's reach: the last
    layer's context against its cache as read back, over the edge of 16384 and of a block."""
    import limited
    import synth
    import w4format
    cfg = w4format.Config(synth.tiny_arch(hidden=256, n_head=10, n_kv=2))
    n, cap = 16381, 16500
    e = limited.Engine(config=cfg, tensors=synth.iter_tensors(cfg, 4), quiet=True, max_context=cap,
                       kv_dtype="q8", fused=False)
    try:
        g = np.random.default_rng(57)
        for kv in e.KC:
            k, v = rows(g, n, cfg.n_kv, 0.3)
            hv.kv_rows_q8(Dev(k), Dev(v), cfg.n_kv * HD, kv, 0, cfg.n_kv, HD, cap, n)
        e._set_i32(e.d_pos, n)
        e._set_i32(e.d_tok, 7)
        e._set_i32(e.d_step, 0)
        for pos in range(n, n + 8):
            e._step_eager()
            hv.synchronize()
            assert np.isfinite(e.download_logits()).all()
            if pos in (n, 16383, 16384, n + 7):
                ko, vo = (Dev(nbytes=(pos + 1) * cfg.n_kv * HD * 4) for _ in range(2))
                hv.kv_read_q8(e.KC[-1], ko, vo, 0, cfg.n_kv, HD, cap, pos + 1)
                val = np.stack([x.get(F32, (pos + 1, cfg.n_kv, HD)) for x in (ko, vo)]).swapaxes(1, 2)
                q = e._download(e.d_qkv, (cfg.n_head, HD), F32)
                near(e._download(e.d_ctx, (cfg.n_head, HD), F32),
                     *R.attention(q, val, pos, cfg.group, float(e.attn_scale)))
            e._argmax_into_next()
        hv.synchronize()
        assert e._get_i32(e.d_pos) == n + 8
    finally:
        e.free()


@pytest.mark.parametrize("nkv,group,pos0,ntok", [(8, 5, 11, 231), (8, 8, 30, 220), (2, 4, 60, 40),
                                                 (2, 3, 81, 1)])
def test_zeros_that_are_all_a_row_sees_of_a_block(hv, nkv, group, pos0, ntok):
    """The first rows of a block are zeros that the queries look for; the rest of it, of the usual
    size, is behind the queries. What little weight the other blocks have is theirs in full."""
    n = pos0 + ntok
    g = np.random.default_rng(58)
    k, v = rows(g, n, nkv, 0.3)
    v[64:82] = 0
    ref = R.Cache(nkv, n + 9)
    ref.write(k, v, 0)
    q = np.repeat(ref.val[0, :, 75], group, 0)[None].repeat(ntok, 0) * 1.5
    q = (q + 0.3 * g.standard_normal(q.shape)).astype(F32)
    got = run(hv, ref, q, pos0, group)
    for t in some(ntok, *(p - pos0 for p in (75, 76, 80, 81, 82, 95, 96))):
        near(got[t], *R.attention(q[t], ref.val, pos0 + t, group, float(SCALE)))


@pytest.mark.parametrize("nkv,group,pos0,ntok", [(8, 7, 1, 13), (8, 5, 6, 11), (1, 2, 0, 28),
                                                 (2, 4, 26, 1), (2, 8, 96, 29)])
def test_few_open_rows_of_every_size(hv, nkv, group, pos0, ntok):
    """V from 1e-28 to 1e28, row by row, and all of it tiny behind a zero that has the weight."""
    n = pos0 + ntok
    for seed in range(8):
        g = np.random.default_rng(600 + seed)
        k, v = rows(g, n, nkv, 0.3)
        if seed < 4:
            v *= (10.0 ** g.uniform(-28, 28, n)).astype(F32)[:, None, None]
        else:
            v *= F32(2e-27)
            v[0] = 0
        ref = R.Cache(nkv, n + 9)
        ref.write(k, v, 0)
        q = queries(g, ref, ntok, nkv * group)
        if seed < 4:
            q[:, ::3] = 0
        else:
            q = (np.repeat(ref.val[0, :, 0], group, 0)[None].repeat(ntok, 0) * 1.2 + 0.2 * q).astype(F32)
        got = run(hv, ref, q, pos0, group)
        for t in range(ntok):
            near(got[t], *R.attention(q[t], ref.val, pos0 + t, group, float(SCALE)))
