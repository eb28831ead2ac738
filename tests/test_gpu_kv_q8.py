"""The 8-bit KV cache on a B200: writing (one row, runs, with the head norms and rotation in
the same pass), reading back, attention of one token and of runs, and the engine over it,
against the numpy model of kv_q8_ref.py."""
import numpy as np
import pytest

import hv_oracle as O
import kv_q8_ref as R
import synth
import w4format
from gpu_util import Dev, bits

pytestmark = pytest.mark.gpu
F32 = np.float32
HD = 128


def rows(g, n, nkv, spread=1.0):
    k = (g.standard_normal((n, nkv, HD)) * np.exp(spread * g.standard_normal((1, nkv, HD))))
    return k.astype(F32), g.standard_normal((n, nkv, HD)).astype(F32)


def i32(x):
    return Dev(np.array([x], np.int32))


def new_cache(hv, nkv, cap, fill=0):
    n = hv.kv_q8_size(nkv, HD, cap)
    (_, _, held, _), _ = R.parts(nkv, cap)
    b = np.full(n, fill, np.uint8)
    b[held:] = 0
    return Dev(b)


def write(hv, kv, k, v, pos0, cap):
    nkv = k.shape[1]
    hv.kv_rows_q8(Dev(k), Dev(v), nkv * HD, kv, pos0, nkv, HD, cap, len(k))


def read(hv, kv, nkv, cap, pos0=0, n=None):
    n = cap - pos0 if n is None else n
    ko, vo = (Dev(nbytes=n * nkv * HD * 4) for _ in range(2))
    hv.kv_read_q8(kv, ko, vo, pos0, nkv, HD, cap, n)
    out = np.stack([x.get(F32, (n, nkv, HD)) for x in (ko, vo)])
    return out.swapaxes(1, 2)                                  # [2, nkv, n, 128]


def same(a, b):
    """Equal bit for bit, any NaN counting as any other."""
    return np.array_equal(np.where(np.isnan(a), 0, bits(a)), np.where(np.isnan(b), 0, bits(b)))


def check_buffer(kv, ref):
    """Codes, scales, open rows and length of the device buffer against the model's."""
    (a, b, c, end), nblk = R.parts(ref.nkv, ref.cap)
    got, want = kv.get(np.uint8), ref.buffer()
    closed = ref.held // R.BLK
    cut = lambda x: x[:a].reshape(ref.nkv, nblk, 2, 4096)[:, :closed]  # noqa: E731
    assert np.array_equal(cut(got), cut(want))
    sc = lambda x: x[a:a + ref.nkv * nblk * 8].view(F32).reshape(ref.nkv, nblk, 2)[:, :closed]  # noqa: E731
    assert same(sc(got), sc(want))
    if ref.held:
        n = (ref.held - 1) % R.BLK + 1
        tl = lambda x: x[b:c].view(F32).reshape(ref.nkv, 2, 32, HD)[:, :, :n]  # noqa: E731
        assert same(tl(got), tl(want))
    assert np.array_equal(got[c:c + 8 * ref.nkv], want[c:c + 8 * ref.nkv])


@pytest.mark.parametrize("nkv,cap,cuts", [
    (1, 1, [1]), (2, 40, [1, 1, 30, 1]), (8, 64, [64]), (3, 200, [5, 27, 32, 65, 1, 31, 39]),
    (8, 97, [33, 63, 1]), (2, 4352, [4096, 128, 1, 100])])
def test_rows_are_quantised_as_written(hv, nkv, cap, cuts):
    g = np.random.default_rng(cap)
    k, v = rows(g, sum(cuts), nkv)
    ref, kv, at = R.Cache(nkv, cap), new_cache(hv, nkv, cap, 0xFF), 0
    for n in cuts:
        ref.write(k[at:at + n], v[at:at + n], at)
        if n == 1:
            hv.kv_append_q8(Dev(k[at]), Dev(v[at]), kv, i32(at), nkv, HD, cap)
        else:
            write(hv, kv, k[at:at + n], v[at:at + n], at, cap)
        at += n
        check_buffer(kv, ref)
    assert same(read(hv, kv, nkv, cap), ref.val)
    if at > 3:
        assert same(read(hv, kv, nkv, cap, 3, at - 3), ref.val[:, :, 3:at])


def test_one_row_at_a_time_equals_one_run(hv):
    nkv, cap, n = 2, 100, 97
    k, v = rows(np.random.default_rng(4), n, nkv)
    a, b = new_cache(hv, nkv, cap), new_cache(hv, nkv, cap, 0x55)
    write(hv, a, k, v, 0, cap)
    for t in range(n):
        hv.kv_append_q8(Dev(k[t]), Dev(v[t]), b, i32(t), nkv, HD, cap)
    assert same(read(hv, a, nkv, cap), read(hv, b, nkv, cap))


def test_going_back_and_gaps(hv):
    nkv, cap = 2, 256
    g = np.random.default_rng(5)
    ref, kv = R.Cache(nkv, cap), new_cache(hv, nkv, cap)
    for pos0, n in ((0, 100), (90, 3),       # back inside the open block
                    (96, 1), (95, 4),        # over the edge of the last block and back
                    (40, 1),                 # into a complete block: reopened from its codes
                    (41, 60), (0, 32), (31, 1), (5, 2), (0, 200), (64, 64),
                    (130, 5),                # a gap: 128 are held
                    (128, 128), (10, 1), (200, 1)):
        k, v = rows(g, n, nkv)
        ref.write(k, v, pos0)
        if n == 1:
            hv.kv_append_q8(Dev(k[0]), Dev(v[0]), kv, i32(pos0), nkv, HD, cap)
        else:
            write(hv, kv, k, v, pos0, cap)
        check_buffer(kv, ref)
        assert same(read(hv, kv, nkv, cap), ref.val), (pos0, n)


def test_append_outside_the_cache_writes_nothing(hv):
    nkv, cap = 2, 64
    k, v = rows(np.random.default_rng(6), 10, nkv)
    kv = new_cache(hv, nkv, cap)
    write(hv, kv, k, v, 0, cap)
    before = kv.get(np.uint8)
    for p in (-1, 64, 1 << 30, -(1 << 31), 11):
        hv.kv_append_q8(Dev(k[0]), Dev(v[0]), kv, i32(p), nkv, HD, cap)
        assert np.array_equal(kv.get(np.uint8), before)


def test_blocks_of_hard_values(hv):
    """Zeros, one non-finite value, the largest and the smallest floats, halves of a step."""
    nkv, cap = 1, 256
    k, v = rows(np.random.default_rng(7), cap, nkv)
    k[0:32] = 0
    k[40, 0, 7] = np.nan
    k[70, 0, 127] = np.inf
    v[100, 0, 0] = -np.inf
    k[128:160] = np.ldexp(k[128:160], -140).astype(F32)              # subnormals
    k[160:192] *= F32(3e38) / np.abs(k[160:192]).max()
    k[192] = (np.arange(128) - 63.5).astype(F32)                      # ties at scale 1
    k[192, 0, 0], k[193:224] = 127, 0
    v[224:256] = F32(1e-45)
    ref, kv = R.Cache(nkv, cap), new_cache(hv, nkv, cap)
    ref.write(k, v, 0)
    write(hv, kv, k, v, 0, cap)
    check_buffer(kv, ref)
    got = read(hv, kv, nkv, cap)
    assert same(got, ref.val)
    assert np.isnan(got[0, 0, 32:96]).all() and np.isnan(got[1, 0, 96:128]).all()


def test_strided_rows(hv):
    nkv, cap, n, ld = 3, 80, 50, 7 * HD
    g = np.random.default_rng(8)
    src = g.standard_normal((n, ld)).astype(F32)
    k, v = src[:, HD:4 * HD].reshape(n, 3, HD), src[:, 4 * HD:].reshape(n, 3, HD)
    d, kv, ref = Dev(src), new_cache(hv, nkv, cap), R.Cache(nkv, cap)
    hv.kv_rows_q8(int(d) + 4 * HD, int(d) + 16 * HD, ld, kv, 0, nkv, HD, cap, n)
    ref.write(k, v, 0)
    assert same(read(hv, kv, nkv, cap), ref.val)


@pytest.mark.parametrize("nq,nkv,pos0,ntok", [(8, 2, 0, 40), (4, 4, 37, 91), (5, 1, 31, 1),
                                              (16, 8, 64, 32)])
def test_qk_rows_is_qk_rows_then_the_write(hv, nq, nkv, pos0, ntok):
    cap, eps = 160, 1e-5
    g = np.random.default_rng(pos0 + ntok)
    qkv = g.standard_normal((ntok, (nq + 2 * nkv) * HD)).astype(F32)
    qn, kn = ((1 + 0.01 * g.standard_normal(HD)).astype(F32) for _ in range(2))
    cos_t, sin_t = (x.astype(F32) for x in O.rope_tables(cap, HD, 1e6))
    dev = [Dev(x) for x in (qkv, qn, kn, cos_t, sin_t)]
    hk, hvv = rows(g, pos0, nkv) if pos0 else (None, None)
    kv, ref = new_cache(hv, nkv, cap), R.Cache(nkv, cap)
    if pos0:
        write(hv, kv, hk, hvv, 0, cap)
        ref.write(hk, hvv, 0)
    qo, qf = Dev(nbytes=ntok * nq * HD * 4), Dev(nbytes=ntok * nq * HD * 4)
    kf, vf = Dev(nbytes=nkv * cap * HD * 4), Dev(nbytes=nkv * cap * HD * 4)
    hv.qk_rows_q8(*dev, pos0, qo, kv, nq, nkv, HD, cap, eps, ntok)
    hv.qk_rows(*dev, pos0, qf, kf, vf, nq, nkv, HD, cap, eps, ntok)
    assert np.array_equal(bits(qo.get(F32)), bits(qf.get(F32)))
    k32, v32 = (x.get(F32, (nkv, cap, HD))[:, pos0:pos0 + ntok].swapaxes(0, 1)
                for x in (kf, vf))
    ref.write(np.ascontiguousarray(k32), np.ascontiguousarray(v32), pos0)
    check_buffer(kv, ref)


# ---- attention -----------------------------------------------------------------------

SCALE = F32(1.0 / np.sqrt(HD))


def filled(hv, seed, nkv, n, cap, look=3.0):
    """A cache of n positions whose other bytes are 0xFF (NaN scales, NaN rows)."""
    g = np.random.default_rng(seed)
    k, v = rows(g, n, nkv, 0.3)
    ref = R.Cache(nkv, cap)
    ref.write(k, v, 0)
    return g, ref, Dev(ref.buffer(0xFF))


def queries(g, ref, ntok, nq):
    q = g.standard_normal((ntok, nq, HD))
    n, group = ref.held, nq // ref.nkv
    for h in range(nq):                         # weights that are not flat
        q[:, h] += 1.5 * np.nan_to_num(ref.val[0, h // group, g.integers(0, n)])
    return q.astype(F32)


def scratch(hv, nq, group, cap, ntok=1):
    return Dev(nbytes=hv.attn_q8_scratch(nq, group, cap, ntok))


def near(got, want, tol):
    off = np.abs(got.astype(np.float64) - want)
    assert np.isfinite(got).all()
    assert (off <= tol).all(), float((off / tol).max())


@pytest.mark.parametrize("nkv,group,n", [
    (1, 1, 1), (2, 4, 2), (8, 2, 31), (8, 4, 32), (8, 8, 33), (2, 5, 63), (1, 3, 64), (4, 6, 65),
    (2, 7, 97), (8, 2, 300), (1, 8, 1000), (8, 4, 4225), (3, 4, 2048), (1, 4, 9000)])
def test_decode_attention(hv, nkv, group, n):
    nq, cap = nkv * group, n + 37
    g, ref, kv = filled(hv, n + group, nkv, n, cap)
    q, ctx = queries(g, ref, 1, nq), Dev(np.full((nq, HD), 7, F32))
    s = scratch(hv, nq, group, cap)
    for pos in sorted({n - 1, n // 2, 0, max(0, n - 33)}):     # whole and part of the cache
        hv.attn_decode_q8(Dev(q), kv, ctx, Dev(np.array([SCALE])), i32(pos), nq, HD, group, cap,
                          s)
        near(ctx.get(F32, (nq, HD)), *R.attention(q[0], ref.val, pos, group, float(SCALE)))


@pytest.mark.parametrize("nkv,group,pos0,ntok", [
    (1, 1, 0, 1), (2, 4, 0, 33), (8, 2, 256, 44), (2, 5, 31, 70), (4, 8, 100, 129), (1, 3, 5, 200),
    (8, 4, 992, 64), (2, 1, 0, 256), (1, 8, 3000, 17), (2, 4, 4000, 3), (2, 7, 511, 1),
    (8, 4, 1000, 32), (8, 2, 0, 256), (5, 3, 700, 40), (1, 1, 9000, 2), (40, 1, 2000, 5)])
def test_rows_attention(hv, nkv, group, pos0, ntok):
    nq, n = nkv * group, pos0 + ntok
    cap = n + 50
    g, ref, kv = filled(hv, n + group, nkv, n, cap)
    q, ctx = queries(g, ref, ntok, nq), Dev(np.full((ntok + 1, nq, HD), 7, F32))
    hv.attn_rows_q8(Dev(q), kv, ctx, Dev(np.array([SCALE])), pos0, nq, HD, group, cap, ntok,
                    scratch(hv, nq, group, cap, ntok))
    got = ctx.get(F32, (ntok + 1, nq, HD))
    assert (got[ntok] == 7).all()                              # rows behind the last stay
    for t in {0, 1, ntok // 2, ntok - 2, ntok - 1} & set(range(ntok)):
        near(got[t], *R.attention(q[t], ref.val, pos0 + t, group, float(SCALE)))
    # the same rows over the cache when it holds more positions: still causal
    if ntok > 4:
        m = ntok - 4
        part = Dev(np.full((m, nq, HD), 7, F32))
        hv.attn_rows_q8(Dev(q), kv, part, Dev(np.array([SCALE])), pos0, nq, HD, group, cap, m,
                        scratch(hv, nq, group, cap, m))
        near(part.get(F32, (m, nq, HD))[m - 1],
             *R.attention(q[m - 1], ref.val, pos0 + m - 1, group, float(SCALE)))


def test_positions_not_held_give_nan(hv):
    nkv, group, n, cap = 2, 4, 40, 64
    nq = nkv * group
    g, ref, kv = filled(hv, 1, nkv, n, cap)
    q, sc = queries(g, ref, 4, nq), Dev(np.array([SCALE]))
    for pos in (-1, 40, 63, 64, 1 << 30, -(1 << 31)):
        ctx = Dev(np.zeros((nq, HD), F32))
        hv.attn_decode_q8(Dev(q[0]), kv, ctx, sc, i32(pos), nq, HD, group, cap,
                          scratch(hv, nq, group, cap))
        assert np.isnan(ctx.get(F32)).all(), pos
    ctx = Dev(np.zeros((4, nq, HD), F32))
    hv.attn_rows_q8(Dev(q), kv, ctx, sc, 38, nq, HD, group, cap, 4,
                    scratch(hv, nq, group, cap, 4))
    got = ctx.get(F32, (4, nq, HD))
    assert np.isnan(got[2:]).all()
    for t in (0, 1):
        near(got[t], *R.attention(q[t], ref.val, 38 + t, group, float(SCALE)))
    empty = new_cache(hv, nkv, cap, 0xFF)
    hv.attn_decode_q8(Dev(q[0]), empty, ctx, sc, i32(0), nq, HD, group, cap,
                      scratch(hv, nq, group, cap))
    assert np.isnan(ctx.get(F32, (4, nq, HD))[0]).all()


@pytest.mark.parametrize("size", [1e-20, 1.0, 1e4, 1e18])
def test_sizes_of_q_and_k(hv, size):
    """q k^T is what counts: q as large as k is small, and the other way round."""
    nkv, group, n, cap = 2, 4, 150, 160
    g = np.random.default_rng(11)
    k, v = rows(g, n, nkv, 0.3)
    ref = R.Cache(nkv, cap)
    ref.write((k / F32(size)).astype(F32), (v * F32(size)).astype(F32), 0)
    kv, q = Dev(ref.buffer(0xFF)), (g.standard_normal((1, 8, HD)) * size).astype(F32)
    ctx = Dev(np.zeros((8, HD), F32))
    hv.attn_decode_q8(Dev(q), kv, ctx, Dev(np.array([SCALE])), i32(n - 1), 8, HD, group, cap,
                      scratch(hv, 8, group, cap))
    near(ctx.get(F32, (8, HD)), *R.attention(q[0], ref.val, n - 1, group, float(SCALE)))
    q3 = np.repeat(q, 3, 0)
    ctx = Dev(np.zeros((3, 8, HD), F32))
    hv.attn_rows_q8(Dev(q3), kv, ctx, Dev(np.array([SCALE])), n - 3, 8, HD, group, cap, 3,
                    scratch(hv, 8, group, cap, 3))
    near(ctx.get(F32, (3, 8, HD))[2], *R.attention(q[0], ref.val, n - 1, group, float(SCALE)))


def test_steep_weights_and_bad_queries(hv):
    """Scores far apart (one weight takes all), a zero query (all weights equal), a NaN and an
    infinity in one head's query: only that head's context is lost."""
    nkv, group, n, cap = 1, 4, 333, 352
    g, ref, kv = filled(hv, 12, nkv, n, cap)
    q = queries(g, ref, 1, 4)
    q[0, 0] = ref.val[0, 0, 200] * 30
    q[0, 1] = 0
    sc = Dev(np.array([SCALE]))
    for bad in (None, np.nan, np.inf):
        if bad is not None:
            q[0, 2, 5] = bad
        for ntok in (0, 2):                       # 0: the decode call
            qq = np.repeat(q, max(1, ntok), 0)
            ctx = Dev(np.zeros((max(1, ntok), 4, HD), F32))
            if ntok:
                hv.attn_rows_q8(Dev(qq), kv, ctx, sc, n - ntok, 4, HD, group, cap, ntok,
                                scratch(hv, 4, group, cap, ntok))
            else:
                hv.attn_decode_q8(Dev(qq), kv, ctx, sc, i32(n - 1), 4, HD, group, cap,
                                  scratch(hv, 4, group, cap))
            got = ctx.get(F32, (max(1, ntok), 4, HD))[-1]
            live = [0, 1, 3] if bad is not None else [0, 1, 2, 3]
            want, tol = R.attention(np.nan_to_num(q[0], posinf=0), ref.val, n - 1, group,
                                    float(SCALE))
            near(got[live], want[live], tol[live])
            if bad is not None:
                assert np.isnan(got[2]).all()


def test_a_poisoned_block_poisons_what_reads_it(hv):
    nkv, group, cap = 1, 2, 128
    g = np.random.default_rng(13)
    k, v = rows(g, 100, nkv, 0.3)
    v[70, 0, 3] = np.inf
    ref, sc = R.Cache(nkv, cap), Dev(np.array([SCALE]))
    ref.write(k, v, 0)
    kv, q, ctx = Dev(ref.buffer()), g.standard_normal((2, HD)).astype(F32), Dev(nbytes=1024)
    for pos, lost in ((63, False), (64, True), (99, True)):
        hv.attn_decode_q8(Dev(q), kv, ctx, sc, i32(pos), 2, HD, group, cap,
                          scratch(hv, 2, group, cap))
        got = ctx.get(F32, (2, HD))
        assert np.isnan(got).all() if lost else np.isfinite(got).all(), pos
    out = Dev(np.zeros((4, 2, HD), F32))
    hv.attn_rows_q8(Dev(np.stack([q] * 4)), kv, out, sc, 62, 2, HD, group, cap, 4,
                    scratch(hv, 2, group, cap, 4))
    got = out.get(F32, (4, 2, HD))
    assert np.isfinite(got[:2]).all() and np.isnan(got[2:]).all()


def test_open_rows_that_are_not_finite_reach_only_who_sees_them(hv):
    """Rows of the open block stay f32: a NaN or infinity in one is seen from its position on."""
    nkv, group, cap, n = 1, 4, 128, 60
    g = np.random.default_rng(16)
    k, v = rows(g, n, nkv, 0.3)
    v[45, 0, 7], k[50, 0, 9], v[58, 0, 0] = np.inf, np.nan, np.nan
    ref, sc = R.Cache(nkv, cap), Dev(np.array([SCALE]))
    ref.write(k, v, 0)
    kv = Dev(ref.buffer(0xFF))
    q = g.standard_normal((30, 4, HD)).astype(F32)
    out, s = Dev(np.zeros((30, 4, HD), F32)), scratch(hv, 4, group, cap, 30)
    hv.attn_rows_q8(Dev(q), kv, out, sc, 30, 4, HD, group, cap, 30, s)
    got = out.get(F32, (30, 4, HD))
    for t in (0, 1, 2, 14):
        near(got[t], *R.attention(q[t], ref.val, 30 + t, group, float(SCALE)))
    for t in range(15, 30):
        assert not np.isfinite(got[t][:, 7]).any()
        assert t < 20 or np.isnan(got[t]).all()
    one = Dev(np.zeros((4, HD), F32))
    for pos, lost in ((44, False), (45, True), (59, True)):
        hv.attn_decode_q8(Dev(q[0]), kv, one, sc, i32(pos), 4, HD, group, cap, s)
        x = one.get(F32, (4, HD))
        assert (not np.isfinite(x[:, 7]).any()) if lost else np.isfinite(x).all(), pos


@pytest.mark.parametrize("n0,cap", [(30, 200), (1010, 4000), (4000, 20000)])
def test_captured_decode_follows_the_device_position(hv, n0, cap):
    """Append and attention captured once, replayed while *pos moves over block edges, equal
    to direct calls; two graphs with a scratch each, on two streams."""
    nkv, group = 2, 4
    nq = nkv * group
    g = np.random.default_rng(14)
    k, v = rows(g, n0 + 40, nkv)
    q = g.standard_normal((nq, HD)).astype(F32)
    dq, sc = Dev(q), Dev(np.array([SCALE]))
    want = []
    kv = new_cache(hv, nkv, cap)
    write(hv, kv, k[:n0], v[:n0], 0, cap)
    s = scratch(hv, nq, group, cap)
    for t in range(n0, n0 + 40):
        ctx = Dev(nbytes=nq * HD * 4)
        hv.kv_append_q8(Dev(k[t]), Dev(v[t]), kv, i32(t), nkv, HD, cap)
        hv.attn_decode_q8(dq, kv, ctx, sc, i32(t), nq, HD, group, cap, s)
        want.append(ctx.get(F32))
    lanes = []
    for _ in range(2):
        L = dict(kv=new_cache(hv, nkv, cap), s=scratch(hv, nq, group, cap), pos=i32(n0),
                 k=Dev(k[0]), v=Dev(v[0]), ctx=Dev(nbytes=nq * HD * 4), st=hv.stream_create())
        write(hv, L["kv"], k[:n0], v[:n0], 0, cap)
        hv.synchronize()
        hv.capture_begin(L["st"])
        hv.kv_append_q8(L["k"], L["v"], L["kv"], L["pos"], nkv, HD, cap, L["st"])
        hv.attn_decode_q8(dq, L["kv"], L["ctx"], sc, L["pos"], nq, HD, group, cap, L["s"],
                          L["st"])
        L["graph"] = hv.capture_end(L["st"])
        L["exec"] = hv.graph_instantiate(L["graph"])
        lanes.append(L)
    for i, t in enumerate(range(n0, n0 + 40)):
        for L in lanes:
            L["k"].put(k[t])
            L["v"].put(v[t])
            L["pos"].put(np.array([t], np.int32))
        hv.synchronize()
        for L in lanes:
            hv.graph_launch(L["exec"], L["st"])
        for L in lanes:
            assert np.array_equal(bits(L["ctx"].get(F32)), bits(want[i])), t
    for L in lanes:
        hv.graph_destroy(L["graph"], L["exec"])
        hv.stream_destroy(L["st"])


def test_same_call_same_bits(hv):
    nkv, group, n = 8, 4, 3000
    g, ref, kv = filled(hv, 15, nkv, n, n)
    q, sc = queries(g, ref, 20, 32), Dev(np.array([SCALE]))
    s, s2, out = scratch(hv, 32, group, n), scratch(hv, 32, group, n, 20), []
    for _ in range(3):
        a, b = Dev(nbytes=32 * HD * 4), Dev(nbytes=20 * 32 * HD * 4)
        hv.attn_decode_q8(Dev(q[0]), kv, a, sc, i32(n - 1), 32, HD, group, n, s)
        hv.attn_rows_q8(Dev(q), kv, b, sc, n - 20, 32, HD, group, n, 20, s2)
        out.append((bits(a.get(F32)), bits(b.get(F32))))
    for a, b in out[1:]:
        assert np.array_equal(a, out[0][0]) and np.array_equal(b, out[0][1])


# Runs of 2^21 (row, position) pairs and more with over 64 rows a head take a kernel of their own.

@pytest.mark.parametrize("nkv,group,pos0,ntok", [
    (1, 1, 15001, 200), (2, 5, 4000, 71), (4, 8, 100, 250), (8, 8, 0, 200), (1, 3, 5, 1000),
    (8, 4, 31, 257), (2, 1, 9300, 129), (1, 8, 9000, 33), (5, 7, 1023, 65), (8, 2, 3840, 256)])
def test_long_runs_attention(hv, nkv, group, pos0, ntok):
    nq, n = nkv * group, pos0 + ntok
    assert ntok * group > 64 and ntok * nq * n >= 1 << 21
    cap = n + 50
    g, ref, kv = filled(hv, n + group, nkv, n, cap)
    q, ctx = queries(g, ref, ntok, nq), Dev(np.full((ntok + 1, nq, HD), 7, F32))
    s = scratch(hv, nq, group, cap, ntok)
    for _ in range(2):                                         # the scratch is ready again
        hv.attn_rows_q8(Dev(q), kv, ctx, Dev(np.array([SCALE])), pos0, nq, HD, group, cap, ntok,
                        s)
    got = ctx.get(F32, (ntok + 1, nq, HD))
    assert (got[ntok] == 7).all()
    for t in {0, 1, ntok // 2, ntok - 2, ntok - 1}:
        near(got[t], *R.attention(q[t], ref.val, pos0 + t, group, float(SCALE)))


def test_long_run_over_positions_that_are_lost_or_not_held(hv):
    """A poisoned block, non-finite rows of the open block and rows past the length, seen from
    their positions on; a NaN query and an infinite one lose their own rows only."""
    nkv, group, cap, pos0, n = 8, 8, 288, 40, 250
    nq, ntok = nkv * group, 230                                # positions 250 .. 269: not held
    assert ntok * nq * (pos0 + ntok) >= 1 << 21
    g = np.random.default_rng(21)
    k, v = rows(g, n, nkv, 0.3)
    v[170, 2, 3] = np.inf                                      # block 160 .. 191 of head 2
    v[231, 1, 7], k[240, 1, 9] = np.inf, np.nan                # the open block, 224 ..
    ref = R.Cache(nkv, cap)
    ref.write(k, v, 0)
    kv, sc = Dev(ref.buffer(0xFF)), Dev(np.array([SCALE]))
    q = g.standard_normal((ntok, nq, HD)).astype(F32)
    q[50, 0, 1], q[50, 1, 1], q[51, 60, 127] = np.nan, np.inf, -np.inf
    ctx = Dev(np.full((ntok + 1, nq, HD), 7, F32))
    hv.attn_rows_q8(Dev(q), kv, ctx, sc, pos0, nq, HD, group, cap, ntok,
                    scratch(hv, nq, group, cap, ntok))
    got = ctx.get(F32, (ntok + 1, nq, HD))
    assert (got[ntok] == 7).all()
    assert np.isnan(got[n - pos0:ntok]).all()
    assert np.isnan(got[50, :2]).all() and np.isnan(got[51, 60]).all()
    for t in (0, 49, 50, 51, 119, 120, 183, 190, 191, 199, 200, 209):
        pos = pos0 + t
        head = np.arange(nq) // group
        lost = (head == 2) & (pos >= 160)
        part = (head == 1) & (pos >= 231)
        bad = lost | part
        if t == 50:
            bad |= np.arange(nq) < 2
        if t == 51:
            bad |= np.arange(nq) == 60
        assert np.isnan(got[t][lost]).all()
        assert not np.isfinite(got[t][part][:, 7]).any()
        if pos >= 240:
            assert np.isnan(got[t][head == 1]).all()
        clean = np.nan_to_num(q[t], posinf=0, neginf=0)
        want, tol = R.attention(clean, np.nan_to_num(ref.val, posinf=0), pos, group,
                                float(SCALE))
        near(got[t][~bad], want[~bad], tol[~bad])


@pytest.mark.parametrize("size", [1e-20, 1.0, 1e4, 1e18])
def test_long_run_sizes_of_q_and_k(hv, size):
    nkv, group, pos0, ntok, cap = 8, 8, 30, 220, 256
    nq, n = nkv * group, pos0 + ntok
    g = np.random.default_rng(22)
    k, v = rows(g, n, nkv, 0.3)
    ref = R.Cache(nkv, cap)
    ref.write((k / F32(size)).astype(F32), (v * F32(size)).astype(F32), 0)
    q = (g.standard_normal((ntok, nq, HD)) * size).astype(F32)
    q[-1, 0], q[-1, 1] = 0, ref.val[0, 0, 100] * F32(30) * F32(size) * F32(size)
    ctx = Dev(np.zeros((ntok, nq, HD), F32))
    hv.attn_rows_q8(Dev(q), Dev(ref.buffer(0xFF)), ctx, Dev(np.array([SCALE])), pos0, nq, HD,
                    group, cap, ntok, scratch(hv, nq, group, cap, ntok))
    got = ctx.get(F32, (ntok, nq, HD))
    for t in (0, 100, ntok - 1):
        near(got[t], *R.attention(q[t], ref.val, pos0 + t, group, float(SCALE)))


@pytest.mark.parametrize("scale", [0.0, -0.07, 1e-30, 3.0])
def test_scales_of_any_sign(hv, scale):
    """Zero makes all weights equal; below it the smallest products weigh most."""
    for nkv, group, pos0, ntok in ((2, 4, 70, 1), (2, 4, 70, 5), (8, 8, 30, 220), (1, 1, 500, 40)):
        nq, n = nkv * group, pos0 + ntok
        g, ref, kv = filled(hv, 41, nkv, n, n + 9)
        q = (0.3 * g.standard_normal((ntok, nq, HD))).astype(F32)
        sc, ctx = Dev(np.array([scale], F32)), Dev(np.zeros((ntok, nq, HD), F32))
        s = scratch(hv, nq, group, n + 9, ntok)
        hv.attn_rows_q8(Dev(q), kv, ctx, sc, pos0, nq, HD, group, n + 9, ntok, s)
        got = ctx.get(F32, (ntok, nq, HD))
        for t in {0, ntok // 2, ntok - 1}:
            near(got[t], *R.attention(q[t], ref.val, pos0 + t, group, float(F32(scale))))
        hv.attn_decode_q8(Dev(q[-1:]), kv, ctx, sc, i32(n - 1), nq, HD, group, n + 9, s)
        near(ctx.get(F32, (ntok, nq, HD))[0],
             *R.attention(q[-1], ref.val, n - 1, group, float(F32(scale))))


@pytest.mark.parametrize("ntok", [1, 4, 40])
@pytest.mark.parametrize("first", [600, 1056])
@pytest.mark.parametrize("small", [1e-31, 1e-20, 1e20, 1e30])
def test_values_of_very_different_sizes(hv, ntok, small, first):
    """The first blocks' V (or all of it) apart from the usual by many orders: their weights
    count all the same, in whole chunks of them too."""
    nkv, group, pos0, cap = 8, 8, 1000, 1056
    nq, n = nkv * group, pos0 + ntok
    g = np.random.default_rng(43)
    k, v = rows(g, n, nkv, 0.3)
    v[:first] *= F32(small)
    ref = R.Cache(nkv, cap)
    ref.write(k, v, 0)
    q = queries(g, ref, ntok, nq)
    ctx = Dev(np.zeros((ntok, nq, HD), F32))
    hv.attn_rows_q8(Dev(q), Dev(ref.buffer(0xFF)), ctx, Dev(np.array([SCALE])), pos0, nq, HD,
                    group, cap, ntok, scratch(hv, nq, group, cap, ntok))
    got = ctx.get(F32, (ntok, nq, HD))
    for t in {0, ntok - 1}:
        near(got[t], *R.attention(q[t], ref.val, pos0 + t, group, float(SCALE)))


def test_offsets_past_32_bits(hv):
    """4.3 GB of codes: the last head's last blocks. What was there before is zeros (K and V
    values of 0, so weights of exp(0))."""
    nkv, cap, new = 32, (1 << 19) + 96, 80
    n0 = cap - new - 7
    (_, _, at, end), _ = R.parts(nkv, cap)
    kv = Dev(nbytes=end)
    nblk = -(-cap // R.BLK)
    hv.memset8(int(kv), 0x80, nkv * nblk * 2 * 4096)           # codes of 0, scales of 1
    one = np.ones(nkv * nblk * 2, F32)
    hv.upload(int(kv) + nkv * nblk * 2 * 4096, one.ctypes.data, one.nbytes)
    held = np.full(nkv * 2, n0 // 32 * 32, np.int32)           # whole blocks
    hv.upload(int(kv) + at, held.ctypes.data, held.nbytes)
    n0 = int(held[0])
    g = np.random.default_rng(42)
    k, v = rows(g, new, nkv, 0.1)
    hv.kv_rows_q8(Dev(k), Dev(v), nkv * HD, kv, n0, nkv, HD, cap, new)
    ref = R.Cache(nkv, 128)
    ref.write(k, v, 0)
    got = read(hv, kv, nkv, cap, n0, new)
    assert same(got, ref.val[:, :, :new])
    assert (read(hv, kv, nkv, cap, n0 - 40, 40) == 0).all()
    val = ref.val[:, :, :new].astype(np.float64)
    for ntok in (1, 2, 70):                                    # each attention kernel
        q = (4 * g.standard_normal((ntok, nkv, HD)) * SCALE + k[-1] / 4).astype(F32)
        ctx = Dev(np.zeros((ntok, nkv, HD), F32))
        s = scratch(hv, nkv, 1, cap, ntok)
        pos0 = n0 + new - ntok
        hv.attn_rows_q8(Dev(q), kv, ctx, Dev(np.array([SCALE])), pos0, nkv, HD, 1, cap, ntok, s)
        got = ctx.get(F32, (ntok, nkv, HD))
        for h in (0, 17, nkv - 1):
            seen = new
            x = (val[0, h, :seen] @ q[-1, h].astype(np.float64)) * float(SCALE)
            w = np.exp(x - max(x.max(), 0))
            total = w.sum() + n0 * np.exp(-max(x.max(), 0))
            want, size = w @ val[1, h] / total, w @ np.abs(val[1, h]) / total
            big = (np.abs(val[0, h]) @ np.abs(q[-1, h])).max() * float(SCALE)
            peak = np.abs(val[1, h]).max()
            n = n0 + new
            # the bound of kv_q8_ref.attention; the sum of the weights adds its n terms apart
            # from the values, whose sum has `new` of them that are not zero
            tol = (96 * R.U * 2 * big + (n / 8 + 64) * R.U) * size
            tol += 2.0 ** -32 * n * (w / total).max() * peak
            near(got[-1, h], want, tol)


def test_scratch_does_for_every_shorter_run(hv):
    for nq, group, cap in ((8, 1, 500), (40, 5, 20000), (32, 4, 4096), (64, 8, 40960),
                           (148, 1, 8192), (16, 2, 257), (6, 3, 1 << 20)):
        sizes = [hv.attn_q8_scratch(nq, group, cap, n) for n in range(1, 300)]
        assert sizes == sorted(sizes)
    # one for the longest: short runs of many chunks, long ones of one, single tokens
    nkv, group, n = 8, 5, 3000
    nq = nkv * group
    g, ref, kv = filled(hv, 23, nkv, n, n)
    q, sc = queries(g, ref, 256, nq), Dev(np.array([SCALE]))
    need = hv.attn_q8_scratch(nq, group, n, 256)
    room = np.full(need + 4096, 0x5A, np.uint8)
    room[:need] = 0
    s = Dev(room)
    for ntok in (256, 3, 21, 1, 64, 13, 256, 7):
        ctx = Dev(np.zeros((ntok, nq, HD), F32))
        if ntok == 1:
            hv.attn_decode_q8(Dev(q[:1]), kv, ctx, sc, i32(n - 1), nq, HD, group, n, s)
        else:
            hv.attn_rows_q8(Dev(q[:ntok]), kv, ctx, sc, n - ntok, nq, HD, group, n, ntok, s)
        got = ctx.get(F32, (ntok, nq, HD))
        for t in {0, ntok - 1}:
            near(got[t], *R.attention(q[t], ref.val, n - ntok + t, group, float(SCALE)))
        assert (s.get(np.uint8)[need:] == 0x5A).all(), ntok


def test_captured_run_equals_the_direct_one(hv):
    """A write of a run and its attention captured, on a stream that is not the default one."""
    nkv, group, cap, pos0, ntok = 4, 4, 1000, 700, 200
    nq = nkv * group
    g = np.random.default_rng(24)
    k, v = rows(g, pos0 + ntok, nkv, 0.3)
    q, sc = Dev(g.standard_normal((ntok, nq, HD)).astype(F32)), Dev(np.array([SCALE]))
    out = []
    for graph in (False, True):
        kv, s = new_cache(hv, nkv, cap), scratch(hv, nq, group, cap, ntok)
        write(hv, kv, k[:pos0], v[:pos0], 0, cap)
        dk, dv, ctx = Dev(k[pos0:]), Dev(v[pos0:]), Dev(np.zeros((ntok, nq, HD), F32))
        hv.synchronize()
        st = hv.stream_create()
        if graph:
            hv.capture_begin(st)
        hv.kv_rows_q8(dk, dv, nkv * HD, kv, pos0, nkv, HD, cap, ntok, st)
        hv.attn_rows_q8(q, kv, ctx, sc, pos0, nq, HD, group, cap, ntok, s, st)
        if graph:
            gr = hv.capture_end(st)
            ex = hv.graph_instantiate(gr)
            for _ in range(3):                                 # the same run again: a rewind
                hv.graph_launch(ex, st)
        hv.stream_synchronize(st)
        out.append(bits(ctx.get(F32)))
        if graph:
            hv.graph_destroy(gr, ex)
        hv.stream_destroy(st)
    assert np.array_equal(*out)


# ---- the engine ----------------------------------------------------------------------

def engine(arch, seed, cap, **kw):
    import limited
    cfg = w4format.Config(arch)
    return limited.Engine(config=cfg, tensors=synth.iter_tensors(cfg, seed), quiet=True,
                          max_context=cap, **kw)


@pytest.mark.parametrize("prefill", ["steps", "batched"])
def test_engine_over_the_8bit_cache(hv, prefill):
    """The first layer's cache is the f32 engine's rows quantised (they do not depend on
    attention); the last layer's context is attention over what its cache reads back; the
    graph-replayed decode gives the direct one's tokens."""
    arch = synth.tiny_arch(hidden=512, n_head=8, n_kv=2)
    ids = synth.prompt_ids(w4format.Config(arch), 3, 300)
    cap = 352
    a = engine(arch, 3, cap, kv_dtype="q8", fused=False, prefill=prefill)
    f = engine(arch, 3, cap, fused=False, prefill=prefill)
    try:
        c = a.cfg
        assert a.kv_bytes == c.n_layer * hv.kv_q8_size(c.n_kv, HD, cap)
        lf, la = f.logits(ids), a.logits(ids)
        assert np.isfinite(la).all() and la.shape == lf.shape
        n = len(ids)
        k32, v32 = (f._download(p, (c.n_kv, cap, HD), F32)[:, :n].swapaxes(0, 1)
                    for p in (f.KC[0], f.VC[0]))
        ref = R.Cache(c.n_kv, cap)
        ref.write(k32, v32, 0)
        assert same(read(hv, a.KC[0], c.n_kv, cap, 0, n), ref.val[:, :, :n])
        if prefill == "steps":
            q = a._download(a.d_qkv, (c.n_head, HD), F32)
            ctx = a._download(a.d_ctx, (c.n_head, HD), F32)
        else:
            m = (n - 1) % a.PREFILL_BATCH
            at = m * c.n_head * HD * 4
            q = a._download(a._pf["q"] + at, (c.n_head, HD), F32)
            ctx = a._download(a._pf["ctx"] + at, (c.n_head, HD), F32)
        val = read(hv, a.KC[-1], c.n_kv, cap, 0, n)
        near(ctx, *R.attention(q, val, n - 1, c.group, float(a.attn_scale)))
        toks, _, _ = a.generate(ids, 40, stop_on_eos=False)
        assert a.generate(ids, 40, stop_on_eos=False, use_graph=True)[0] == toks
        assert a.generate(ids, 40)[0] == toks                  # a shorter cache written over
        for fused_only in (a.profile_step, lambda: a._step_fused(0)):
            with pytest.raises(ValueError):
                fused_only()
        assert a.step_status() == 0
    finally:
        a.free()
        f.free()


def test_engine_q8_with_odd_group_and_long_context(hv):
    """A group of 5 query heads and a capacity over the reference-order attention's 16384."""
    arch = synth.tiny_arch(hidden=256, n_head=10, n_kv=2)
    a = engine(arch, 4, 20000, kv_dtype="q8", fused=False, prefill="batched")
    try:
        ids = synth.prompt_ids(a.cfg, 4, 600)
        toks, _, _ = a.generate(ids, 8, stop_on_eos=False)
        assert len(toks) == 8
    finally:
        a.free()
