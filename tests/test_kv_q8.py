"""The 8-bit KV cache without a GPU: its numpy model, its size, and what its entry points
refuse (checked on the host before anything is launched)."""
import numpy as np
import pytest

import hvdrv
import kv_q8_ref as R

F32 = np.float32
P = 1 << 20                          # a pointer that no refused call may follow


def test_codes_are_within_half_a_step():
    g = np.random.default_rng(0)
    for scale in (1e-30, 1.0, 3e37):
        x = (g.standard_normal((32, 128)) * scale).astype(F32)
        c, s = R.quantise(x)
        # f32(x / s) is off by at most u |x / s| <= 127 u, f32(c s) by u |x|
        err = np.abs(R.values(c, s).astype(np.float64) - x.astype(np.float64))
        assert np.abs(c).max() == 127
        assert err.max() <= float(s) * (0.5 + 3 * 127 * R.U)
    c, s = R.quantise(np.zeros((32, 128), F32))
    assert s == 1 and not c.any()


def test_arrangement_is_a_permutation():
    for at in R.positions():
        assert np.array_equal(np.sort(at.ravel()), np.arange(4096))


def test_the_models_cache_does_not_depend_on_the_calls():
    g = np.random.default_rng(1)
    k, v = g.standard_normal((2, 100, 2, 128)).astype(F32)
    a, b = R.Cache(2, 128), R.Cache(2, 128)
    a.write(k, v, 0)
    for lo, hi in ((0, 1), (1, 31), (31, 33), (33, 96), (96, 100)):
        b.write(k[lo:hi], v[lo:hi], lo)
    assert np.array_equal(a.buffer(), b.buffer())


@pytest.mark.parametrize("nkv,cap", [(1, 1), (2, 32), (8, 4352), (3, 33), (8, 131072)])
def test_size(nkv, cap):
    assert hvdrv.kv_q8_size(nkv, 128, cap) == R.parts(nkv, cap)[0][3]


def refused(code, fn, *a):
    with pytest.raises(hvdrv.CudaError) as e:
        fn(*a)
    assert e.value.code == code, str(e.value)


INVALID, UNSUPPORTED = 1001, 1002


def test_write_and_read_refusals():
    refused(INVALID, hvdrv.kv_q8_size, 0, 128, 64)
    refused(INVALID, hvdrv.kv_q8_size, 2, 128, 0)
    refused(UNSUPPORTED, hvdrv.kv_q8_size, 2, 64, 64)
    app = lambda k=P, v=P, kv=P, pos=P, nkv=2, hd=128, cap=64: hvdrv.kv_append_q8(  # noqa: E731
        k, v, kv, pos, nkv, hd, cap)
    for kw in (dict(k=0), dict(v=0), dict(kv=0), dict(pos=0), dict(nkv=0), dict(cap=0),
               dict(k=P + 4), dict(v=P + 8), dict(kv=P + 8)):
        refused(INVALID, lambda: app(**kw))
    refused(UNSUPPORTED, lambda: app(hd=64))
    rows = lambda k=P, v=P, ld=256, kv=P, pos0=0, nkv=2, hd=128, cap=64, ntok=4: (  # noqa: E731
        hvdrv.kv_rows_q8(k, v, ld, kv, pos0, nkv, hd, cap, ntok))
    for kw in (dict(k=0), dict(v=0), dict(kv=0), dict(ntok=0), dict(pos0=-1), dict(ld=252),
               dict(ld=258), dict(pos0=61), dict(ntok=65), dict(pos0=0x7FFFFFFF),
               dict(k=P + 4)):
        refused(INVALID, lambda: rows(**kw))
    refused(UNSUPPORTED, lambda: rows(hd=256))
    refused(UNSUPPORTED, lambda: rows(cap=1 << 30, ntok=(1 << 21) + 64))
    read = lambda kv=P, ko=P, vo=P, pos0=0, cap=64, ntok=4: hvdrv.kv_read_q8(  # noqa: E731
        kv, ko, vo, pos0, 2, 128, cap, ntok)
    for kw in (dict(kv=0), dict(ko=0), dict(vo=0), dict(ntok=0), dict(pos0=-1), dict(pos0=61),
               dict(ko=P + 4)):
        refused(INVALID, lambda: read(**kw))
    qk = lambda qkv=P, nq=4, pos0=0, ntok=4, cap=64, q=P: hvdrv.qk_rows_q8(  # noqa: E731
        qkv, P, P, P, P, pos0, q, P, nq, 2, 128, cap, 1e-5, ntok)
    for kw in (dict(qkv=0), dict(nq=0), dict(pos0=-1), dict(ntok=0), dict(pos0=61),
               dict(q=0), dict(qkv=P + 4)):
        refused(INVALID, lambda: qk(**kw))


def test_attention_refusals():
    dec = lambda q=P, kv=P, ctx=P, scale=P, pos=P, nq=8, hd=128, group=4, cap=64, s=P: (  # noqa: E731
        hvdrv.attn_decode_q8(q, kv, ctx, scale, pos, nq, hd, group, cap, s))
    for kw in (dict(q=0), dict(kv=0), dict(ctx=0), dict(scale=0), dict(pos=0), dict(s=0),
               dict(nq=0), dict(group=0), dict(group=3), dict(cap=0), dict(q=P + 4),
               dict(ctx=P + 4), dict(s=P + 4)):
        refused(INVALID, lambda: dec(**kw))
    refused(UNSUPPORTED, lambda: dec(hd=64))
    refused(UNSUPPORTED, lambda: dec(nq=18, group=9))
    rows = lambda q=P, kv=P, pos0=0, ntok=4, cap=64, group=4: hvdrv.attn_rows_q8(  # noqa: E731
        q, kv, P, P, pos0, 8, 128, group, cap, ntok, P)
    for kw in (dict(q=0), dict(kv=0), dict(pos0=-1), dict(ntok=0), dict(pos0=61), dict(group=5)):
        refused(INVALID, lambda: rows(**kw))
    refused(INVALID, hvdrv.attn_q8_scratch, 8, 3, 64, 1)
    refused(INVALID, hvdrv.attn_q8_scratch, 8, 4, 64, 0)
    refused(UNSUPPORTED, hvdrv.attn_q8_scratch, 18, 9, 64, 1)


def test_scoring_refusals():
    lp = lambda x=P, ld=100, rows=2, n=100, tok=P, top=5, o=P, ids=P, s=P: (  # noqa: E731
        hvdrv.logprob_rows(x, ld, rows, n, tok, top, o, P, ids, P, s))
    for kw in (dict(x=0), dict(ld=99), dict(rows=0), dict(n=0), dict(tok=0), dict(top=-1),
               dict(o=0), dict(ids=0), dict(s=0), dict(n=4, ld=4)):
        refused(INVALID, lambda: lp(**kw))
    refused(UNSUPPORTED, lambda: lp(top=33))
    refused(INVALID, hvdrv.logprob_scratch, 0, 10, 0)
    refused(UNSUPPORTED, hvdrv.logprob_scratch, 1, 100, 33)


def test_engine_refuses_the_fused_step_over_q8():
    import limited
    import synth
    with pytest.raises(ValueError, match="fused=False"):
        limited.Engine(config=synth.tiny_arch(), tensors={}, kv_dtype="q8")
    with pytest.raises(ValueError, match="kv_dtype"):
        limited.Engine(config=synth.tiny_arch(), tensors={}, kv_dtype="q4")


def test_scratch_sizes_refuse_what_their_calls_refuse():
    for a in ((32769, 1, 64, 1), (8, 4, (1 << 30) + 1, 1), (8, 4, 0x7FFFFFFF, 4), (8, 4, 64, 65536)):
        refused(UNSUPPORTED, hvdrv.attn_q8_scratch, *a)
    refused(UNSUPPORTED, hvdrv.logprob_scratch, 1, (1 << 30) + 1, 0)
