"""Shared prefixes, weights added up and eviction without a GPU: what their entry points refuse
(checked on the host before anything is launched)."""
import numpy as np
import pytest

import hvdrv
import span_ref as R

P = 1 << 20                          # a pointer that no refused call may follow
INVALID, UNSUPPORTED = 1001, 1002


def refused(code, fn, *a, **kw):
    with pytest.raises(hvdrv.CudaError) as e:
        fn(*a, **kw)
    assert e.value.code == code, str(e.value)


def shared(q=P, pk=P, pv=P, pcap=64, plen=P, tk=P, tv=P, tcap=8, row0=P, tlen=P, ctx=P, scale=P, nq=8,
           hd=128, group=4, nseq=2, nrow=3, s=P):
    hvdrv.attn_shared(q, pk, pv, pcap, plen, tk, tv, tcap, row0, tlen, ctx, scale, nq, hd, group,
                      nseq, nrow, s)


def test_shared_attention_refusals():
    for kw in (dict(q=0), dict(pk=0), dict(pv=0), dict(plen=0), dict(tk=0), dict(tv=0), dict(tlen=0),
               dict(ctx=0), dict(scale=0), dict(s=0), dict(pcap=-1), dict(tcap=0), dict(nq=0),
               dict(group=0), dict(group=3), dict(nseq=0), dict(nrow=0), dict(row0=0),
               dict(q=P + 4), dict(pk=P + 8), dict(pv=P + 8), dict(tk=P + 8), dict(tv=P + 2),
               dict(ctx=P + 4), dict(s=P + 8)):
        refused(INVALID, shared, **kw)
    for kw in (dict(hd=64), dict(nq=18, group=9), dict(nrow=65536), dict(nseq=65536),
               dict(pcap=(1 << 24) + 1), dict(tcap=(1 << 24) + 1)):
        refused(UNSUPPORTED, shared, **kw)


def test_write_of_a_batch_refusals():
    def qk(qkv=P, qn=P, kn=P, cos=P, sin=P, cap=64, base=P, row0=P, tlen=P, q=P, tk=P, tv=P, nq=8, nkv=2,
           hd=128, tcap=8, nseq=2, nrow=3):
        hvdrv.qk_shared(qkv, qn, kn, cos, sin, cap, base, row0, tlen, q, tk, tv, nq, nkv, hd, tcap,
                        1e-5, nseq, nrow)
    for kw in (dict(qkv=0), dict(qn=0), dict(kn=0), dict(cos=0), dict(sin=0), dict(cap=0), dict(base=0),
               dict(tlen=0), dict(q=0), dict(tk=0), dict(tv=0), dict(nq=0), dict(nkv=0), dict(tcap=0),
               dict(nseq=0), dict(nrow=0), dict(row0=0), dict(qkv=P + 4), dict(q=P + 8),
               dict(tk=P + 8), dict(tv=P + 8)):
        refused(INVALID, qk, **kw)
    for kw in (dict(hd=64), dict(nrow=65536), dict(tcap=(1 << 24) + 1)):
        refused(UNSUPPORTED, qk, **kw)


def test_mass_refusals():
    def dec(q=P, k=P, v=P, ctx=P, mi=0, mo=P, scale=P, pos=P, nq=8, hd=128, group=4, cap=64, s=P):
        hvdrv.attn_decode_mass(q, k, v, ctx, mi, mo, scale, pos, nq, hd, group, cap, s)

    def rows(q=P, k=P, v=P, ctx=P, mi=0, mo=P, scale=P, pos0=0, nq=8, hd=128, group=4, cap=64, ntok=4,
             s=P):
        hvdrv.attn_rows_mass(q, k, v, ctx, mi, mo, scale, pos0, nq, hd, group, cap, ntok, s)
    for fn in (dec, rows):
        for kw in (dict(q=0), dict(k=0), dict(v=0), dict(ctx=0), dict(mo=0), dict(scale=0), dict(s=0),
                   dict(nq=0), dict(group=0), dict(group=3), dict(cap=0), dict(q=P + 4),
                   dict(k=P + 8), dict(v=P + 8), dict(ctx=P + 8), dict(s=P + 4)):
            refused(INVALID, fn, **kw)
        for kw in (dict(hd=64), dict(nq=18, group=9), dict(cap=(1 << 24) + 1)):
            refused(UNSUPPORTED, fn, **kw)
    refused(INVALID, dec, pos=0)
    for kw in (dict(pos0=-1), dict(ntok=0), dict(pos0=61), dict(pos0=0x7FFFFFFF)):
        refused(INVALID, rows, **kw)


def evict(kc=P, vc=P << 4, set_=1 << 16, mass=P << 8, cap=64, len_=P, added=0, kd=None, vd=None, set_d=1 << 16,
          md=None, dcap=64, lo=P, kept=0, limit=60, keep=40, recent=8, nkv=2, hd=128, nset=2, s=P):
    kd, vd, md = (kc if kd is None else kd, vc if vd is None else vd, mass if md is None else md)
    hvdrv.kv_evict(kc, vc, set_, mass, cap, len_, added, kd, vd, set_d, md, dcap, lo, kept, limit,
                   keep, recent, nkv, hd, nset, s)


def test_eviction_refusals():
    for kw in (dict(kc=0), dict(vc=0), dict(mass=0), dict(len_=0), dict(kd=0), dict(vd=0), dict(md=0),
               dict(lo=0), dict(s=0), dict(cap=0), dict(dcap=0), dict(added=-1), dict(nkv=0),
               dict(nset=0), dict(keep=0), dict(recent=-1), dict(recent=41), dict(keep=61),
               dict(limit=65), dict(set_=2 * 64 * 128 - 8), dict(set_d=2 * 64 * 128 - 8),
               dict(set_=(1 << 16) + 4), dict(kc=P + 8), dict(vd=P + 8), dict(s=P + 8),
               # in place, but not as the source is arranged
               dict(md=P << 9), dict(dcap=63, limit=63), dict(set_d=1 << 17),
               # neither in place nor apart
               dict(kd=P + 256), dict(vd=(P << 4) + 256), dict(kd=P << 5, vd=P << 5, md=P << 9),
               dict(kd=P << 5, vd=P << 6, md=(P << 8) + 16)):
        refused(INVALID, evict, **kw)
    for kw in (dict(hd=64), dict(cap=(1 << 24) + 1, set_=1 << 36, set_d=1 << 36),
               dict(nkv=65536, set_=1 << 34, set_d=1 << 34)):
        refused(UNSUPPORTED, evict, **kw)


def test_scratch_sizes_refuse_what_their_calls_refuse():
    for a in ((0, 4, 64, 8, 1, 1), (8, 3, 64, 8, 1, 1), (8, 4, -1, 8, 1, 1), (8, 4, 64, 0, 1, 1),
              (8, 4, 64, 8, 0, 1), (8, 4, 64, 8, 1, 0)):
        refused(INVALID, hvdrv.attn_shared_scratch, *a)
    for a in ((18, 9, 64, 8, 1, 1), (8, 4, 64, 8, 1, 65536), (8, 4, (1 << 24) + 1, 8, 1, 1)):
        refused(UNSUPPORTED, hvdrv.attn_shared_scratch, *a)
    for a in ((8, 3, 64, 1), (8, 4, 0, 1), (8, 4, 64, 0)):
        refused(INVALID, hvdrv.attn_mass_scratch, *a)
    for a in ((18, 9, 64, 1), (8, 4, (1 << 24) + 1, 1), (8, 4, 64, 65536)):
        refused(UNSUPPORTED, hvdrv.attn_mass_scratch, *a)
    refused(INVALID, hvdrv.kv_evict_scratch, 0, 64, 1)
    refused(UNSUPPORTED, hvdrv.kv_evict_scratch, 2, (1 << 24) + 1, 1)


@pytest.mark.parametrize("fn,small,large", [
    (hvdrv.attn_shared_scratch, (8, 4, 100, 8, 1, 1), (8, 4, 33000, 600, 64, 256)),
    (hvdrv.attn_mass_scratch, (8, 4, 100, 1), (8, 4, 33000, 256)),
    (hvdrv.kv_evict_scratch, (2, 100, 1), (2, 33000, 36))])
def test_scratch_sizes_cover_every_smaller_call(fn, small, large):
    g = np.random.default_rng(0)
    most = fn(*large)
    for _ in range(300):
        fixed = 2 if fn is not hvdrv.kv_evict_scratch else 0
        a = [x if i < fixed else int(g.integers(1, x + 1)) for i, x in enumerate(large)]
        assert 0 < fn(*a) <= most, a
    assert fn(*small) <= most


def test_plain_eviction():
    m = np.array([0, 3, np.nan, 3, 1, np.inf, 0, 9], np.float32)
    assert R.evict(m, 8, 8, 3, 1).tolist() == list(range(8))
    assert R.evict(m, 8, 7, 4, 1).tolist() == [1, 2, 5, 7]
    assert R.evict(m, 8, 7, 5, 2).tolist() == [1, 2, 5, 6, 7]
    assert R.evict(m, 7, 5, 3, 3).tolist() == [4, 5, 6]


# ---- the engine's arguments -----------------------------------------------------------------

def test_engine_refusals():
    import limited
    import synth
    make = lambda **kw: limited.Engine(config=synth.tiny_arch(), tensors={}, **kw)  # noqa: E731
    for kw in (dict(kv_keep=64), dict(kv_keep=64, kv_dtype="f16"), dict(kv_keep=64, fused=False),
               dict(kv_keep=64, kv_dtype="q8", fused=False),
               dict(kv_keep=0, kv_dtype="f16", fused=False),
               dict(kv_keep=64, kv_recent=65, kv_dtype="f16", fused=False),
               dict(kv_keep=64, kv_recent=-1, kv_dtype="f16", fused=False),
               dict(kv_recent=8, kv_dtype="f16", fused=False)):
        with pytest.raises(ValueError, match="kv_keep"):
            make(**kw)


def test_many_refusals():
    """Checked before any device work: an engine without a device will do."""
    import limited
    import synth
    import w4format
    e = object.__new__(limited.Engine)
    e.cfg, e.world, e.kv_f16 = w4format.Config(synth.tiny_arch()), 1, True
    e.cfg.max_context = 64
    v = e.cfg.vocab
    for prompt, branches in (([], [[1]]), ([1], []), ([1, v], [[1]]), ([1], [[-1]]), ([1.5], [[1]]),
                             ([1], [[1]] * 257), ([1] * 60, [[1] * 5]), ([[1]], [[1]])):
        with pytest.raises(ValueError):
            e.score_many(prompt, branches)
        with pytest.raises(ValueError):
            e.generate_many(prompt, branches, 1)
    with pytest.raises(ValueError, match="without a token"):
        e.score_many([1, 2], [[3], []])
    with pytest.raises(ValueError):
        e.generate_many([1] * 30, [[1] * 5, []], 30)
    with pytest.raises(ValueError):
        e.generate_many([1], [[1]], -1)
    assert e.generate_many([1], [[1], []], 0) == [[], []]
    for kw in (dict(kv_f16=False), dict(world=2)):
        for k, x in kw.items():
            setattr(e, k, x)
        with pytest.raises(ValueError, match="f16"):
            e.score_many([1], [[1]])
        e.kv_f16 = True


def rows_seen(texts, most):
    """What Engine._many_prompts runs, on a stand-in for the device part."""
    import limited
    e = object.__new__(limited.Engine)
    e.PREFILL_BATCH = most
    log, parts = [], []
    e._many_run = lambda mb, rows, tlen, toks: log.append((list(rows), list(tlen), toks.tolist()))
    e._many_prompts({}, [np.array(t, np.int32) for t in texts], parts.append)
    return log, parts


@pytest.mark.parametrize("sizes,most", [([1], 4), ([3, 1, 4, 2], 4), ([9, 1], 4), ([4, 4], 4),
                                        ([1] * 9, 4), ([13], 5), ([2, 300, 7], 256)])
def test_ragged_prompts_go_through_in_order(sizes, most):
    texts = [[100 * s + i for i in range(n)] for s, n in enumerate(sizes)]
    log, parts = rows_seen(texts, most)
    got = [[] for _ in texts]
    for (rows, tlen, toks), part in zip(log, parts):
        assert sum(rows) == len(toks) <= most
        at = 0
        for s, n in enumerate(rows):                       # rows stand sequence after sequence
            got[s] += toks[at:at + n]
            at += n
            assert tlen[s] == len(got[s])
        assert [(s, tlen[s] - rows[s], rows[s]) for s in range(len(texts)) if rows[s]] == [
            p[:3] for p in part]
        for s, lo, n, row in part:
            assert toks[row:row + n] == texts[s][lo:lo + n]
    assert got == texts
    assert len(log) == -(-sum(sizes) // most)
