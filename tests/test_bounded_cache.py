"""The bounded cache's bookkeeping without a GPU: how many positions a layer holds after a prompt and
after every decode step, on a stand-in for the library that follows the length as the device does
and refuses rows outside the cache."""
import numpy as np
import pytest


class Device:
    """The calls that move the length or write rows; all others do nothing."""

    def __init__(self):
        self.held = 0

    def __getattr__(self, name):
        return lambda *a, **kw: 0

    def kv_evict(self, kc, vc, set_, mass, cap, len_, added, kd, vd, set_d, mass_d, dcap, len_out, kept,
                 limit, keep, recent, *rest):
        n = self.held + added
        assert 0 <= n <= cap and 0 < keep <= limit and 0 <= recent <= keep
        self.held = keep if n > limit else n

    def qk_rows(self, qkv, qn, kn, cos, sin, pos0, q, kc, vc, nq, nkv, hd, cap, eps, m, s, f16):
        assert f16 and pos0 == self.held and pos0 + m <= cap

    def attn_rows_mass(self, q, kc, vc, ctx, mi, mo, scale, pos0, nq, hd, group, cap, m, *rest):
        assert pos0 == self.held and pos0 + m <= cap

    def kv_append(self, k, v, kc, vc, pos, nkv, hd, cap, s, f16):
        assert f16 and 0 <= self.held < cap

    def attn_decode_mass(self, q, kc, vc, ctx, mi, mo, scale, pos, nq, hd, group, cap, *rest):
        assert 0 <= self.held < cap


def engine(monkeypatch, keep, max_context, run=8):
    import limited
    import synth
    import w4format
    dev = Device()
    monkeypatch.setattr(limited, "hvdrv", dev)
    e = object.__new__(limited.Engine)
    e.cfg = w4format.Config(synth.tiny_arch(n_layer=1))
    e.cfg.max_context = max_context
    e.PREFILL_BATCH = run
    e.kv_keep, e.kv_recent, e.kv_f16, e.fused = keep, keep // 4, True, False
    e.shard, e.layers = dict(n_kv=e.cfg.n_kv), [dict.fromkeys(("an", "qn", "kn", "fn", "qkv", "o", "gu", "down"), 0)]
    names = ("kv", "mass", "evict_scr", "mass_scr", "scale", "cos", "sin", "emb16",
             "tok", "pos", "step", "gen", "h", "hn", "qkv", "ctx", "o", "gu", "act", "onorm", "logits")
    for n in names:
        setattr(e, "d_" + n, 0)
    e.KC = e.VC = [0]
    e.head, e._stream_cur, e.prefill_mode = (0, 0, 0, 0, 0), 0, "batched"
    e._pf = dict.fromkeys(("tok", "h", "hn", "a8", "sa", "qkv", "q", "ctx", "o", "gu", "act", "part",
                           "ticket"), 0) | {"n": run}
    e._gemm = e._gemv = lambda *a: None

    e.d_held, e._held = 1, 0

    def set_i32(ptr, value):
        if ptr == e.d_held:
            dev.held = value
    e._set_i32 = set_i32
    return e, dev


@pytest.mark.parametrize("keep,max_context", [(1, 100), (5, 100), (8, 100), (20, 100), (5, 10), (60, 64)])
def test_a_decode_step_finds_room_after_every_prompt(monkeypatch, keep, max_context):
    e, dev = engine(monkeypatch, keep, max_context)
    cap = e.kv_cap
    for n in range(1, max_context):
        e._prefill_batched([1] * n, argmax=False)
        assert e._held == dev.held < cap, n
        for _ in range(min(max_context - n, 2 * cap)):
            e._step_eager()
            assert 0 < dev.held < cap


def test_a_prompt_of_the_whole_context(monkeypatch):
    for keep in (5, 90, 100, 200):
        e, dev = engine(monkeypatch, keep, 100)
        e._prefill_batched([1] * 100, argmax=False)
        assert 0 < dev.held == e._held <= e.kv_cap


# ---- K and V of an eviction's destination -------------------------------------------------

P = 1 << 30
ONE = 2 * 64 * 128                   # values of a cache of 2 heads, 64 positions


def evict(kd, vd, set_d, nset, in_place=False):
    import hvdrv
    kc, vc = (kd, vd) if in_place else (P << 8, P << 9)
    mass = P << 10
    hvdrv.kv_evict(kc, vc, set_d if in_place else ONE, mass, 64, P << 11, 0, kd, vd, set_d,
                   mass if in_place else P << 12, 64, P << 11, 0, 60, 40, 8, 2, 128, nset, P << 13)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("nset,set_d,off", [
    (1, 0, 0), (1, 0, ONE - 8), (1, 0, 8 - ONE),
    (2, ONE, ONE), (2, ONE, -ONE), (2, 2 * ONE, 2 * ONE), (2, 2 * ONE, 3 * ONE - 8),
    (3, 2 * ONE, ONE + 8), (3, 2 * ONE, ONE - 8), (3, 2 * ONE, 2 * ONE), (3, 2 * ONE, -4 * ONE), (3, 2 * ONE, 5 * ONE - 8),
    (36, 2 * ONE, 70 * ONE), (36, 2 * ONE, -70 * ONE), (36, 3 * ONE, 2 * ONE + 8), (36, 3 * ONE, ONE - 8),
    (4, 1 << 38, (1 << 38) + 64), (4, 1 << 38, -3 * (1 << 38))])
def test_eviction_refuses_v_on_k(in_place, nset, set_d, off):
    import hvdrv
    kd = P << 20
    with pytest.raises(hvdrv.CudaError, match="K and V of the destination") as e:
        evict(kd, kd + 2 * off, set_d, nset, in_place)
    assert e.value.code == 1001


# ---- the buffers of many continuations ------------------------------------------------------

def test_buffers_of_many_continuations_are_kept_but_laid_out_by_the_call(monkeypatch):
    e, dev = engine(monkeypatch, 5, 100)
    held, n = {}, [0]

    def alloc(nbytes):
        n[0] += 1
        held[n[0] << 12] = nbytes
        return n[0] << 12
    e._buffers, e._many = [], None
    dev.alloc, dev.free = alloc, held.pop
    dev.attn_shared_scratch = lambda nq, group, pcap, tcap, nseq, nrow: 8 * tcap * nseq + 100
    per = e.cfg.n_layer * 2 * e.cfg.n_kv * e.cfg.head_dim * 2
    most, calls = {}, [(2, 10), (40, 10), (3, 90), (2, 10), (40, 10), (1, 400), (2, 10)]
    for nseq, tcap in calls + calls:
        before = dict(held)
        mb = e._many_buffers(nseq, tcap)
        assert mb["tcap"] == tcap
        assert held[mb["tails"]] >= nseq * tcap * per and held[mb["scr"]] >= 8 * tcap * nseq + 100
        assert held[mb["hl"]] >= nseq * e.cfg.hidden * 4 and held[mb["tlen"]] >= 4 * nseq
        assert held[mb["row0"]] >= 4 * (nseq + 1)
        assert len(held) == len(e._buffers) == 7
        if (nseq, tcap) in most:
            assert held == before                            # a call of a size that was there allocates nothing
        most[nseq, tcap] = True

    def fails(nbytes):
        raise MemoryError
    dev.alloc = fails
    with pytest.raises(MemoryError):
        e._many_buffers(41, 500)
    dev.alloc = alloc
    mb = e._many_buffers(41, 500)                            # what could not be had is asked for again
    assert held[mb["tails"]] >= 41 * 500 * per and len(held) == len(e._buffers) == 7
