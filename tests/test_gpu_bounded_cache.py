"""A bounded cache that a prompt fills exactly, or nearly, on a B200: decode steps find room, write
their own row and no other, and their logits are finite."""
import numpy as np
import pytest

from gpu_util import Dev

pytestmark = pytest.mark.gpu
F32, F16, HD = np.float32, np.float16, 128


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("pos", [-3, -1, 0, 7, 8, 9, 2 ** 31 - 1, -2 ** 31])
def test_append_outside_the_cache_writes_nothing(hv, dtype, pos):
    nkv, cap, margin = 3, 8, 16
    g = np.random.default_rng(1)
    k, v = g.standard_normal((2, nkv, HD)).astype(F32)
    whole = g.standard_normal((2, margin + nkv * cap + margin, HD)).astype(dtype)
    dev = [Dev(x) for x in whole]
    at = margin * HD * whole.itemsize
    hv.kv_append(Dev(k), Dev(v), int(dev[0]) + at, int(dev[1]) + at, Dev(np.array([pos], np.int32)), nkv, HD,
                 cap, f16=dtype == F16)
    for d, want, x in zip(dev, whole, (k, v)):
        if 0 <= pos < cap:
            want[margin:-margin].reshape(nkv, cap, HD)[:, pos] = x.astype(dtype)
        assert np.array_equal(d.get(dtype, want.shape).view(np.uint8), want.view(np.uint8))


def caches(e):
    c = e.cfg
    return np.stack([e._download(p, (c.n_kv, e.kv_cap, HD), F16) for l in range(c.n_layer)
                     for p in (e.KC[l], e.VC[l])]).view(np.uint16)


def test_decode_after_prompts_that_fill_the_bounded_cache(hv):
    import limited
    import synth
    import w4format
    cfg = w4format.Config(synth.tiny_arch(hidden=512, n_head=8, n_kv=2))
    keep = 96
    e = limited.Engine(config=cfg, tensors=synth.iter_tensors(cfg, 7), quiet=True, max_context=1100,
                       kv_dtype="f16", fused=False, prefill="batched", kv_keep=keep)
    try:
        cap = e.kv_cap
        assert cap == keep + 256
        ids = synth.prompt_ids(cfg, 7, 1030)
        for n in (cap - 1, cap, cap + 1, 256, 512, 768, 1024, 1025):
            e._prefill(ids[:n])
            held = e._get_i32(e.d_held)
            assert held == e._held < cap, n
            for _ in range(3):
                before = caches(e)
                e._decode_one()
                assert np.isfinite(e.download_logits()).all()
                now = e._get_i32(e.d_held)
                if now == held + 1:                          # else the cache was thinned
                    same = np.arange(cap) != held
                    assert np.array_equal(caches(e)[:, :, same], before[:, :, same])
                else:
                    assert held + 1 == cap and now == keep
                held = now
            direct, _, _ = e.generate(ids[:n], 20, stop_on_eos=False, use_graph=False)
            assert e.generate(ids[:n], 20, stop_on_eos=False, use_graph=True)[0] == direct
            assert e._get_i32(e.d_held) < cap
    finally:
        e.free()
