"""Scores far beyond what f32 tells apart: a position that no other comes near has all of the weight,
and equal ones share it, by every kernel that attention may go to."""
import numpy as np
import pytest

import span_ref as R
from test_gpu_shared import near, run_mass, run_shared, SCALE

pytestmark = pytest.mark.gpu
F32, F16, HD = np.float32, np.float16, 128


def keys(g, nkv, n, tops):
    """Keys in {-1, 0, 1} but at `tops`: twos, all of them along the queries below."""
    k = g.integers(-1, 2, (nkv, n, HD)).astype(F16)
    k[:, tops] = 2
    return k


@pytest.mark.parametrize("size", [1e4, 3e6, 3e7, 1e9, 1e12, 1e30])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("nkv,group,nseq,plen", [
    (2, 4, 3, 700), (8, 4, 40, 1500), (1, 8, 70, 5000), (2, 3, 200, 3001)])    # few rows, then tiles
def test_shared(hv, size, sign, nkv, group, nseq, plen):
    """Queries of one value: a key of twos has twice the score that any other can have. With the
    sign turned, it is the others that count: contexts are means of values between 1 and 2."""
    g = np.random.default_rng(plen)
    tops = [plen // 2, plen - 3]
    pk, tk = keys(g, nkv, plen, tops), keys(g, nseq * nkv, 20, []).reshape(nseq, nkv, 20, HD)
    pv, tv = ((1 + g.random(x.shape)).astype(F16) for x in (pk, tk))
    q = np.full((nseq, nkv * group, HD), size, F32)
    got = run_shared(hv, q, pk, pv, plen, tk, tv, None, [20 - s % 20 for s in range(nseq)], scale=sign * SCALE)
    assert np.isfinite(got).all()
    if sign > 0:
        # two equal scores, the next one log2 e * size * 128 * SCALE under them: 0 of the weight.
        # Their weights are equal, so only roundings of two terms and of the quotient remain
        want = pv[:, tops].astype(np.float64).mean(1).repeat(group, 0)
        assert np.abs(got - want).max() <= 64 * R.U
    assert (got >= 1 - 64 * R.U).all() and (got <= 2 + 64 * R.U).all()


@pytest.mark.parametrize("size", [1e3, 1e5, 1e7])
@pytest.mark.parametrize("where", ["first", "middle", "every third"])
@pytest.mark.parametrize("nkv,group,nseq,plen", [(2, 4, 3, 700), (8, 4, 40, 1500), (4, 8, 200, 3001)])
def test_scores_far_below_the_others(hv, size, where, nkv, group, nseq, plen):
    """Positions whose scores lie 2^18 to 2^31 below take nothing from what the others are told
    apart by: contexts are those of the others alone, at their own bound."""
    g = np.random.default_rng(plen)
    t = np.arange(plen)
    far = {"first": t < 300, "middle": (t > 250) & (t < 600), "every third": t % 3 == 0}[where]
    step = F16(2.0 ** np.round(np.log2(1 / size)))           # scores of the others are a few units
    pk = (g.integers(-8, 9, (nkv, plen, HD)) * step).astype(F16)
    pk[:, far] = -2
    tk = (g.integers(-8, 9, (nseq, nkv, 20, HD)) * step).astype(F16)
    pv, tv = (g.standard_normal(x.shape).astype(F16) for x in (pk, tk))
    q = np.full((nseq, nkv * group, HD), size, F32)
    tails = [20 - s % 20 for s in range(nseq)]
    got = run_shared(hv, q, pk, pv, plen, tk, tv, None, tails)
    some = [0, nseq // 2, nseq - 1]
    near(got[some], *R.shared(q[some], pk[:, ~far], pv[:, ~far], int((~far).sum()), tk[some], tv[some], None,
                              [tails[s] for s in some], SCALE))


@pytest.mark.parametrize("size", [1e4, 3e6, 3e7, 1e9, 1e12, 1e30])
@pytest.mark.parametrize("nkv,group,pos0,ntok", [(2, 4, 900, 1), (1, 2, 100, 20), (8, 4, 1000, 200), (2, 8, 0, 300)])
def test_mass(hv, size, nkv, group, pos0, ntok):
    """Contexts as above; weights are formed a second time and cannot be told from each other out
    there, but no weight is under 0 or over 1."""
    g = np.random.default_rng(ntok)
    n = pos0 + ntok
    k = keys(g, nkv, n, [0, n // 3])
    v = (1 + g.random(k.shape)).astype(F16)
    q = np.full((ntok, nkv * group, HD), size, F32)
    ctx, m = run_mass(hv, q, k, v, n - 1 if ntok == 1 else pos0, None, ntok == 1)
    want = np.stack([v[:, [0, n // 3] if pos0 + t >= n // 3 else [0]].astype(np.float64).mean(1) for t in range(ntok)])
    assert np.abs(ctx - want.repeat(group, 1)).max() <= 64 * R.U
    assert np.isfinite(m).all() and (m >= 0).all()
    assert (m <= ntok * group * (1 + (ntok * group + 64) * R.U)).all() or size < 1e7
    if ntok == 1 or size < 1e5:
        # (with ntok 1 the scores are formed once; 1e4 is 2^17 in the exponent, of which 2^-22 is 1 / 32)
        assert np.abs(m.sum(1) - ntok * group).max() <= ntok * group * (2 ** -4 if ntok > 1 else 64 * R.U)
