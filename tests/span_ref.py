"""Plain 64-bit forms of the attention over binary16 caches (shared prefixes, weights added up) and
of eviction, shared by their tests."""
import numpy as np

F32 = np.float32
HD = 128
U = 2.0 ** -24                      # half an f32 step, relative


def attend(q, k, v, scale):
    """One query head q [128] over k, v [n, 128] (binary16 values) in 64 bits -> context, a bound
    on an f32 evaluation's error, weights, a bound on theirs (relative, then absolute).

    With u = 2^-24: a score is a sum of 128 products, q in two 11-bit terms (4u of |q||k|), at
    most 16 partial sums of an accumulator that may cut instead of round (2u each), then the
    scale and log2 e (2u each), so |dx| <= 44 u B, B = scale * max_t sum_i |q_i k_ti|; values of q
    under 2^-14 of its largest are exact to 2^-38 of that only, which adds 2^-37 max|q| sum_i
    |k_ti| to B u^-1 / 44, less than 2^-18 max|q| sum_i |k_ti| to B; subtracting the maximum and
    2^x add 4 u B; weights are off by that on both sides of the quotient: 96 u B, and 4 u for
    2^x and the quotient themselves. The weighted sum adds each of the n positions once in tiles
    of at least 16: (n / 8 + 64) u of sum w |v| covers it with the sum of the weights.
    A weight enters the second product as two binary16 terms and is then exact to 2^-22 (in the
    64 u) or to half of binary16's smallest step, 2^-25. At the least it stands as 2^8 times itself
    over 2^m, m a whole number at most 1 over the largest exponent so far, which is 2^-32 of the
    largest weight, and where m rose meanwhile what stood was scaled down, another 2^-32:
    2^-31 n max w max|v|."""
    n = len(k)
    if n == 0:
        return np.zeros(HD), np.full(HD, 1e-37), np.zeros(0), np.zeros(0)
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    x = (k @ q) * scale
    big = (np.abs(k) @ np.abs(q) + 2.0 ** -18 * np.abs(q).max() * np.abs(k).sum(1)).max() * abs(scale)
    w = np.exp(x - x.max())
    w /= w.sum()
    off = 96 * U * big + 4 * U
    tol = (off + (n / 8 + 64) * U) * (w @ np.abs(v)) + 2.0 ** -31 * n * w.max() * np.abs(v).max(0)
    return w @ v, tol + 1e-37, w, off * w + (n / 8 + 64) * U * w + 2.0 ** -124


def rows_of(row0, nrow, tlen):
    """(row, sequence, positions of its tail that it sees) of every row that has a sequence."""
    out = []
    for s in range(len(tlen)):
        lo, hi = (s, s + 1) if row0 is None else (row0[s], row0[s + 1])
        out += [(r, s, max(0, tlen[s] - (hi - 1 - r))) for r in range(lo, hi)]
    return out


def shared(q, pk, pv, plen, tk, tv, row0, tlen, scale):
    """q [nrow, nq, 128]; pk, pv [nkv, pcap, 128]; tk, tv [nseq, nkv, tcap, 128] -> context f64
    and its bound; rows without a sequence NaN."""
    nrow, nq, _ = q.shape
    nkv = tk.shape[1]
    out, tol = np.full(q.shape, np.nan), np.zeros(q.shape)
    for r, s, n in rows_of(row0, nrow, tlen):
        for h in range(nq):
            g = h // (nq // nkv)
            k = np.concatenate([pk[g, :plen], tk[s, g, :n]])
            v = np.concatenate([pv[g, :plen], tv[s, g, :n]])
            out[r, h], tol[r, h] = attend(q[r, h], k, v, scale)[:2]
    return out, tol


def mass(q, k, v, pos0, mass_in, scale):
    """Causal: row t of q [ntok, nq, 128] over positions 0 .. pos0 + t of k, v [nkv, cap, 128] ->
    context, bound, mass [nkv, pos0 + ntok], bound. A mass is a sum of rows * heads weights, each
    added once (in any order: one u a weight), to mass_in, which counts before pos0."""
    ntok, nq, _ = q.shape
    nkv = k.shape[0]
    group, n = nq // nkv, pos0 + ntok
    out, tol = np.empty(q.shape), np.empty(q.shape)
    m = np.zeros((nkv, n))
    if mass_in is not None:
        m[:, :pos0] = mass_in[:, :pos0]
    mt = 4 * U * np.abs(m)
    for t in range(ntok):
        for h in range(nq):
            g, e = h // group, pos0 + t + 1
            out[t, h], tol[t, h], w, wt = attend(q[t, h], k[g, :e], v[g, :e], scale)
            m[g, :e] += w
            mt[g, :e] += wt + (ntok * group + 8) * U * w
    return out, tol, m, mt


def evict(mass, n, limit, keep, recent):
    """Positions that stay of one cache and head, in order: mass [cap]."""
    if n <= limit:
        return np.arange(n)
    old = mass[:n - recent].astype(np.float64)
    old = np.where(np.isnan(old), np.inf, old) if not np.isposinf(old).any() else np.where(
        np.isnan(old), np.inf, np.where(np.isposinf(old), np.finfo(np.float64).max, old))
    best = np.lexsort((np.arange(old.size), -old))[:keep - recent]
    return np.concatenate([np.sort(best), np.arange(n - recent, n)])
