"""A plain numpy model of the 8-bit KV cache (include/hive_b200.h, hv_kv_q8_size) and of
attention over it, shared by its tests."""
import numpy as np

F32 = np.float32
BLK, HD = 32, 128
U = 2.0 ** -24                      # half an f32 step, relative


def quantise(x):
    """A block x f32 [32, 128] -> codes int [32, 128], scale f32 (NaN if x is not finite)."""
    x = np.asarray(x, F32)
    if not np.isfinite(x).all():
        return np.zeros(x.shape, np.int64), F32(np.nan)
    s = F32(np.abs(x).max() / F32(127))
    if s == 0:
        s = F32(1)
    with np.errstate(over="ignore"):
        t = (x / s).astype(F32) + np.where(x < 0, F32(-0.5), F32(0.5))
    return np.clip(np.trunc(t.astype(F32)), -127, 127).astype(np.int64), s


def values(c, s):
    return (c.astype(F32) * s).astype(F32)


def parts(nkv, cap):
    """Byte offsets of (scales, tail, held, end) in the buffer, and the blocks per head."""
    nblk = -(-cap // BLK)
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    a = nkv * nblk * 2 * BLK * HD
    b = a + up(nkv * nblk * 8)
    c = b + nkv * 2 * BLK * HD * 4
    return (a, b, c, c + up(nkv * 8)), nblk


def positions():
    """[which][r, d] -> byte of position r, dim d among a block's 4096 codes."""
    r, d = np.meshgrid(np.arange(BLK), np.arange(HD), indexing="ij")
    k = ((2 * (r // 8) + d // 64) * 512 + (4 * (r % 8) + d // 4 % 4) * 16
         + 4 * (d // 16 % 4) + d % 4)
    v = ((d // 16) * 512 + (4 * (d % 8) + r // 2 % 4) * 16 + 8 * (d // 8 % 2)
         + 4 * (r // 16) + 2 * (r // 8 % 2) + r % 2)
    return np.stack([k, v])


class Cache:
    """What the buffer holds: rows written in order, blocks quantised when complete."""

    def __init__(self, nkv, cap):
        self.nkv, self.cap, self.held = nkv, cap, 0
        self.val = np.full((2, nkv, cap, HD), np.nan, F32)
        self.codes = np.zeros((2, nkv, -(-cap // BLK), BLK, HD), np.int64)
        self.scale = np.ones((2, nkv, -(-cap // BLK)), F32)
        self.last = np.full((2, nkv, BLK, HD), np.nan, F32)     # f32 rows of the last block

    def write(self, k, v, pos0):
        """k, v [ntok, nkv, 128]."""
        if pos0 > self.held:
            return
        b0 = pos0 // BLK
        if pos0 % BLK and (self.held - 1) // BLK != b0:
            self.last[:] = self.val[:, :, b0 * BLK:(b0 + 1) * BLK]
        for t in range(len(k)):
            p = pos0 + t
            row = np.stack([k[t], v[t]])
            self.last[:, :, p % BLK] = row
            self.val[:, :, p] = row
            # rows of an open block read as f32 again
            b, r = p // BLK, p % BLK
            self.val[:, :, b * BLK:p + 1] = self.last[:, :, :r + 1]
            if r == BLK - 1:
                for w in range(2):
                    for h in range(self.nkv):
                        c, s = quantise(self.last[w, h])
                        self.codes[w, h, b], self.scale[w, h, b] = c, s
                        self.val[w, h, b * BLK:p + 1] = values(c, s)
        self.held = pos0 + len(k)
        self.val[:, :, self.held:] = np.nan

    def buffer(self, rest=0):
        """The library's buffer with these contents; bytes it does not define are `rest`."""
        (a, b, c, end), nblk = parts(self.nkv, self.cap)
        buf = np.full(end, rest, np.uint8)
        at, closed = positions(), self.held // BLK
        codes = buf[:a].reshape(self.nkv, nblk, 2, BLK * HD)
        scales = buf[a:a + self.nkv * nblk * 8].view(F32).reshape(self.nkv, nblk, 2)
        for w in range(2):
            for h in range(self.nkv):
                for j in range(closed):
                    codes[h, j, w, at[w]] = (self.codes[w, h, j] + 128).astype(np.uint8)
                    scales[h, j, w] = self.scale[w, h, j]
        tail = buf[b:c].view(F32).reshape(self.nkv, 2, BLK, HD)
        rows = (self.held - 1) % BLK + 1 if self.held else 0
        tail[:, :, :rows] = self.last.swapaxes(0, 1)[:, :, :rows]
        buf[c:c + self.nkv * 8].view(np.int32)[:] = self.held
        return buf


def attention(q, val, pos, group, scale):
    """q [nq, 128] over positions 0..pos of val [2, nkv, cap, 128] in 64 bits -> ctx f64, and a
    bound on an f32 evaluation's error per element.

    With u = 2^-24: a score is a sum of 128 products, q in two 11-bit terms (4u of |q||k|),
    at most 16 partial sums of an accumulator that may cut instead of round (2u each), then
    the scale and log2 e (2u each), so |dx| <= 44 u B, B = scale * max_t sum_i |q_i k_ti|;
    subtracting the maximum and 2^x add 4u |x| <= 4 u B; weights are off by that on both sides
    of the quotient: 96 u B. (Keys of the open block have two terms too, the second exact to
    2^-38 of the block's largest, which adds 2^-14 sum_i |q_i| times that to B.) The weighted
    sum adds each of the n positions once in tiles of 16 and 32: (n / 8 + 64) u of sum w |v|
    covers it with the sum of the weights.
    A weight enters the second product as two binary16 terms, and what is left is at most half
    of binary16's smallest step, 2^-25, whatever the weight. At the least it stands as 2^11
    times w s over the largest w s, s the scale that its block's values have been divided by:
    codes go to 127, the open block's values to 2^10. So w |v| is off by at most 2^-36 127
    max(w s) = 2^-36 max(w V) in a coded block, where V is a block's largest |v|, and by 2^-36
    2^10 max(w s) <= 2^-33 max(w V) in the open one, whose second terms of v add 2^-34 V w. The
    n positions together: 2^-32 n max(w V)."""
    q = q.astype(np.float64)
    out, tol = np.empty(q.shape), np.empty(q.shape)
    n = pos + 1
    for h in range(q.shape[0]):
        k, v = val[:, h // group, :n].astype(np.float64)
        x = (k @ q[h]) * scale
        big = (np.abs(k) @ np.abs(q[h])).max() * abs(scale)
        big += 2.0 ** -14 * np.abs(q[h]).sum() * np.abs(k[n // BLK * BLK:]).max(initial=0)
        peak = np.abs(v).max(1)
        peak = np.maximum.reduceat(peak, np.arange(0, n, BLK)).repeat(BLK)[:n]
        w = np.exp(x - x.max())
        w /= w.sum()
        out[h] = w @ v
        tol[h] = (96 * U * big + (n / 8 + 64) * U) * (w @ np.abs(v))
        tol[h] += 2.0 ** -32 * n * (w * peak).max() + 1e-37
    return out, tol
