"""The 8-bit layer operators in float64 (numpy), from their definitions."""
import numpy as np

BLOCK = 64


def nearest(v):
    """To the nearest whole number, halves away from zero, within +-127."""
    return np.clip(np.sign(v) * np.floor(np.abs(v) + 0.5), -127, 127)


def norm8(x, res, w, eps, norm=True):
    """(sum, q, scales); rows in float64."""
    s = x if res is None else x + res
    t = s * w if norm else s
    most = np.abs(t).max(1)
    live = most > 0
    q = nearest(np.divide(t * 127, most[:, None], out=np.zeros_like(t), where=live[:, None]))
    rms = np.sqrt((s * s).mean(1) + eps) if norm else 1.0
    return s, q.astype(np.int8), np.where(live, most / 127 / rms, 1.0)


def gemm8(a, sa, w, sw, bias=None):
    """(sums, products) of int8 rows."""
    acc = a.astype(np.float64) @ w.astype(np.float64).T          # below 2^53: exact
    y = acc * np.asarray(sa, np.float64)[:, None] * np.asarray(sw, np.float64)
    return acc, y if bias is None else y + np.asarray(bias, np.float64)


def slots():
    """Where each position of a block stands among the 64 bytes of a dim of V."""
    p = np.arange(BLOCK)
    return (p // 4 % 4) * 16 + p // 16 * 4 + p % 4


class Cache:
    """One cache: q [seq][head][position][dim] and s [seq][head][block], for K and V."""

    def __init__(self, n_seq, heads, cap, dim):
        self.shape = (n_seq, heads, cap, dim)
        self.q = {n: np.zeros(self.shape, np.int64) for n in "kv"}
        self.s = {n: np.zeros((n_seq, heads, cap // BLOCK), np.float32) for n in "kv"}

    def fill(self, r):
        """Random contents."""
        for n in "kv":
            self.q[n] = np.clip(np.rint(r.normal(0, 32, self.shape)), -127, 127).astype(np.int64)
            self.s[n] = r.uniform(0.01, 0.04, self.s[n].shape).astype(np.float32)
        return self

    def write(self, j, pos, rows):
        """rows: {"k": [n][head][dim], "v": ...} float64 at positions pos .. of sequence j."""
        cap = self.shape[2]
        for n in "kv":
            x = rows[n]
            lo, hi = max(pos, 0), min(pos + len(x), cap)
            for b in range(lo // BLOCK, (hi + BLOCK - 1) // BLOCK if hi > lo else 0):
                p0, p1 = max(lo, b * BLOCK), min(hi, (b + 1) * BLOCK)
                y = x[p0 - pos:p1 - pos].transpose(1, 0, 2)                       # [head][n][dim]
                fin = np.isfinite(y)
                new = (np.abs(np.where(fin, y, 0)).max((1, 2)) / 127).astype(np.float32)
                old = self.s[n][j, :, b].copy()
                s = np.maximum(new, old) if p0 > b * BLOCK else new
                sd = s.astype(np.float64)[:, None, None]
                one = np.where(sd > 0, sd, 1)
                if p0 > b * BLOCK:
                    was = self.q[n][j, :, b * BLOCK:p0]
                    grown = (s > old)[:, None, None]
                    self.q[n][j, :, b * BLOCK:p0] = np.where(grown, nearest(was * old.astype(np.float64)[:, None, None] / one), was)
                q = nearest(np.where(fin, y, 0) / one)
                q = np.where(np.isinf(y), np.sign(np.where(np.isnan(y), 0, y)) * 127, q)
                self.q[n][j, :, p0:p1] = np.where(sd > 0, q, 0)
                self.s[n][j, :, b] = s

    def values(self, n):
        return self.q[n] * np.repeat(self.s[n].astype(np.float64), BLOCK, 2)[..., None]

    def stored(self):
        """(k8, v8, k_scales, v_scales) as the library lays them out."""
        ns, h, cap, d = self.shape
        v = self.q["v"].reshape(ns, h, cap // BLOCK, BLOCK, d)
        v8 = np.empty((ns, h, cap // BLOCK, d, BLOCK), np.int8)
        v8[..., slots()] = v.transpose(0, 1, 2, 4, 3)
        return self.q["k"].astype(np.int8), v8, self.s["k"], self.s["v"]


def attend(q, k, v, pos, scale, window=0, sinks=0, steps=8.0e6):
    """q [n][G * heads][dim] over k, v [heads][cap][dim]; row i sees positions up to pos + i.
    steps: the whole numbers that the largest value of a row of q, and the largest weight of a block, count.
    Returns (out, bound): bound on what the operator's arithmetic may lose (see below)."""
    n, hq, d = q.shape
    heads, cap, _ = k.shape
    g = hq // heads
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    p = np.arange(cap)
    for i in range(n):
        last = pos + i
        seen = (p <= last) & ((p > last - window) | (p < sinks) if window else True)
        if not seen.any():
            continue
        for h in range(hq):
            kk, vv = k[h // g][seen], v[h // g][seen]
            s = scale * (kk @ q[i, h])
            e = np.exp(s - s.max())
            w = e / e.sum()
            out[i, h] = w @ vv
            # a weight's relative error, twice (the sum has it too).  The score: q in whole numbers of max|q| / steps, half
            # a one off against |k|; six roundings of it (the step's factor and its inverse, scale x log2 e, the block's
            # scale, two of the sum, the product); the difference from the maximum; the exponential's unit in the last
            # place.  Then the block's scale, the rescaling of the sums at each block and their additions
            u = 2.0 ** -24
            score = abs(scale) * np.abs(kk).sum(1) * np.abs(q[i, h]).max() / (2 * steps) + 8 * u * np.abs(s) + u * np.abs(s - s.max())
            blocks = (seen.sum() + 2 * BLOCK) // BLOCK + 1
            # a block's weights are whole numbers of its largest / steps, half a one off against |v|
            at = p[seen] // BLOCK
            top = np.zeros(cap // BLOCK)
            np.maximum.at(top, at, w)
            whole = (top[at] / (2 * steps)) @ np.abs(vv)
            bound[i, h] = (2 * score.max() + (4 * blocks + 24) * u) * (w @ np.abs(vv)) + 1.01 * whole
    return out, bound
