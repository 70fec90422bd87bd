"""The 8-bit paged K/V pool and the log probabilities in float64 (numpy), from
their definitions in include/g4hip.h."""
import numpy as np


def exponent(amax):
    """The least e >= -64 with amax <= 127 * 2^e."""
    m, x = np.frexp(np.asarray(amax, np.float64))
    return np.where(np.asarray(amax) > 0, np.maximum(x - 7 + (m > 127 / 128), -64), -64)


def normed(x, w=None, eps=1e-6):
    x = np.asarray(x, np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(eps)))
    return y if w is None else y * w.astype(np.float64)


def rotated(x, cs):
    """x [rows][heads][dim], cs [rows][dim / 2][2]."""
    half = x.shape[-1] // 2
    c, s = (cs[:, None, :, i].astype(np.float64) for i in (0, 1))
    return np.concatenate([x[..., :half] * c - x[..., half:] * s, x[..., :half] * s + x[..., half:] * c], -1)


class Pool:
    """K or V pages: codes int8 [pages][page_size][heads][dim], scale [pages][heads]."""

    def __init__(self, codes, scale):
        self.codes, self.scale = codes.copy(), scale.copy()
        self.border = np.inf  # how near a value has come to the border of two codes

    def append(self, x, table, first):
        """Rows x [n][heads][dim] at positions first, first + 1, ... of the page list."""
        ps, n = self.codes.shape[1], len(x)
        for j in range(first // ps, (first + n - 1) // ps + 1):
            pg = table[j]
            if pg < 0 or pg >= len(self.codes):
                continue
            a, b = max(first, j * ps), min(first + n, (j + 1) * ps)
            new, lo = x[a - first:b - first], a - j * ps
            for h in range(x.shape[1]):
                old = self.scale[pg, h]
                if not np.all(np.isfinite(new[:, h])) or (lo and np.isnan(old)):
                    self.scale[pg, h] = np.nan
                    self.codes[pg, lo:lo + b - a, h] = 0
                    continue
                s = 2.0 ** exponent(np.abs(new[:, h]).max())
                if lo:
                    s = max(s, float(old))
                    self.codes[pg, :lo, h] = np.clip(np.rint(self.codes[pg, :lo, h] * (float(old) / s)), -127, 127)
                self.scale[pg, h] = s
                y = new[:, h] / s
                self.border = min(self.border, np.abs(y - np.floor(y) - 0.5).min())
                self.codes[pg, lo:lo + b - a, h] = np.rint(y)

    def values(self):
        with np.errstate(invalid="ignore"):
            return self.codes * self.scale[:, None, :, None].astype(np.float64)


def attend(q, k, v, table, pos, window, scale):
    """One row: q [heads][dim] at position pos over value pools k, v; the output, sum p |v|, the largest sum |q k|."""
    heads, dim = q.shape
    g = heads // k.shape[2]
    out, mag, reach = np.zeros((heads, dim)), np.zeros((heads, dim)), np.zeros((heads, 1))
    if pos < 0:
        return out, mag, reach
    ps = k.shape[1]
    t = np.arange(max(0, pos + 1 - window) if window else 0, pos + 1)
    pg = np.clip(np.asarray(table)[t // ps], 0, len(k) - 1)
    for h in range(heads):
        x = (k[pg, t % ps, h // g] @ q[h].astype(np.float64)) * float(np.float32(scale))
        p = np.exp(x - x.max())
        p /= p.sum()
        vv = v[pg, t % ps, h // g]
        out[h], mag[h] = p @ vv, p @ np.abs(vv)
        reach[h] = (np.abs(k[pg, t % ps, h // g]) @ np.abs(q[h].astype(np.float64))).max() * abs(scale)
    return out, mag, reach


def logprobs(x, token, ntop):
    """One row: (logprob, entropy, ids, their logprobs)."""
    x = np.asarray(x, np.float32)
    order = np.lexsort((np.arange(x.size), np.where(np.isnan(x), np.inf, -x.astype(np.float64)), np.isnan(x)))[:ntop]
    y = x.astype(np.float64)
    if np.isnan(y).any() or y.max() == np.inf or y.max() == -np.inf:
        return np.nan, np.nan, order, np.full(ntop, np.nan)
    z = y - y.max()
    lp = z - np.log(np.exp(z).sum())
    p = np.exp(lp)
    ent = -(p[p > 0] * lp[p > 0]).sum()
    return lp[token] if 0 <= token < x.size else np.nan, ent, order, lp[order]
