"""The 4-bit paged K/V pool, its weighed rows and their eviction in float64 (numpy), from their definitions in
include/g4hip.h."""
import numpy as np

LEVELS = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
VALUES = np.concatenate([LEVELS, -LEVELS])
BORDERS = np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5])
EVEN_ABOVE = (.75, 1.75, 3.5)  # the borders that go to the code above them


def encode(x):
    """Rows x [..., dim]: codes [..., dim] and scale bytes [..., dim / 32], of finite rows and others; how near a value
    is to the border of two codes or of two scales, relative to it."""
    x = np.asarray(x, np.float64)
    b = x.reshape(x.shape[:-1] + (-1, 32))
    fine = np.isfinite(x).all(-1)
    top = np.abs(np.where(fine[..., None, None], b, 0)).max(-1)
    m, e = np.frexp(top)
    e = np.where(top > 0, np.maximum(e - 3 + (m > 0.875), -20), -20)
    y = np.where(fine[..., None, None], b, 0) / 2.0 ** e[..., None]
    a = np.abs(y)
    codes = np.searchsorted(BORDERS, a) + np.isin(a, EVEN_ABOVE)
    codes = (codes | np.signbit(y) << 3).reshape(x.shape).astype(np.uint8)
    near = min(np.abs(a[..., None] - BORDERS).min(), np.abs(m[top > 0] - 0.875).min(initial=1.0))
    return np.where(fine[..., None], codes, 0).astype(np.uint8), np.where(fine[..., None], e + 127, 255).astype(np.uint8), near


def values(codes, scale):
    s = np.where(scale == 255, np.nan, 2.0 ** (scale.astype(np.float64) - 127))
    return VALUES[codes] * np.repeat(s, 32, -1)


class Pool:
    """K or V pages: codes [pages][page_size][heads][dim] (one a byte here), scale bytes [pages][page_size][heads][dim / 32]."""

    def __init__(self, codes, scale):
        self.codes, self.scale = codes.copy(), scale.copy()
        self.border = np.inf

    def append(self, x, table, first):
        """Rows x [n][heads][dim] at places first, first + 1, ... of the page list."""
        codes, scale, near = encode(x)
        self.border = min(self.border, near)
        ps = self.codes.shape[1]
        for i in range(len(x)):
            pg, slot = table[(first + i) // ps], (first + i) % ps
            if 0 <= pg < len(self.codes):
                self.codes[pg, slot], self.scale[pg, slot] = codes[i], scale[i]

    def values(self):
        return values(self.codes, self.scale)

    def packed(self):
        return (self.codes[..., ::2] | self.codes[..., 1::2] << 4).astype(np.uint8)

    def by_tile(self):
        """V's scales as the pool lies: [pages][page_size / 16][heads][dim / 32][16]."""
        p, ps, h, nb = self.scale.shape
        return np.ascontiguousarray(self.scale.reshape(p, ps // 16, 16, h, nb).transpose(0, 1, 3, 4, 2))


def unpack(codes):
    return np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[:-1] + (-1,))


def by_row(scale):
    p, t, h, nb, _ = scale.shape
    return scale.transpose(0, 1, 4, 2, 3).reshape(p, 16 * t, h, nb)


def attend(q, k, v, table, pos, window, scale):
    """One row: q [heads][dim] at place pos over value pools k, v. The output, sum p |v|, the reach of the scores' sums
    (of |k| (|q| + its block's largest / 32)), and the weights [heads][first ..= pos]."""
    heads, dim = q.shape
    g = heads // k.shape[2]
    out, mag, reach = np.zeros((heads, dim)), np.zeros((heads, dim)), np.zeros((heads, 1))
    ps = k.shape[1]
    first = max(0, pos + 1 - window) if window else 0
    t = np.arange(first, pos + 1)
    pg = np.clip(np.asarray(table)[t // ps], 0, len(k) - 1)
    p = np.zeros((heads, len(t)))
    scale = float(np.float32(scale))
    for h in range(heads):
        kk, qq = k[pg, t % ps, h // g], q[h].astype(np.float64)
        x = (kk @ qq) * scale
        top = np.repeat(np.abs(qq.reshape(-1, 32)).max(-1), 32)
        e = np.exp(x - x.max())
        p[h] = e / e.sum()
        vv = v[pg, t % ps, h // g]
        out[h], mag[h] = p[h] @ vv, p[h] @ np.abs(vv)
        reach[h] = (np.abs(kk) @ (np.abs(qq) + top / 32)).max() * abs(scale)
    return out, mag, reach, p


def chosen(mass, first, recent, keep):
    """Places that a head keeps of its rows' masses, in order."""
    n = len(mass)
    middle = np.arange(first, n - recent)
    heavy = np.where(mass[middle] > 0, mass[middle], 0).astype(np.float64)
    heavy = middle[np.argsort(-heavy, kind="stable")[:keep - first - recent]]
    return np.concatenate([np.arange(first), np.sort(heavy), np.arange(n - recent, n)]).astype(np.int64)


def evict(k, v, mass, table, lens, keep, first, recent, max_len):
    """Pools k, v and mass [pages][page_size][heads] in place; (kept, lengths after)."""
    pages, ps, heads = mass.shape
    kept = np.full((len(lens), heads, keep), -1, np.int32)
    after = np.array(lens)
    for s, n in enumerate(lens):
        if n > max_len:
            continue
        if n <= keep:
            kept[s, :, :n] = np.arange(n)
            continue
        t = np.arange(n)
        ids = np.asarray(table[s])[t // ps]
        there, pg = (ids >= 0) & (ids < pages), np.clip(ids, 0, pages - 1)
        for h in range(heads):
            m = np.where(there, mass[pg, t % ps, h], 0)
            src = chosen(m, first, recent, keep)
            kept[s, h] = src
            dst = np.flatnonzero((src != np.arange(keep)) & there[:keep])
            for a in (k.codes, k.scale, v.codes, v.scale):
                a[pg[dst], dst % ps, h] = a[pg[src[dst]], src[dst] % ps, h]
            mass[pg[dst], dst % ps, h] = m[src[dst]]
        after[s] = keep
    return kept, after
