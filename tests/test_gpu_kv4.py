"""The 4-bit paged K/V pool on the GPU: the prologue's codes, scales and q, the values read back, the attention and
the weights that it adds up, and the eviction, against float64 (kv4_oracle).

Codes and scales are equal to the oracle's: both round a value that is off by at most about 1e-13 of itself, and the
oracle's distance to the next border is checked to be more than 1e-9. q: as in the 8-bit pool's tests, (parts + 10) *
2^-24 of what |x0| + |x1| would be with the parts' magnitudes in their place.

Attention: a score is a sum in f32 of at most 5 terms (q's parts of 5 bits) for each 128 dims, each of them off by
2^-23 of its own magnitudes' sum: R = sum |k| (|q| + its block's largest / 32) bounds those of the first part, and the
others are 2^-5 of it and less. With 6 roundings more (q's last part, the scale, the exponent) a score is off by U (2 * 1.1
+ 5 J + 6) R, J = max(1, dim / 128), a weight by that of itself, the quotient by twice that, and its sums (over at most n
/ 32 steps and 40 joins) by (40 + n / 32) U more. P is held to 2^-40 of the largest, each of n times at most the
largest |v|. A weight that is added up: the same of itself, and of the sum of m of them m U."""
import numpy as np
import pytest

import g4hip
import kv4_oracle as K4
import kv8_oracle as K8

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def slack(hd, n, reach):
    """How far a weight may be off, of itself."""
    return U * (2 * (2.2 + 5 * max(1, hd // 128) + 6) * reach + 40 + n / 32)


class Case:
    """A batch with its pages on the host and the device; `rows` new rows per sequence, lengths counting them."""

    def __init__(self, ctx, lens, rows, nqh, nkh, hd, ps, seed, spare=2, window=0, scale=1.0, parts=1, extra_rows=0,
                 max_len=None):
        self.ctx, self.parts, self.hd = ctx, parts, hd
        self.lens, self.n = np.asarray(lens), np.asarray(rows)
        rng = self.rng = np.random.default_rng(seed)
        S, R = len(lens), int(self.n.sum()) + extra_rows
        max_len = max_len or max(1, int(self.lens.max()))
        self.width = -(-max_len // ps)
        per = np.minimum(-(-np.maximum(self.lens, 1) // ps), self.width)
        self.pages = int(per.sum()) + spare
        order = rng.permutation(self.pages)
        self.table = np.full((S, self.width), -1, np.int32)
        at = 0
        for s in range(S):
            self.table[s, :per[s]] = order[at:at + per[s]]
            at += per[s]
        self.starts = np.concatenate([[0], np.cumsum(self.n)]).astype(np.uint32)
        self.one = extra_rows == 0 and np.all(self.n == 1)
        self.p = ctx.kv4_params(S, nqh, nkh, hd, ps, self.width, max_len, self.pages, num_rows=R,
                                max_rows=max(1, int(self.n.max())), window=window, scale=scale)
        shape = (2, self.pages, ps, nkh)
        codes = rng.integers(0, 16, (*shape, hd)).astype(np.uint8)
        exps = rng.integers(-3, 1, (*shape, hd // 32)) + 127 - 1
        self.k, self.v = (K4.Pool(codes[i], exps[i].astype(np.uint8)) for i in (0, 1))
        self.mass = np.abs(rng.normal(size=shape[1:])).astype(np.float32)
        self.q = rng.normal(0, 1.0 / np.sqrt(hd), (R, nqh, hd)).astype(np.float32)

    def up(self):
        c = self.ctx
        self.dk, self.dv = c.from_numpy(self.k.packed()), c.from_numpy(self.v.packed())
        self.dks, self.dvs = c.from_numpy(self.k.scale), c.from_numpy(self.v.by_tile())
        self.dm = c.from_numpy(self.mass)
        self.dt, self.dl = c.from_numpy(self.table), c.from_numpy(self.lens.astype(np.uint32))
        self.ds = None if self.one else c.from_numpy(self.starts)
        self.cache = (self.dk, self.dv, self.dks, self.dvs)
        return self

    def row(self, r):
        """(sequence, place) of row r."""
        s = int(np.searchsorted(self.starts, r, side="right")) - 1
        return s, int(self.lens[s]) - int(self.n[s]) + r - int(self.starts[s])

    def attention(self, workspace=None, mass=False, ops=None):
        c, p = self.ctx, self.p
        out = c.from_numpy(np.full(self.q.shape, 7.5, np.float32))
        ws = workspace
        if ws is None:  # of any content
            ws = c.from_numpy(np.full(c.attn4_workspace_bytes(p, mass), 0xff, np.uint8))
        c.pagedAttn4(c.from_numpy(self.q), *self.cache, self.dt, self.dl, out, p, ws, row_starts=self.ds,
                     mass=self.dm if mass else None, ops=ops)
        return out.download(np.float32).reshape(self.q.shape)

    def check_attention(self, got, rows=None, what=""):
        k, v = self.k.values(), self.v.values()
        total = int(self.n.sum())
        for r in range(total) if rows is None else rows:
            s, pos = self.row(r)
            if pos < 0:
                assert np.all(got[r] == 0), (what, r)
                continue
            want, mag, reach, _ = K4.attend(self.q[r], k, v, self.table[s], pos, self.p.sliding_window, self.p.scale)
            ps = self.k.codes.shape[1]
            pages = np.clip(self.table[s][:pos // ps + 1], 0, self.pages - 1)
            tol = slack(self.hd, pos + 1, reach) * mag + 2.0 ** -40 * (pos + 1) * np.nanmax(np.abs(v[pages])) + 1e-30
            off = float((np.abs(got[r] - want) / tol).max())
            assert off <= 1, (what, r, s, pos, off)
        assert np.all(got[total:] == 7.5), what

    def weighed(self):
        """Adds what the call's rows give to every cached row, and how far each may be off."""
        k, v = self.k.values(), self.v.values()
        more, tol = np.zeros(self.mass.shape), np.zeros(self.mass.shape)
        ps, g = k.shape[1], self.q.shape[1] // k.shape[2]
        for r in range(int(self.n.sum())):
            s, pos = self.row(r)
            if pos < 0:
                continue
            _, _, reach, p = K4.attend(self.q[r], k, v, self.table[s], pos, self.p.sliding_window, self.p.scale)
            t = np.arange(pos + 1 - p.shape[1], pos + 1)
            ids = self.table[s][t // ps]
            there = (ids >= 0) & (ids < self.pages)
            for h in range(len(p)):
                at = (ids[there], t[there] % ps, h // g)
                more[at] += p[h][there]
                tol[at] += p[h][there] * slack(self.hd, pos + 1, reach[h, 0]) + 2.0 ** -126
        return more, tol + (int(self.n.max()) * g + 2) * U * more

    def check_mass(self, before, what="", times=1):
        more, tol = self.weighed()
        got = self.dm.download(np.float32).reshape(self.mass.shape)
        want = before.astype(np.float64) + times * more
        off = np.abs(got - want) / (times * tol + times * U * np.abs(want) + 1e-38)
        assert np.nanmax(off) <= 1, (what, np.nanmax(off), np.unravel_index(np.nanargmax(off), off.shape))
        assert np.array_equal(got[more == 0], before[more == 0], equal_nan=True), what


def table_of(ctx, hd, rows, theta=1e4):
    t = ctx.empty(rows * hd, np.float32)
    ctx.ropeTable(theta, 0, None, hd, rows, t)
    return t, t.download(np.float32).reshape(rows, hd // 2, 2)


def prologue(c: Case, q=None, k=None, v=None, table=None, qw=None, kw=None, positions=None, rope_rows=None,
             with_mass=True):
    """Runs the prologue and checks q, codes, scales and masses; returns q."""
    ctx, p, hd = c.ctx, c.p, c.hd
    R = p.num_rows
    pos = np.asarray(c.lens if positions is None else positions).astype(np.int64)
    rows_of_table = rope_rows or p.max_seq_len
    host_table = table_of(ctx, hd, max(int(pos.max()), rows_of_table, 1))[1]
    freqs = ctx.from_numpy(np.ones(hd // 2, np.float16))
    out = ctx.from_numpy(np.full(R * p.num_q_heads * hd, 3.25, np.float32))
    dev = [None if x is None else ctx.from_numpy(x) for x in (q, k, v, qw, kw)]
    cache = c.cache if k is not None else (None, None, None, None)
    ctx.pagedAttnPrologue4(dev[0], dev[1], dev[2], c.parts, dev[3], dev[4], freqs, out if q is not None else None,
                           *cache, c.dt, c.dl, p, row_starts=c.ds, mass=c.dm if with_mass else None,
                           positions=None if positions is None else ctx.from_numpy(pos.astype(np.uint32)),
                           rope_cs=table, rope_rows=rows_of_table if table else 0)
    got = out.download(np.float32).reshape(R, p.num_q_heads, hd)
    done = np.zeros(R, bool)
    for s in range(p.num_seqs):
        a, n, L = int(c.starts[s]), int(c.n[s]), int(c.lens[s])
        if n == 0 or L < n or L > p.max_seq_len or n > p.max_rows:
            continue
        if pos[s] < n or (table and pos[s] > rows_of_table):
            continue
        done[a:a + n] = True
        cs = host_table[pos[s] - n:pos[s]]
        if q is not None:
            y = q[:, a:a + n].astype(np.float64)
            x, half = K8.normed(y.sum(0), qw), hd // 2
            rms = np.sqrt((y.sum(0) ** 2).mean(-1, keepdims=True) + 1e-6)
            mag = np.abs(y).sum(0) / rms * np.abs(qw.astype(np.float64))
            mag = np.tile(mag[..., :half] + mag[..., half:], 2)
            off = np.abs(got[a:a + n] - K8.rotated(x, cs)) / ((c.parts + 10) * U * mag + 1e-30)
            assert off.max() <= 1, off.max()
        if k is not None:
            with np.errstate(invalid="ignore"):
                kk = K8.rotated(K8.normed(k[:, a:a + n].astype(np.float64).sum(0), kw), cs)
                vv = K8.normed(v[:, a:a + n].astype(np.float64).sum(0))
            c.k.append(kk, c.table[s], L - n)
            c.v.append(vv, c.table[s], L - n)
            for t in range(L - n, L):
                pg = c.table[s, t // p.page_size]
                if with_mass and 0 <= pg < c.pages:
                    c.mass[pg, t % p.page_size] = 0
    assert np.all(got[~done] == 3.25)
    if k is not None:
        check_pools(c)
    return got


def check_pools(c):
    assert min(c.k.border, c.v.border) > 1e-9
    for pool, d, ds, rows in ((c.k, c.dk, c.dks, lambda x: x), (c.v, c.dv, c.dvs, K4.by_row)):
        shape = pool.by_tile().shape if rows is K4.by_row else pool.scale.shape
        np.testing.assert_array_equal(rows(ds.download(np.uint8).reshape(shape)), pool.scale)
        codes = K4.unpack(d.download(np.uint8).reshape(pool.packed().shape))
        np.testing.assert_array_equal(np.where(codes == 8, 0, codes), np.where(pool.codes == 8, 0, pool.codes))
    np.testing.assert_array_equal(c.dm.download(np.float32).reshape(c.mass.shape), c.mass)


def projections(c, seed, spread=1.0):
    rng, p = np.random.default_rng(seed), c.p
    return [rng.normal(0, spread, (c.parts, p.num_rows, n, c.hd)).astype(np.float32)
            for n in (p.num_q_heads, p.num_kv_heads, p.num_kv_heads)] + [
        (1 + 0.1 * rng.normal(size=c.hd)).astype(np.float16) for _ in range(2)]


SHAPES = [  # lens, rows, query heads, K/V heads, dim, page size, parts
    ([1], [1], 8, 1, 256, 16, 1),
    ([16, 17, 5, 33], [1, 1, 1, 1], 8, 1, 256, 16, 6),
    ([40, 100, 7], [40, 33, 1], 4, 2, 128, 32, 2),
    ([90], [90], 8, 1, 512, 16, 1),
    ([70, 3, 150], [5, 3, 101], 2, 2, 64, 64, 3),
    ([130, 31], [97, 0], 16, 1, 128, 96, 1),
    ([3, 50], [1, 1], 5, 1, 64, 16, 1),
    ([30, 9], [7, 9], 9, 3, 512, 1024, 5),
]


@pytest.mark.parametrize("lens,rows,nqh,nkh,hd,ps,parts", SHAPES)
@pytest.mark.parametrize("form", ["angles", "table", "angles, moved", "table, moved"])
def test_prologue(ctx, lens, rows, nqh, nkh, hd, ps, parts, form):
    c = Case(ctx, lens, rows, nqh, nkh, hd, ps, 11, parts=parts, extra_rows=2 if len(lens) > 1 else 0).up()
    q, k, v, qw, kw = projections(c, 12)
    gone = np.array([1000, 0, 7, 300])[:len(lens)] if "moved" in form else 0
    most = int((c.lens + gone).max())
    table = table_of(ctx, hd, most)[0] if "table" in form else None
    prologue(c, q, k, v, table, qw, kw, positions=c.lens + gone if "moved" in form else None, rope_rows=most)


def test_prologue_q_alone_kv_alone_and_without_masses(ctx):
    c = Case(ctx, [20, 9], [3, 9], 8, 2, 128, 16, 21).up()
    q, k, v, qw, kw = projections(c, 22)
    prologue(c, q=q, qw=qw)
    check_pools(c)
    prologue(c, k=k, v=v, kw=kw, with_mass=False)
    prologue(c, k=k, v=v, kw=kw)


def test_zero_rows_small_rows_and_the_border_of_a_scale(ctx):
    """Rows of zeros and rows that the norm leaves small (its eps) have the least scale; 7 belongs to a scale of 1."""
    c = Case(ctx, [48], [48], 1, 1, 64, 16, 41).up()
    k, v = np.zeros((1, 48, 1, 64), np.float32), np.zeros((1, 48, 1, 64), np.float32)
    v[0, 16:32, 0, 5] = 3.0   # one element: the norm makes it nearly 8, above 7: a scale of 2, a code of 4
    v[0, 32:, 0, :] = 2.0 ** -14  # 2^-14 / sqrt(2^-28 + 1e-6), 0.061
    v[0, 40:, 0, :] = 2.0 ** -36  # 2^-26 after the norm: below half of the least step
    ctx.pagedAttnPrologue4(None, ctx.from_numpy(k), ctx.from_numpy(v), 1, None, ctx.from_numpy(np.ones(64, np.float16)),
                           None, None, *c.cache, c.dt, c.dl, c.p, row_starts=c.ds)
    ks = c.dks.download(np.uint8).reshape(c.k.scale.shape)[c.table[0]]
    vs = K4.by_row(c.dvs.download(np.uint8).reshape(c.v.by_tile().shape))[c.table[0]]
    codes = K4.unpack(c.dv.download(np.uint8).reshape(c.v.packed().shape))[c.table[0]]
    assert np.all(ks == 107) and np.all(vs[0] == 107) and np.all(vs[2, 8:] == 107)
    assert np.all(vs[1] == [128, 107]) and np.all(codes[1, :, 0, 5] == 6) and np.count_nonzero(codes[1]) == 16
    assert np.all(codes[2, 8:] == 0) and np.all(vs[2, :8] == 121) and np.all(codes[2, :8] == 6)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_non_finite_rows_mark_themselves_and_their_head(ctx, bad, hd):
    c = Case(ctx, [24, 20], [1, 1], 4, 2, hd, 16, 51, max_len=64).up()
    for step in (0, 1):
        c.lens += 1
        c.dl.upload(c.lens.astype(np.uint32))
        q, k, v, qw, kw = projections(c, 52 + step)
        if step == 0:
            k[0, 0, 1, 7] = bad
            v[0, 1, 0, hd - 2] = bad
        prologue(c, q, k, v, None, qw, kw)
    assert (c.k.scale == 255).sum() == (c.v.scale == 255).sum() == hd // 32
    got = c.attention(mass=True)
    assert np.all(np.isnan(got[0, 2:])) and np.all(np.isfinite(got[0, :2]))
    assert np.all(np.isnan(got[1, :2])) and np.all(np.isfinite(got[1, 2:]))
    # the row written again is a row like any other
    c.lens -= 1
    c.dl.upload(c.lens.astype(np.uint32))
    c.mass = c.dm.download(np.float32).reshape(c.mass.shape)
    q, k, v, qw, kw = projections(c, 55)
    prologue(c, q, k, v, None, qw, kw)
    c.check_attention(c.attention())


def test_lengths_starts_positions_and_pages_that_do_not_hold(ctx):
    """A sequence shorter than its rows, one longer than max_seq_len, one of length 0, bad page ids; positions below a
    sequence's rows or past the table; starts that descend, pass num_rows or hold more than max_rows rows."""
    c = Case(ctx, [2, 99, 0, 20, 20, 30], [3, 1, 1, 2, 1, 3], 8, 1, 256, 16, 61, extra_rows=3, max_len=48)
    c.table[3, 1] = c.pages + 5
    c.table[4, 1] = -7
    c.up()
    q, k, v, qw, kw = projections(c, 62)
    prologue(c, q, k, v, None, qw, kw)
    table = table_of(ctx, 256, 60)[0]
    prologue(c, q, k, v, table, qw, kw, positions=[9, 9, 9, 1, 60, 61], rope_rows=60)
    prologue(c, q, k, v, None, qw, kw, positions=[9, 9, 9, 1, 60, 2], rope_rows=60)
    got = c.attention(mass=True)
    n = c.starts
    assert np.all(got[n[0]:n[3]] == 0)  # nothing to see
    c.check_attention(got, range(int(n[3]), int(n[6])))
    before, c.mass = c.mass, c.dm.download(np.float32).reshape(c.mass.shape)
    assert np.all(np.isfinite(c.mass)) and np.count_nonzero(before != c.mass) >= 60
    # starts: sequence 1 descends, sequence 3 passes num_rows, sequence 5 holds too many
    c.ds.upload(np.array([0, 3, 2, 4, 400, 5, 11], np.uint32))
    c.dl.upload(np.full(6, 40, np.uint32))
    out = ctx.from_numpy(np.full(q.shape[1:], 7.5, np.float32))
    pools = [d.download(np.uint8) for d in c.cache]
    ws = ctx.alloc(ctx.attn4_workspace_bytes(c.p, True))
    ctx.pagedAttn4(ctx.from_numpy(c.q), *c.cache, c.dt, c.dl, out, c.p, ws, row_starts=c.ds)
    assert np.all(out.download(np.float32).reshape(q.shape[1:])[5:] == 7.5)
    dq = ctx.from_numpy(np.full(q.shape[1:], 3.25, np.float32))
    ctx.pagedAttnPrologue4(ctx.from_numpy(q), ctx.from_numpy(k), ctx.from_numpy(v), 1, ctx.from_numpy(qw),
                           ctx.from_numpy(kw), None, dq, *c.cache, c.dt, c.dl, c.p, row_starts=c.ds)
    assert np.all(dq.download(np.float32).reshape(q.shape[1:])[5:] == 3.25)
    for s in (3, 4, 5):  # nothing appended for them
        pages = c.table[s][(c.table[s] >= 0) & (c.table[s] < c.pages)]
        for a, d in zip(pools, c.cache):
            assert np.array_equal(a.reshape(c.pages, -1)[pages], d.download(np.uint8).reshape(c.pages, -1)[pages])


@pytest.mark.parametrize("hd,nkh,ps", [(64, 3, 16), (128, 1, 32), (256, 1, 48), (512, 2, 16)])
def test_values(ctx, hd, nkh, ps):
    c = Case(ctx, [5 * ps], [1], nkh, nkh, hd, ps, 71)
    c.k.scale[1, 3], c.v.scale[0, 2] = 255, 255
    c.k.scale[2] = c.rng.integers(100, 141, c.k.scale[2].shape)
    c.up()
    pages = np.array([3, 0, 3, -1, c.pages, 5, 1, 2], np.int32)
    n = ps * nkh * hd
    k, v = ctx.empty(len(pages) * n, np.uint16), ctx.empty(len(pages) * n, np.uint16)
    ctx.kv4Values(*c.cache, ctx.from_numpy(pages), len(pages), ps, nkh, hd, c.pages, k, v)
    for pool, out in ((c.k, k), (c.v, v)):
        got = out.download(np.uint16).view(np.float16).reshape(len(pages), ps, nkh, hd)
        with np.errstate(over="ignore"):
            want = pool.values().astype(np.float16)
        for i, pg in enumerate(pages):
            assert np.array_equal(got[i], want[pg] if 0 <= pg < c.pages else np.zeros_like(got[i]), equal_nan=True)


ATTN = [  # lens, rows, query heads, K/V heads, dim, page size, window
    ([1], [1], 8, 1, 256, 16, 0),
    ([600], [1], 8, 1, 256, 16, 512),
    ([1, 2, 15, 16, 17, 31, 127, 128, 129, 700], [1] * 10, 8, 1, 256, 16, 0),
    ([33, 250, 1030], [1] * 3, 8, 1, 512, 16, 0),
    ([1500, 64, 65], [1] * 3, 8, 1, 512, 32, 100),
    ([900, 3, 260], [1] * 3, 8, 2, 128, 32, 300),
    ([900, 3, 260], [1] * 3, 4, 4, 64, 64, 0),
    ([333, 77], [1] * 2, 16, 1, 128, 48, 0),
    ([333, 77], [1] * 2, 48, 3, 256, 16, 64),
    ([12, 400, 5], [4, 2, 3], 8, 2, 128, 32, 128),
    ([12, 400, 5, 9], [4, 2, 3, 0], 8, 1, 256, 16, 0),
    ([100], [100], 8, 1, 256, 16, 0),
    ([100], [100], 8, 1, 512, 16, 0),
    ([260], [130], 8, 1, 512, 16, 33),
    ([300, 20, 170], [60, 20, 1], 8, 1, 256, 16, 40),
    ([300, 20, 170], [60, 20, 1], 8, 2, 128, 32, 0),
    ([150, 90], [150, 33], 6, 2, 64, 16, 0),
    ([150, 90], [150, 33], 5, 1, 256, 80, 70),
    ([150, 90], [40, 33], 16, 1, 512, 16, 0),
]


@pytest.mark.parametrize("mass", [False, True])
@pytest.mark.parametrize("lens,rows,nqh,nkh,hd,ps,window", ATTN)
def test_attention(ctx, lens, rows, nqh, nkh, hd, ps, window, mass):
    c = Case(ctx, lens, rows, nqh, nkh, hd, ps, 81, window=window, scale=0.8,
             extra_rows=0 if set(rows) == {1} else 2).up()
    got = c.attention(mass=mass)
    total = int(c.n.sum())
    rows = range(total) if total < 60 else sorted({*range(0, total, 7), total - 1, total - 2})
    c.check_attention(got, rows)
    if mass:
        c.check_mass(c.mass)
        first = c.dm.download(np.uint32)
        c.dm.upload(c.mass)
    assert np.array_equal(c.attention(mass=mass).view(np.uint32), got.view(np.uint32))  # the sums' order is fixed
    if mass:
        assert np.array_equal(c.dm.download(np.uint32), first)


FULL = [  # lens, rows, query heads, K/V heads: 9 to 16 columns of a K/V head, the few-rows kernel's most
    ([300, 33], [2, 2], 8, 1),
    ([700], [1], 16, 1),
    ([41, 260, 7], [1, 1, 1], 9, 1),
    ([150, 90], [4, 3], 8, 2),
    ([500, 9, 64], [4, 1, 3], 4, 1),
]


@pytest.mark.parametrize("mass", [False, True])
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("lens,rows,nqh,nkh", FULL)
def test_attention_of_nine_to_sixteen_columns(ctx, lens, rows, nqh, nkh, hd, mass):
    """Drafts to verify, many query heads to a K/V head: every column's output, operand blocks and weights."""
    c = Case(ctx, lens, rows, nqh, nkh, hd, 16, 85, window=0 if nqh != 9 else 100, scale=0.8).up()
    assert 8 < max(rows) * nqh // nkh <= 16
    got = c.attention(mass=mass)
    c.check_attention(got)
    if mass:
        c.check_mass(c.mass)
        c.dm.upload(c.mass)
    if hd >= 256 and nqh * hd % 256 == 0:
        ops = ctx.zeros(ctx.batch_operand_bytes(nqh * hd, c.p.num_rows), np.uint8)
        assert np.array_equal(c.attention(mass=mass, ops=ops).view(np.uint32), got.view(np.uint32))
        b = ops.download(np.uint8).reshape(nqh * hd // 256, -1)  # one tile of 16 rows: hi + lo, sums, 2^-e
        m = b[:, :16384].reshape(-1, 8, 2, 4, 16, 16).copy().view(np.float16).astype(np.float64).sum(2)
        m = m.transpose(3, 0, 1, 2, 4).reshape(16, -1, 256) * b[:, -64:].copy().view(np.float32).T[..., None]
        want = got.reshape(len(got), -1, 256)
        assert (np.abs(m[:len(got)] - want) <= 2.0 ** -22 * np.abs(want).max(-1, keepdims=True)).all()


@pytest.mark.parametrize("nkh,ragged", [(1, False), (3, True)])
def test_attention_of_many_sequences(ctx, nkh, ragged):
    """More sequences than a wave has lanes, some without positions or rows; shares that end inside one."""
    rng = np.random.default_rng(7)
    lens, rows = rng.integers(0, 400, 300), np.ones(300, int)
    lens[60:200] = 0
    if ragged:
        rows = rng.integers(0, 3, 300)
    c = Case(ctx, lens, rows, 4 * nkh, nkh, 128, 32, 86, extra_rows=int(ragged)).up()
    got = c.attention(mass=True)
    total = int(c.n.sum())
    c.check_attention(got, range(0, total, 3))
    for r in range(total):
        assert np.any(got[r] != 0) == (c.row(r)[1] >= 0), r
    c.n = np.where(c.lens < c.n, 0, c.n)
    more = c.dm.download(np.float32).sum(dtype=np.float64) - c.mass.sum(dtype=np.float64)
    seen = sum(c.row(r)[1] >= 0 and c.n[c.row(r)[0]] > 0 for r in range(total))
    assert abs(more - 4 * nkh * seen) <= 1e-4 * seen  # every row and head gives one


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("hd,nkh", [(64, 2), (128, 1), (256, 1), (512, 1)])
def test_attention_of_a_long_cache(ctx, rows, hd, nkh):
    c = Case(ctx, [13011, 150], [rows, min(rows, 2)], 8 * nkh, nkh, hd, 48, 91).up()
    got = c.attention(mass=rows == 1)
    total = int(c.n.sum())
    c.check_attention(got, sorted({0, rows // 2, rows - 1, total - 1}))
    if rows == 1:
        c.check_mass(c.mass)


@pytest.mark.parametrize("rows", [1, 20])
def test_attention_masks_and_extremes(ctx, rows):
    """Pages outside the window or behind the length may hold anything: NaN scales there stay there. A dominant key
    whose values are 0 leaves the others their share; scales far apart meet in one row."""
    c = Case(ctx, [300, 300], [rows, rows], 8, 1, 256, 16, 101, window=100, max_len=400)
    far = [c.table[s, j] for s in (0, 1) for j in range((300 - rows - 100) // 16)]
    for pool in (c.k, c.v):
        pool.scale[far] = 255
        pool.scale[-2:] = 255
        for s in (0, 1):
            pool.scale[c.table[s, 18], 12:] = 255  # behind position 299
    c.mass[far] = np.nan
    for s in (0, 1):
        c.table[s, 19:] = c.pages - 1
    # sequence 1: V scales from 2^-20 to 2^13, K's from 2^-40 to 2^4
    c.v.scale[c.table[1, 11:18]] = c.rng.choice([107, 117, 127, 140], c.v.scale[c.table[1, 11:18]].shape)
    c.k.scale[c.table[1, 11:18]] = c.rng.choice([87, 107, 125, 131], c.k.scale[c.table[1, 11:18]].shape)
    # sequence 0: position 290 - rows is far above the rest, its values zero
    pg, slot = c.table[0, (290 - rows) // 16], (290 - rows) % 16
    c.v.codes[pg, slot] = 0
    d = c.rng.choice([-1.0, 1.0], 256).astype(np.float32)
    c.q[:rows] = c.q[:rows] * np.float32(0.01) + np.float32(0.02) * d
    c.k.scale[c.table[0, 11:19]] -= np.uint8(4) * (c.k.scale[c.table[0, 11:19]] < 255)
    c.k.codes[pg, slot, 0] = np.where(d > 0, 6, 14)
    c.k.scale[pg, slot] = 127
    c.up()
    got = c.attention(mass=True)
    c.check_attention(got)
    c.check_mass(c.mass)


@pytest.mark.parametrize("hd,rows,window", [(256, 2, 0), (256, 2, 20), (512, 2, 0), (128, 70, 0), (256, 40, 30),
                                            (512, 40, 0), (64, 300, 0)])
def test_a_row_that_is_not_finite_stays_with_the_rows_that_see_it(ctx, hd, rows, window):
    """The rows before it do not see it, though their step of positions holds it."""
    c = Case(ctx, [101 if rows == 2 else 80 + rows], [rows], 8, 1, hd, 16, 111, window=window).up()
    bad = 100
    pg, slot = c.table[0, bad // 16], bad % 16
    ks, vs = c.k.scale.copy(), c.v.scale.copy()
    pos = c.lens[0] - rows + np.arange(rows)
    sees = (pos >= bad) & ((window == 0) | (pos - window < bad))
    assert 0 < sees.sum() < rows
    for k, v in ((True, False), (False, True), (True, True)):
        for pool, scale, dev, put, on in ((c.k, ks, c.dks, lambda: c.k.scale, k), (c.v, vs, c.dvs, c.v.by_tile, v)):
            pool.scale[:] = scale
            if on:
                pool.scale[pg, slot] = 255
            dev.upload(put())
        c.dm.upload(c.mass)
        got = c.attention(mass=True)
        assert np.isnan(got[sees]).all(), (k, v)
        c.check_attention(got, np.flatnonzero(~sees), what=(k, v))


@pytest.mark.parametrize("hd,rows", [(256, 1), (512, 1), (64, 90), (128, 90), (256, 90), (512, 90)])
def test_scales_and_q_of_nothing(ctx, hd, rows):
    """Rows of zeros as the append leaves them (2^-20) or slots never written (0 bytes), next to rows that hold
    something; q so small that every score is 0 in f32, q of zeros, q of very different blocks."""
    for what in ("least", "never written", "all never written", "small q", "q of zeros", "blocks"):
        c = Case(ctx, [150], [rows], 8, 1, hd, 16, 121, scale=0.7)
        for pool in (c.k, c.v):
            if what == "least":
                pool.scale[c.table[0, 2:10]] = 107
                pool.codes[c.table[0, 2:10]] = 0
            if "never" in what:
                at = c.table[0, 2 if what[0] == "n" else 0:]
                pool.scale[at], pool.codes[at] = 0, 0
        if what == "blocks":
            c.q *= np.repeat(2.0 ** c.rng.integers(-30, 1, (*c.q.shape[:-1], hd // 32)), 32, -1).astype(np.float32)
        c.q *= np.float32(1e-33 if "small" in what else 0.0 if "zeros" in what else 1.0)
        c.up()
        got = c.attention(mass=True)
        c.check_attention(got, sorted({0, 5, 63, 64, rows - 1} & set(range(rows))), what=what)
        c.check_mass(c.mass, what)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("hd,rows", [(64, 1), (256, 1), (512, 1), (128, 40), (256, 40), (512, 40)])
def test_a_query_that_is_not_finite_is_alone_with_it(ctx, hd, rows, bad):
    c = Case(ctx, [90, 33], [rows, 1], 8, 1, hd, 16, 125, extra_rows=1).up()
    c.q[0, 3, hd - 1] = bad
    got = c.attention()
    assert np.isnan(got[0, 3]).all() and np.isfinite(got[0, [0, 1, 2, 4, 5, 6, 7]]).all()
    c.check_attention(got, range(1, rows + 1))


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("window,bad", [(0, "q"), (25, "q"), (25, "k"), (25, "v")])
def test_weights_of_a_row_that_is_not_finite_stay_with_what_it_sees(ctx, hd, rows, window, bad):
    """One query, or a key or value that the last row alone sees: the rows that the NaN ones do not see (behind them, out of
    their window) get what the others give them."""
    c = Case(ctx, [101], [rows], 8, 1, hd, 16, 127, window=window)
    if bad == "q":
        c.q[0, 3, 5] = np.nan
    else:
        pool = c.k if bad == "k" else c.v
        pool.scale[c.table[0, 100 // 16], 100 % 16] = 255
    c.up()
    c.attention(mass=True)
    got = c.dm.download(np.float32).reshape(c.mass.shape)
    more, tol = np.zeros(c.mass.shape), np.zeros(c.mass.shape)
    nan = np.zeros(c.mass.shape, bool)
    k, v = c.k.values(), c.v.values()
    for r in range(rows):
        pos = 101 - rows + r
        t = np.arange(max(0, pos + 1 - window) if window else 0, pos + 1)
        at = (c.table[0, t // 16], t % 16, 0)
        if r == 0 and bad == "q" or r == rows - 1 and bad != "q":
            nan[at] = True
            if bad != "q":
                continue
        _, _, reach, p = K4.attend(c.q[r], k, v, c.table[0], pos, window, 1.0)
        for h in range(8):
            if np.isfinite(p[h]).all():
                more[at] += p[h]
                tol[at] += p[h] * slack(hd, pos + 1, reach[h, 0]) + 2.0 ** -126
    assert 0 < nan.sum() and np.any(~nan & (more > 0))
    assert np.array_equal(np.isnan(got), nan)
    tol += (rows * 8 + 2) * U * more
    want = c.mass + more
    assert (np.abs(got - want)[~nan] <= (tol + U * want + 1e-38)[~nan]).all()
    assert np.array_equal(got[(more == 0) & ~nan], c.mass[(more == 0) & ~nan])


@pytest.mark.parametrize("scale", [-0.9, 0.0, 1e-30])
@pytest.mark.parametrize("hd,rows,window", [(256, 1, 0), (512, 1, 40), (64, 50, 0), (256, 50, 60), (512, 50, 0)])
def test_scale_of_any_sign(ctx, hd, rows, window, scale):
    c = Case(ctx, [170, 60], [rows, rows], 8, 1, hd, 32, 131, window=window, scale=scale).up()
    got = c.attention(mass=True)
    c.check_attention(got, sorted({0, 7, 8, rows - 1, rows, 2 * rows - 1} & set(range(2 * rows))))
    c.check_mass(c.mass)


@pytest.mark.parametrize("hd,most,sequences", [(128, 9, 700), (256, 40, 300), (512, 17, 200)])
def test_many_rows_of_many_sequences(ctx, hd, most, sequences):
    """More column tiles than a workgroup has threads; sequences without rows, without positions, of one row."""
    rng = np.random.default_rng(141)
    lens, rows = rng.integers(0, 90, sequences), rng.integers(0, most + 1, sequences)
    rows = np.minimum(rows, rng.choice([0, 1, most], sequences))
    rows[3] = most
    lens = np.where(rng.random(sequences) < 0.1, 0, np.maximum(lens, rows))
    lens[100:140] = 0  # a run of nothing
    lens[-2:] = 0
    c = Case(ctx, lens, rows, 8, 1, hd, 16, 142, extra_rows=1).up()
    got = c.attention(mass=True)
    total = int(c.n.sum())
    short = [r for r in range(total) if c.lens[c.row(r)[0]] < c.n[c.row(r)[0]]]
    assert short and np.all(got[short] == 0)
    c.check_attention(got, sorted((set(range(0, total, 11)) | {total - 1}) - set(short)))
    more = c.dm.download(np.float32).sum(dtype=np.float64) - c.mass.sum(dtype=np.float64)
    assert abs(more - 8 * (total - len(short))) <= 1e-4 * total


def test_two_graphs_share_a_workspace(ctx):
    """Prompts and steps captured apart into graphs over one workspace, replayed in turn with eager calls between."""
    a = Case(ctx, [300], [120], 8, 1, 256, 16, 151).up()
    b = Case(ctx, [700, 40], [1, 1], 8, 1, 512, 16, 152).up()
    bytes_ = max(ctx.attn4_workspace_bytes(c.p, True) for c in (a, b))
    ws = ctx.from_numpy(np.full(bytes_, 0xff, np.uint8))
    want = []
    for c in (a, b):
        want.append((c.attention(mass=True), c.dm.download(np.uint32)))
        c.dm.upload(c.mass)
    runs = []
    for c in (a, b):
        q, out = ctx.from_numpy(c.q), ctx.from_numpy(np.full(c.q.shape, 7.5, np.float32))
        ctx.graph_begin()
        ctx.pagedAttn4(q, *c.cache, c.dt, c.dl, out, c.p, ws, row_starts=c.ds, mass=c.dm)
        runs.append((ctx.graph_end(), q, out, c))
    for _ in range(4):
        for i in (0, 1, 1, 0):
            g, _, out, c = runs[i]
            out.upload(np.full(c.q.shape, 7.5, np.float32))
            c.dm.upload(c.mass)
            ctx.graph_launch(g)
            got = out.download(np.float32).reshape(c.q.shape)
            assert np.array_equal(got.view(np.uint32), want[i][0].view(np.uint32))
            assert np.array_equal(c.dm.download(np.uint32), want[i][1])
            eager = runs[1 - i][3]
            assert np.array_equal(eager.attention(ws).view(np.uint32), want[1 - i][0].view(np.uint32))
    for g, *_ in runs:
        ctx.graph_destroy(g)


@pytest.mark.parametrize("far", [2.0 ** -12, 2.0 ** -26, 2.0 ** -36])
@pytest.mark.parametrize("hd,rows", [(256, 1), (512, 1), (64, 20), (256, 20), (512, 20)])
def test_a_weight_far_below_the_largest_keeps_its_share(ctx, hd, rows, far):
    """One key holds all the weight, its values are 0; another's weight is `far` of it, in the same half of 64
    positions or in the other."""
    for a, b in ((3, 10), (3, 40), (40, 3), (70, 3)):
        c = Case(ctx, [100], [rows], 8, 1, hd, 16, 161)
        for pos in range(100):
            pg, slot = c.table[0, pos // 16], pos % 16
            c.k.codes[pg, slot], c.k.scale[pg, slot] = 0, 127
            c.k.codes[pg, slot, 0, 0] = {a: 7, b: 6}.get(pos, 15)  # 6, 4, -6
            c.v.codes[pg, slot] *= np.uint8(pos != a)
        c.q[:] = 0
        c.q[..., 0] = -np.log(far) / 2
        c.up()
        got = c.attention(mass=True)
        c.check_attention(got, what=(a, b))
        c.check_mass(c.mass, (a, b))


@pytest.mark.parametrize("far", [1.37 * 2.0 ** -20, 1.37 * 2.0 ** -28, 1.37 * 2.0 ** -36, 2.0 ** -60, 1.37 * 2.0 ** -100])
@pytest.mark.parametrize("hd,rows", [(64, 1), (128, 1), (256, 1), (512, 1), (64, 20), (128, 20), (256, 20), (512, 20)])
def test_a_small_weight_is_as_exact_as_a_large_one(ctx, hd, rows, far):
    """As above, but held to the errors of a weight relative to itself: P's size costs it no bits (f32 in three parts of 8
    bits with its exponent), down to what f32 can hold. An output of zeros is off by 1e3 tolerances and more."""
    for n, a, b in ((100, 3, 10), (100, 3, 40), (100, 40, 3), (100, 70, 3), (700, 5, 600), (700, 600, 5)):
        c = Case(ctx, [n], [rows], 8, 1, hd, 16, 163)
        pos = np.arange(n)
        pg, slot = c.table[0, pos // 16], pos % 16
        c.k.codes[pg, slot], c.k.scale[pg, slot] = 0, 127
        c.k.codes[pg, slot, 0, 0] = np.where(pos == a, 7, np.where(pos == b, 6, 15))  # 6, 4, -6
        c.v.codes[pg[a], slot[a]] = 0
        c.q[:] = 0
        c.q[..., 0] = -np.log(far) / 2
        c.up()
        got = c.attention()
        k, v = c.k.values(), c.v.values()
        for r in (0, rows - 1):
            want, mag, reach, _ = K4.attend(c.q[r], k, v, c.table[0], n - rows + r, 0, 1.0)
            tol = slack(hd, n, reach) * mag + 1e-38
            held = mag > far / 32  # (where position b's value is not 0)
            assert held.any() and bool((np.abs(want[held]) >= 1e3 * tol[held]).all())
            off = (np.abs(got[r] - want) / tol).max()
            assert off <= 1, (n, a, b, r, off)


@pytest.mark.parametrize("hd,rows", [(64, 1), (128, 1), (256, 1), (512, 1), (64, 20), (128, 20), (256, 20), (512, 20)])
def test_values_of_any_scale(ctx, hd, rows):
    """V's scales from 2^-60 to 2^60, each block's by itself: what the append writes is a small part of them."""
    c = Case(ctx, [150, 40], [rows, rows], 8, 1, hd, 16, 164)
    c.v.scale[:] = c.rng.choice([67, 100, 127, 141, 187], c.v.scale.shape)
    c.up()
    got = c.attention()
    k, v = c.k.values(), c.v.values()
    for r in sorted({0, rows - 1, rows, 2 * rows - 1}):
        s, pos = c.row(r)
        want, mag, reach, _ = K4.attend(c.q[r], k, v, c.table[s], pos, 0, 1.0)
        off = (np.abs(got[r] - want) / (slack(hd, pos + 1, reach) * mag)).max()
        assert off <= 1, (r, off)


@pytest.mark.parametrize("hd,nkh,rows,lens", [(256, 1, [1] * 5, [1, 40, 0, 300, 700]), (512, 1, [1] * 3, [9, 1000, 33]),
                                              (256, 2, [1] * 20, [50 * s for s in range(20)]),
                                              (512, 1, [1] * 40, [30 * s + 1 for s in range(40)]),
                                              (256, 3, [2, 0, 1, 2], [90, 5, 1, 400])])
def test_the_output_as_operand_blocks(ctx, hd, nkh, rows, lens):
    """Per super-block and row: f16 hi + lo of y 2^e (22 bits of the block's largest), the sub-blocks' sums in three
    f16 parts (33 bits, of 32 terms added in f32), and 2^-e; the blocks of the padding are not written."""
    c = Case(ctx, lens, rows, 8 * nkh, nkh, hd, 16, 171).up()
    R = c.p.num_rows
    assert R == c.n.sum()
    nblk, ntv = 8 * nkh * hd // 256, 1 if R <= 16 else 2 if R <= 32 else 4
    size = ctx.batch_operand_bytes(8 * nkh * hd, R)
    for mass in (False, True):
        ops = ctx.from_numpy(np.full(size, 0x5a, np.uint8))
        y = c.attention(ops=ops, mass=mass)
        assert np.array_equal(y.view(np.uint32), c.attention().view(np.uint32))
        b = ops.download(np.uint8).reshape(nblk, -1)
        main, sums = ntv * 8 * 2 * 1024, ntv * 1024
        assert b.shape[1] == main + sums + 64 * ntv
        m = b[:, :main].reshape(nblk, ntv, 8, 2, 4, 16, 16).copy().view(np.float16).astype(np.float64)
        m = m.transpose(3, 0, 1, 5, 2, 4, 6).reshape(2, nblk, 16 * ntv, 256)  # [hi, lo][block][row][32 s + 8 q + j]
        sc = b[:, main + sums:].copy().view(np.float32).reshape(nblk, 16 * ntv).astype(np.float64)
        p = b[:, main:main + sums].reshape(nblk, ntv, 4, 16, 16).copy().view(np.float16).astype(np.float64)
        p = p.reshape(nblk, ntv, 4, 16, 2, 4).transpose(0, 1, 3, 2, 4, 5).reshape(nblk, 16 * ntv, 8, 4)
        want = y.reshape(R, nblk, 256).transpose(1, 0, 2).astype(np.float64)
        top = np.abs(want).max(-1, keepdims=True)
        assert (np.abs((m[0] + m[1])[:, :R] * sc[:, :R, None] - want) <= 2.0 ** -22 * top).all()
        sub = (want / sc[:, :R, None]).reshape(nblk, R, 8, 32)
        tol = 32 * U * np.abs(sub).sum(-1) + 2.0 ** -24 * 64
        assert (np.abs(p[:, :R].sum(-1) * 64 - sub.sum(-1)) <= tol).all() and np.all(p[:, :R, :, 3] == 0)
        raw = b[:, :main].reshape(nblk, ntv, 8, 2, 4, 16, 16).transpose(0, 1, 5, 2, 3, 4, 6).reshape(nblk, 16 * ntv, -1)
        assert np.all(raw[:, R:] == 0x5a)


@pytest.mark.parametrize("change", [dict(hd=128), dict(num_seqs=65), dict(num_rows=6, max_rows=3), dict(ops=8)])
def test_operand_blocks_that_are_refused(ctx, change):
    b, ws = ctx.zeros(1 << 20, np.uint8), ctx.zeros(1 << 24, np.uint8)
    ops = b.offset(change.get("ops", 0))
    p = ctx.kv4_params(**{**dict(num_seqs=2, nqh=8, nkh=1, hd=256, page_size=16, max_pages=4, max_seq_len=64,
                                 num_pages=9), **{k: v for k, v in change.items() if k != "ops"}})
    with pytest.raises(g4hip.G4Error):
        ctx.pagedAttn4(b, b, b, b, b, b, b, b, p, ws, row_starts=b if p.num_rows != p.num_seqs else None, ops=ops)


def test_attention_of_far_pages(ctx):
    """Pools of more than 4 GiB: page offsets past 32 bits."""
    hd, ps, pages = 512, 16, (1 << 32) // (16 * 256) + 40
    c = Case(ctx, [100, 70], [1, 1], 8, 1, hd, ps, 111)
    small, shift = c.pages, pages - c.pages
    row = ps * hd // 2
    pools = [ctx.alloc(pages * row) for _ in range(2)]
    scales = [ctx.alloc(pages * ps * hd // 32) for _ in range(2)]
    mass = ctx.alloc(4 * pages * ps)
    for d, x in zip(pools, (c.k.packed(), c.v.packed())):
        d.offset(shift * row).upload(x)
    for d, x in zip(scales, (c.k.scale, c.v.by_tile())):
        d.offset(shift * ps * hd // 32).upload(x)
    mass.offset(4 * shift * ps).upload(c.mass)
    c.up()
    host = c.table.copy()
    c.dt.upload(np.where(host >= 0, host + shift, -1).astype(np.int32))
    c.p.num_pages = pages
    c.cache, c.dm = (*pools, *scales), mass

    def check(pool, d, scale, ds, rows):
        got = d.download(np.uint8, small * row, offset=shift * row).reshape(pool.packed().shape)
        assert np.array_equal(got, pool.packed())
        n = small * ps * hd // 32
        assert np.array_equal(ds.download(np.uint8, n, offset=shift * ps * hd // 32).reshape(scale.shape), scale)

    got = c.attention(mass=True)
    c.check_attention(got)
    back, c.dm = c.dm, ctx.from_numpy(mass.download(np.float32, small * ps, offset=4 * shift * ps))
    c.check_mass(c.mass)
    c.dm = back
    c.mass = mass.download(np.float32, small * ps, offset=4 * shift * ps).reshape(c.mass.shape)
    q, k, v, qw, kw = projections(c, 112)
    ctx.pagedAttnPrologue4(None, ctx.from_numpy(k), ctx.from_numpy(v), 1, None, ctx.from_numpy(kw), None, None,
                           *c.cache, c.dt, c.dl, c.p, mass=mass)
    cs = table_of(ctx, hd, 100)[1]
    for s, L in enumerate(c.lens):
        c.k.append(K8.rotated(K8.normed(k[0, s:s + 1], kw), cs[L - 1:L]), host[s], int(L) - 1)
        c.v.append(K8.normed(v[0, s:s + 1]), host[s], int(L) - 1)
        c.mass[host[s, (L - 1) // ps], (L - 1) % ps] = 0
    assert min(c.k.border, c.v.border) > 1e-9
    check(c.k, pools[0], c.k.scale, scales[0], lambda x: x)
    check(c.v, pools[1], c.v.by_tile(), scales[1], K4.by_row)
    pages_dev = ctx.from_numpy((host[:, 0] + shift).astype(np.int32))
    out = [ctx.empty(2 * ps * hd, np.uint16) for _ in range(2)]
    ctx.kv4Values(*c.cache, pages_dev, 2, ps, 1, hd, pages, *out)
    assert np.array_equal(out[1].download(np.uint16).view(np.float16).reshape(2, ps, 1, hd),
                          c.v.values()[host[:, 0]].astype(np.float16))
    kept = ctx.empty(2 * 60, np.int32)
    ctx.kvEvict4(*c.cache, mass, c.dt, c.dl, c.p, 60, 3, 20, kept, ctx.alloc(ctx.evict4_workspace_bytes(c.p, 60)))
    want, lens = K4.evict(c.k, c.v, c.mass, host, c.lens, 60, 3, 20, 100)
    assert np.array_equal(kept.download(np.int32).reshape(want.shape), want)
    check(c.k, pools[0], c.k.scale, scales[0], lambda x: x)
    check(c.v, pools[1], c.v.by_tile(), scales[1], K4.by_row)
    assert np.array_equal(mass.download(np.float32, small * ps, offset=4 * shift * ps).reshape(c.mass.shape), c.mass)


@pytest.mark.parametrize("hd,ps", [(64, 256), (128, 1024), (256, 512), (512, 256), (512, 1024)])
def test_large_pages(ctx, hd, ps):
    c = Case(ctx, [ps + 700, 300, 2 * ps + 1], [ps + 333, 1, 2], 4, 2, hd, ps, 191, parts=2).up()
    q, k, v, qw, kw = projections(c, 192)
    got = prologue(c, q, k, v, table_of(ctx, hd, c.p.max_seq_len)[0], qw, kw)
    c.q = got * np.float32(0.1)
    total = int(c.n.sum())
    c.check_attention(c.attention(), sorted({0, 63, 64, ps - 1, total - 4, total - 3, total - 2, total - 1}))


def test_steps_beside_a_prompt(ctx):
    rng = np.random.default_rng(211)
    lens, rows = rng.integers(1, 900, 65), np.ones(65, int)
    lens[20], rows[20] = 420, 300
    c = Case(ctx, lens, rows, 8, 1, 256, 16, 212, window=512).up()
    got = c.attention(mass=True)
    total = int(c.n.sum())
    c.check_attention(got, sorted({*range(0, 20), *range(20, 320, 29), 319, *range(320, total)}))
    c.check_mass(c.mass)


@pytest.mark.parametrize("up", [120, 0, -96])
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("rows", [1, 7])
def test_queries_of_any_size(ctx, hd, rows, up):
    """q's blocks of 32 dims have exponents of their own: large or small ones under the inverse scale, and beside each
    other in a row."""
    c = Case(ctx, [90, rows], [rows, rows], 8, 1, hd, 16, 191, scale=2.0 ** -up)
    c.q *= np.float32(2.0 ** up)
    if up <= 0:
        c.q.reshape(-1, 32)[::2] *= np.float32(2.0 ** (-8 if up else -40))
    before = c.mass.copy()
    c.up().check_attention(c.attention(mass=True), what=(hd, rows, up))
    c.check_mass(before, (hd, rows, up))


@pytest.mark.parametrize("hd,theta,divisor", [(64, 1e4, 1), (256, 1e6, 0), (512, 1e6, 1), (128, 5e5, 1)])
def test_prologue_by_theta_and_divisor(ctx, hd, theta, divisor):
    """Angles formed in the launch: the same bits as from a table of its theta and divisors."""
    c = Case(ctx, [61, 300], [9, 40], 8, 2, hd, 32, 181)
    c.p.theta, c.p.apply_divisor = theta, divisor
    freqs = np.random.default_rng(182).choice(np.array([1, 2, 8, 0.5], np.float16), hd // 2)
    n = 400
    t, df = ctx.empty(n * hd, np.float32), ctx.from_numpy(freqs)
    ctx.ropeTable(theta, divisor, df, hd, n, t)
    q, k, v, qw, kw = projections(c, 183)
    for moved in (False, True):
        pos = ctx.from_numpy(np.array([70, 400], np.uint32)) if moved else None
        runs = []
        for table in (None, t):
            c.up()
            out = ctx.from_numpy(np.full(q[0].shape, 3.25, np.float32))
            ctx.pagedAttnPrologue4(*(ctx.from_numpy(x) for x in (q, k, v)), 1, ctx.from_numpy(qw), ctx.from_numpy(kw),
                                   df, out, *c.cache, c.dt, c.dl, c.p, row_starts=c.ds, positions=pos, rope_cs=table,
                                   rope_rows=n if table else 0)
            runs.append([out.download(np.uint32)] + [b.download(np.uint8) for b in c.cache])
        assert all(np.array_equal(a, b) for a, b in zip(*runs))


EVICT = [  # lens, K/V heads, dim, page size, keep, first, recent
    ([50], 1, 256, 16, 40, 0, 0),
    ([50, 41, 40, 39, 0, 200], 1, 64, 16, 40, 4, 10),
    ([300, 77, 120], 3, 128, 48, 77, 0, 77),
    ([300, 77, 120], 2, 512, 32, 76, 76, 0),
    ([2, 3, 1], 2, 256, 16, 1, 0, 0),
    ([2, 3, 1], 2, 256, 16, 1, 1, 0),
    ([2, 3, 1], 2, 64, 16, 1, 0, 1),
    ([5000, 1000], 1, 64, 64, 999, 16, 100),
    ([40000, 33000], 1, 64, 256, 35000, 5, 6000),
    ([70003], 2, 64, 1024, 300, 1, 2),
]


def check_evict(c, keep, first, recent, workspace=None):
    ctx = c.ctx
    kept = ctx.from_numpy(np.full((len(c.lens), c.p.num_kv_heads, keep), 77, np.int32))
    size = ctx.evict4_workspace_bytes(c.p, keep)
    ws = workspace or ctx.from_numpy(np.full(size, 0xff, np.uint8))
    ctx.kvEvict4(*c.cache, c.dm, c.dt, c.dl, c.p, keep, first, recent, kept, ws)
    want, lens = K4.evict(c.k, c.v, c.mass, c.table, c.lens, keep, first, recent, c.p.max_seq_len)
    np.testing.assert_array_equal(kept.download(np.int32).reshape(want.shape), want)
    c.lens = lens
    np.testing.assert_array_equal(c.dl.download(np.uint32), lens)
    c.k.border = c.v.border = np.inf
    check_pools(c)
    return want


@pytest.mark.parametrize("masses", ["of many sizes", "equal", "few values", "zeros and worse"])
@pytest.mark.parametrize("lens,nkh,hd,ps,keep,first,recent", EVICT)
def test_eviction(ctx, lens, nkh, hd, ps, keep, first, recent, masses):
    c = Case(ctx, lens, [1] * len(lens), nkh, nkh, hd, ps, 301)
    m = c.mass
    if masses == "of many sizes":
        m *= 2.0 ** c.rng.integers(-120, 60, m.shape)
    elif masses == "equal":
        m[:] = 0.375
    elif masses == "few values":
        m[:] = c.rng.choice(np.array([0, 1, 1.0000001, 1.5, 256], np.float32), m.shape)
    else:
        m[:] = c.rng.choice(np.array([0, -0.0, -3, np.nan, np.inf, -np.inf, 1e-45, 2e-45, 5], np.float32), m.shape)
    c.up()
    check_evict(c, keep, first, recent)
    check_evict(c, keep, first, recent)  # (nothing is left to cut)


@pytest.mark.parametrize("lens,keep,first,recent", [([33999], 20000, 4, 0), ([60003, 32770], 32000, 0, 3),
                                                    ([98306, 65537, 65800], 400, 1, 0)])
def test_eviction_of_more_candidates_than_fit_in_lds(ctx, lens, keep, first, recent):
    """The last 32768 candidates or fewer in other shares of the waves than those before."""
    c = Case(ctx, lens, [1] * len(lens), 2, 2, 64, 512, 305)
    c.mass *= 2.0 ** c.rng.integers(-20, 20, c.mass.shape)
    c.mass[c.rng.random(c.mass.shape) < 0.2] = 0.25
    check_evict(c.up(), keep, first, recent)


def test_eviction_of_lengths_and_pages_that_do_not_hold(ctx):
    """A sequence past max_seq_len stays; rows of bad page ids count 0, are read clamped and not written."""
    c = Case(ctx, [90, 90, 95, 30], [1] * 4, 2, 2, 128, 16, 311, max_len=96)
    c.table[0, 1], c.table[0, 4] = -3, c.pages + 9
    c.table[1, 5] = c.pages
    c.lens[2] = 97
    c.up()
    kept = check_evict(c, 60, 2, 8)
    assert np.all(kept[2] == -1) and np.all(kept[3, :, 30:] == -1)


def test_eviction_in_graphs_that_share_a_workspace(ctx):
    cases = [Case(ctx, [300, 77, 200], [1] * 3, 2, 2, 128, 16, 321), Case(ctx, [500], [1], 1, 1, 256, 32, 322)]
    ws = ctx.alloc(max(ctx.evict4_workspace_bytes(c.p, 100) for c in cases))
    graphs = []
    for c in cases:
        c.up()
        c.kept = ctx.empty(len(c.lens) * c.p.num_kv_heads * 100, np.int32)
        ctx.graph_begin()
        ctx.kvEvict4(*c.cache, c.dm, c.dt, c.dl, c.p, 100, 4, 20, c.kept, ws)
        graphs.append(ctx.graph_end())
    for turn in range(4):
        for c, g in zip(cases, graphs):
            c.lens = np.array([300, 77, 200][:len(c.lens)] if len(c.lens) > 1 else [500])
            c.dl.upload(c.lens.astype(np.uint32))
            c.mass[:] = np.abs(c.rng.normal(size=c.mass.shape))
            c.dm.upload(c.mass)
            ctx.graph_launch(g)
            want, c.lens = K4.evict(c.k, c.v, c.mass, c.table, c.lens, 100, 4, 20, c.p.max_seq_len)
            assert np.array_equal(c.kept.download(np.int32).reshape(want.shape), want), turn
            assert np.array_equal(c.dl.download(np.uint32), c.lens)
            check_pools(c)
    for g in graphs:
        ctx.graph_destroy(g)


def test_prompt_steps_and_evictions_together(ctx):
    """A prompt appended, attended to and weighed; then decode steps through a captured graph, and every few steps the
    caches are cut to their budget: rows keep their positions' rotation, and every call is held to the oracle."""
    hd, top = 256, 64
    c = Case(ctx, [37, 21], [37, 21], 8, 2, hd, 16, 121, max_len=top, spare=8)
    for s in (0, 1):  # room for the steps
        free = [p for p in range(c.pages) if p not in c.table]
        c.table[s, 2 + (s == 0):4] = free[:2 - (s == 0)]
    c.up()
    q, k, v, qw, kw = projections(c, 122)
    table = table_of(ctx, hd, 200)[0]
    c.q = prologue(c, q, k, v, table, qw, kw, rope_rows=200) * np.float32(0.1)
    got = c.attention(mass=True)
    c.check_attention(got)
    c.check_mass(c.mass)
    c.mass = c.dm.download(np.float32).reshape(c.mass.shape)
    # steps: one row each, read from the same buffers
    c.n[:], c.starts, c.one, c.ds = 1, np.array([0, 1, 2], np.uint32), True, None
    c.p = ctx.kv4_params(2, 8, 2, hd, 16, c.width, top, c.pages)
    bufs = [ctx.empty(2 * n * hd, np.float32) for n in (8, 2, 2)]
    w = [ctx.from_numpy(qw), ctx.from_numpy((kw * np.float16(0.1)).astype(np.float16))]
    qo, out = ctx.empty(2 * 8 * hd, np.float32), ctx.empty(2 * 8 * hd, np.float32)
    ws = ctx.alloc(max(ctx.attn4_workspace_bytes(c.p, True), ctx.evict4_workspace_bytes(c.p, 32)))
    text = c.lens.copy()
    dp = ctx.from_numpy(text.astype(np.uint32))
    graphs = []
    for _ in range(2):
        ctx.graph_begin()
        ctx.advanceSeqLens(c.dl, 2, 1)
        ctx.advanceSeqLens(dp, 2, 1)
        ctx.pagedAttnPrologue4(bufs[0], bufs[1], bufs[2], 1, w[0], w[1], None, qo, *c.cache, c.dt, c.dl, c.p,
                               positions=dp, mass=c.dm, rope_cs=table, rope_rows=200)
        ctx.pagedAttn4(qo, *c.cache, c.dt, c.dl, out, c.p, ws, mass=c.dm)
        graphs.append(ctx.graph_end())
    host_table = table.download(np.float32).reshape(200, hd // 2, 2)
    cuts = 0
    for step in range(70):
        if step % 7 == 0:
            cuts += int((c.lens > 32).sum())
            check_evict(c, 32, 2, 8, ws)
        q, k, v, _, _ = projections(c, 200 + step)
        for b, x in zip(bufs, (q, k, v)):
            b.upload(x)
        ctx.graph_launch(graphs[step % 2])
        c.lens = c.lens + 1
        text += 1
        for s, L in enumerate(c.lens):
            cs = host_table[text[s] - 1:text[s]]
            kn = K8.normed(k[0, s:s + 1], (kw * np.float16(0.1)).astype(np.float16))
            c.k.append(K8.rotated(kn, cs), c.table[s], L - 1)
            c.v.append(K8.normed(v[0, s:s + 1]), c.table[s], L - 1)
            c.mass[c.table[s, (L - 1) // 16], (L - 1) % 16] = 0
        c.q = qo.download(np.float32).reshape(2, 8, hd)
        c.check_attention(out.download(np.float32).reshape(2, 8, hd), what=step)
        c.check_mass(c.mass, step)
        c.mass = c.dm.download(np.float32).reshape(c.mass.shape)
        check_pools(c)
    assert cuts >= 18
    for g in graphs:
        ctx.graph_destroy(g)


def test_refusals(ctx):
    b = ctx.zeros(1 << 16, np.uint8)
    ws = ctx.zeros(1 << 22, np.uint8)
    good = dict(num_seqs=2, nqh=8, nkh=1, hd=256, page_size=16, max_pages=4, max_seq_len=64, num_pages=9)

    def attn(p, q=b, kp=b, wsp=ws, rs=None, mass=None):
        ctx.pagedAttn4(q, kp, b, b, b, b, b, b, p, wsp, row_starts=rs, mass=mass)

    def pro(p, q=b, k=b, v=b, parts=1, rope=None, rows=0, rs=None, qo=b, kw=b, pos=None):
        ctx.pagedAttnPrologue4(q, k, v, parts, b, kw, None, qo, b, b, b, b, b, b, p, row_starts=rs, rope_cs=rope,
                               rope_rows=rows, positions=pos)

    def evict(p, kp=b, mass=b, keep=32, first=0, recent=0, kept=b, wsp=ws):
        ctx.kvEvict4(kp, b, b, b, mass, b, b, p, keep, first, recent, kept, wsp)

    for change in (dict(nqh=7, nkh=2), dict(nqh=17), dict(nqh=65, nkh=65), dict(hd=96), dict(page_size=24),
                   dict(page_size=0), dict(page_size=2048), dict(max_seq_len=65), dict(max_seq_len=0),
                   dict(num_seqs=0), dict(num_rows=3), dict(max_rows=2), dict(num_rows=70000, max_rows=70000),
                   dict(num_pages=0)):
        p = ctx.kv4_params(**{**good, **change})
        for f in (attn, pro):
            with pytest.raises(g4hip.G4Error):
                f(p)
    for change in (dict(nqh=65, nkh=65), dict(hd=96), dict(page_size=24), dict(max_seq_len=65), dict(num_seqs=0),
                   dict(num_pages=0), dict(num_seqs=40000, nqh=2, nkh=2)):
        with pytest.raises(g4hip.G4Error):
            evict(ctx.kv4_params(**{**good, **change}))
    p = ctx.kv4_params(**good)
    for call in (lambda: attn(p, q=None), lambda: attn(p, q=b.offset(4)), lambda: attn(p, kp=b.offset(8)),
                 lambda: attn(p, wsp=ctx.zeros(1, np.uint8).offset(1)), lambda: pro(p, q=None, k=None, v=None),
                 lambda: pro(p, v=None), lambda: pro(p, k=None), lambda: pro(p, parts=0), lambda: pro(p, parts=2),
                 lambda: pro(p, rope=b, rows=63), lambda: pro(p, rope=b.offset(4), rows=64),
                 lambda: pro(p, rope=b, rows=0, pos=b), lambda: pro(p, qo=None), lambda: pro(p, kw=None),
                 lambda: pro(p, k=b.offset(4)), lambda: evict(p, kp=None), lambda: evict(p, mass=None),
                 lambda: evict(p, kept=None), lambda: evict(p, wsp=ctx.zeros(8, np.uint8)),
                 lambda: evict(p, keep=0), lambda: evict(p, keep=65), lambda: evict(p, first=20, recent=13),
                 lambda: evict(p, first=33), lambda: evict(p, first=2, recent=0xffffffff),
                 lambda: evict(p, kp=b.offset(8)),
                 lambda: ctx.kv4Values(b, b, b, b, b, 1, 24, 1, 256, 4, b, b),
                 lambda: ctx.kv4Values(b, b, b, b, b, 0, 16, 1, 256, 4, b, b),
                 lambda: ctx.kv4Values(b, b, b, b, None, 1, 16, 1, 256, 4, b, b)):
        with pytest.raises(g4hip.G4Error):
            call()


def test_starts_that_give_rows_to_many_sequences(ctx):
    """Every other sequence's starts descend, the others hold all rows each: 1024 x 4096 tiles of some 1900 steps are
    more than 32 bits number. Nothing is written or added, and every wait ends."""
    S, rows, hd, top = 2048, 16384, 64, 1 << 17
    p = ctx.kv4_params(S, 16, 1, hd, 1024, top // 1024, top, 2, num_rows=rows, max_rows=rows)
    pool, scale = ctx.zeros(1024 * hd, np.uint8), ctx.from_numpy(np.full(2 * 1024 * hd // 32, 127, np.uint8))
    table, lens = ctx.zeros(S * (top // 1024), np.int32), ctx.from_numpy(np.full(S, top, np.uint32))
    starts = ctx.from_numpy(np.where(np.arange(S + 1) % 2, rows, 0).astype(np.uint32))
    q, out = ctx.zeros(rows * 16 * hd, np.float32), ctx.from_numpy(np.full(rows * 16 * hd, 7.5, np.float32))
    mass = ctx.from_numpy(np.full(2 * 1024, 2.5, np.float32))
    ws = ctx.alloc(ctx.attn4_workspace_bytes(p, True))
    ctx.pagedAttn4(q, pool, pool, scale, scale, table, lens, out, p, ws, row_starts=starts, mass=mass)
    assert np.all(out.download(np.float32) == 7.5) and np.all(mass.download(np.float32) == 2.5)
