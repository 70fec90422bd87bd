"""The 8-bit paged K/V pool on the GPU: the prologue's codes, scales and q, the
values read back, and the attention, against float64 (kv8_oracle).

Codes and scales are equal to the oracle's: both round a value that is off by at
most about 1e-13 of itself, and the oracle's distance to the next border of two
codes is checked to be more than 1e-9. q: a sum of `parts` terms, each partial sum
rounded to 2^-24 of at most the sum of their magnitudes, then the norm's and the
rotation's few roundings: (parts + 10) * 2^-24 of what |x0| + |x1| would be with
the parts' magnitudes in their place. Attention: each of a score's products is off
by a few roundings of itself, the score by those of A = sum |q k|, so a weight p
is off by some 6 * 2^-24 (8 + A) of itself (exp and the sums: the 8) and the
output by that of sum p |v|; and p itself is held to 2^-40 of the largest (f16
pairs at 2^15: the steps below 2^-14 are 2^-24, half of one is 2^-25), each of n
times at most 127 scales."""
import numpy as np
import pytest

import g4hip
import kv8_oracle as K8
import oracle as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


class Case:
    """A batch with its pages on the host and the device; `rows` new rows per sequence, lengths counting them."""

    def __init__(self, ctx, lens, rows, nqh, nkh, hd, ps, seed, spare=2, window=0, scale=1.0, parts=1, extra_rows=0,
                 max_len=None):
        self.ctx, self.parts, self.hd = ctx, parts, hd
        self.lens, self.n = np.asarray(lens), np.asarray(rows)
        rng = self.rng = np.random.default_rng(seed)
        S, R = len(lens), int(self.n.sum()) + extra_rows
        max_len = max_len or max(1, int(self.lens.max()))
        per = -(-np.maximum(self.lens, 1) // ps)
        self.width = -(-max_len // ps)
        per = np.minimum(per, self.width)
        self.pages = int(per.sum()) + spare
        order = rng.permutation(self.pages)
        self.table = np.full((S, self.width), -1, np.int32)
        at = 0
        for s in range(S):
            self.table[s, :per[s]] = order[at:at + per[s]]
            at += per[s]
        self.starts = np.concatenate([[0], np.cumsum(self.n)]).astype(np.uint32)
        self.one = extra_rows == 0 and np.all(self.n == 1)
        self.p = ctx.kv8_params(S, nqh, nkh, hd, ps, self.width, max_len, self.pages, num_rows=R,
                                max_rows=max(1, int(self.n.max())), window=window, scale=scale)
        e = rng.integers(-6, -3, (2, self.pages, nkh))
        codes = np.rint(rng.normal(0, 1, (2, self.pages, ps, nkh, hd)) * 2.0 ** -e[:, :, None, :, None])
        codes = np.clip(codes, -127, 127).astype(np.int8)
        self.k, self.v = (K8.Pool(codes[i], (2.0 ** e[i]).astype(np.float32)) for i in (0, 1))
        self.q = rng.normal(0, 1.5 / np.sqrt(hd), (R, nqh, hd)).astype(np.float32)

    def up(self):
        c = self.ctx
        self.dk, self.dv = c.from_numpy(self.k.codes), c.from_numpy(self.v.codes)
        self.dks, self.dvs = c.from_numpy(self.k.scale), c.from_numpy(self.v.scale)
        self.dt, self.dl = c.from_numpy(self.table), c.from_numpy(self.lens.astype(np.uint32))
        self.ds = None if self.one else c.from_numpy(self.starts)
        self.cache = (self.dk, self.dv, self.dks, self.dvs)
        return self

    def row(self, r):
        """(sequence, position) of row r."""
        s = int(np.searchsorted(self.starts, r, side="right")) - 1
        return s, int(self.lens[s]) - int(self.n[s]) + r - int(self.starts[s])

    def attention(self, workspace=None):
        c, p = self.ctx, self.p
        out = c.from_numpy(np.full(self.q.shape, 7.5, np.float32))
        ws = workspace
        if ws is None:  # of any content
            ws = c.from_numpy(np.full(c.attn8_workspace_bytes(p), 0xff, np.uint8))
        c.pagedAttn8(c.from_numpy(self.q), *self.cache, self.dt, self.dl, out, p, ws, row_starts=self.ds)
        return out.download(np.float32).reshape(self.q.shape)

    def check_attention(self, got, rows=None, what=""):
        k, v = self.k.values(), self.v.values()
        total = int(self.n.sum())
        for r in range(total) if rows is None else rows:
            s, pos = self.row(r)
            want, mag, reach = K8.attend(self.q[r], k, v, self.table[s], pos, self.p.sliding_window, self.p.scale)
            if pos < 0:
                assert np.all(got[r] == 0), (what, r)
                continue
            pages = np.clip(self.table[s][:pos // self.k.codes.shape[1] + 1], 0, self.pages - 1)
            tol = 6 * U * (8 + reach) * mag + 2.0 ** -40 * (pos + 1) * 127 * np.nanmax(self.v.scale[pages]) + 1e-30
            off = float((np.abs(got[r] - want) / tol).max())
            assert off <= 1, (what, r, s, pos, off)
        assert np.all(got[total:] == 7.5), what


def table_of(ctx, hd, rows, theta=1e4):
    t = ctx.empty(rows * hd, np.float32)
    ctx.ropeTable(theta, 0, None, hd, rows, t)
    return t, t.download(np.float32).reshape(rows, hd // 2, 2)


def prologue(c: Case, q=None, k=None, v=None, table=None, qw=None, kw=None, rows_of=None):
    """Runs the prologue and checks q, codes and scales; returns q."""
    ctx, p, hd = c.ctx, c.p, c.hd
    R = p.num_rows
    host_table = table_of(ctx, hd, p.max_seq_len)[1]
    freqs = ctx.from_numpy(np.ones(hd // 2, np.float16))
    out = ctx.from_numpy(np.full(R * p.num_q_heads * hd, 3.25, np.float32))
    dev = [None if x is None else ctx.from_numpy(x) for x in (q, k, v, qw, kw)]
    cache = c.cache if k is not None else (None, None, None, None)
    ctx.pagedAttnPrologue8(dev[0], dev[1], dev[2], c.parts, dev[3], dev[4], freqs, out if q is not None else None,
                           *cache, c.dt, c.dl, p, row_starts=c.ds, rope_cs=table,
                           rope_rows=p.max_seq_len if table else 0)
    got = out.download(np.float32).reshape(R, p.num_q_heads, hd)
    done = np.zeros(R, bool)
    for s in range(p.num_seqs):
        a, n, L = int(c.starts[s]), int(c.n[s]), int(c.lens[s])
        if n == 0 or L < n or L > p.max_seq_len or n > p.max_rows:
            continue
        done[a:a + n] = True
        cs = host_table[L - n:L]
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
    assert np.all(got[~done] == 3.25)
    if k is not None:
        check_pools(c)
    return got


def check_pools(c):
    assert min(c.k.border, c.v.border) > 1e-9
    for pool, d, ds in ((c.k, c.dk, c.dks), (c.v, c.dv, c.dvs)):
        np.testing.assert_array_equal(ds.download(np.float32).reshape(pool.scale.shape), pool.scale)
        np.testing.assert_array_equal(d.download(np.int8).reshape(pool.codes.shape), pool.codes)


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
]


@pytest.mark.parametrize("lens,rows,nqh,nkh,hd,ps,parts", SHAPES)
@pytest.mark.parametrize("with_table", [False, True])
def test_prologue(ctx, lens, rows, nqh, nkh, hd, ps, parts, with_table):
    c = Case(ctx, lens, rows, nqh, nkh, hd, ps, 11, parts=parts, extra_rows=2 if len(lens) > 1 else 0).up()
    q, k, v, qw, kw = projections(c, 12)
    table = table_of(ctx, hd, c.p.max_seq_len)[0] if with_table else None
    prologue(c, q, k, v, table, qw, kw)


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("rows,ps", [(1, 16), (3, 16), (4, 64), (5, 16), (40, 16), (70, 64), (130, 128)])
@pytest.mark.parametrize("with_table", [False, True])
def test_prologue_of_each_launch(ctx, hd, rows, ps, with_table):
    """Few rows, many rows of small pages and of large ones, at each head dim; rows that begin within a page and end
    in another, a sequence of one row and one of none beside them."""
    nqh, nkh = (6, 2) if hd == 64 else (8, 1)
    c = Case(ctx, [3 * ps + rows // 2 + 1, 7, 2 * ps, rows], [rows, 1, 0, rows], nqh, nkh, hd, ps, 13, parts=5).up()
    q, k, v, qw, kw = projections(c, 14)
    prologue(c, q, k, v, table_of(ctx, hd, c.p.max_seq_len)[0] if with_table else None, qw, kw)


def test_prologue_q_alone_and_kv_alone(ctx):
    c = Case(ctx, [20, 9], [3, 9], 8, 2, 128, 16, 21).up()
    q, k, v, qw, kw = projections(c, 22)
    prologue(c, q=q, qw=qw)
    check_pools(c)
    prologue(c, k=k, v=v, kw=kw)


def test_scale_grows_token_by_token(ctx):
    """Rows of growing values, one call each: pages begun, grown and filled; then the same rows again in one call
    over fresh pages. K's norm weight makes its scale grow within a page."""
    c = Case(ctx, [1], [1], 8, 1, 64, 16, 31, max_len=40, spare=4)
    c.table[0, :3] = [2, 0, 3]
    c.up()
    rng = np.random.default_rng(32)
    for n in range(1, 38):
        c.lens[:] = n
        c.dl.upload(c.lens.astype(np.uint32))
        q, k, v, qw, kw = projections(c, 100 + n)
        k[:, :, :, rng.integers(0, 64)] *= 1 + n  # a spike: larger elements after the norm
        prologue(c, q, k, v, None, qw, (kw * np.float16(1 + n % 11)).astype(np.float16))


def test_zero_rows_and_the_border_of_an_octave(ctx):
    c = Case(ctx, [32], [32], 1, 1, 64, 16, 41).up()
    k, v = np.zeros((1, 32, 1, 64), np.float32), np.zeros((1, 32, 1, 64), np.float32)
    # one element only: the norm makes it 8, above 127 * 2^-4 = 7.9375
    v[0, 16:, 0, 5] = 3.0
    q, _, _, qw, kw = projections(c, 42)
    ctx.pagedAttnPrologue8(None, ctx.from_numpy(k), ctx.from_numpy(v), 1, None, ctx.from_numpy(kw), None, None,
                           *c.cache, c.dt, c.dl, c.p, row_starts=c.ds)
    ks, vs = (d.download(np.float32).reshape(-1) for d in (c.dks, c.dvs))
    assert np.all(ks[c.table[0, :2]] == 2.0 ** -64)
    assert list(vs[c.table[0, :2]]) == [2.0 ** -64, 2.0 ** -3]
    codes = c.dv.download(np.int8).reshape(c.v.codes.shape)[c.table[0, 1]]
    assert np.all(codes[:, 0, 5] == 64) and np.count_nonzero(codes) == 16


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_non_finite_rows_mark_their_page_and_head(ctx, bad):
    c = Case(ctx, [24, 20], [1, 1], 4, 2, 128, 16, 51, max_len=64).up()
    for step, poison in ((0, True), (1, False)):  # the row after stays marked
        c.lens += 1
        c.dl.upload(c.lens.astype(np.uint32))
        q, k, v, qw, kw = projections(c, 52 + step)
        if poison:
            k[0, 0, 1, 7] = bad
            v[0, 1, 0, 100] = bad
        prologue(c, q, k, v, None, qw, kw)
        pk, pv = c.table[0, 1], c.table[1, 1]
        assert np.isnan(c.k.scale[pk]).tolist() == [False, True] and np.isnan(c.v.scale[pv]).tolist() == [True, False]
    got = c.attention()
    assert np.all(np.isnan(got[0, 2:])) and np.all(np.isfinite(got[0, :2]))
    assert np.all(np.isnan(got[1, :2])) and np.all(np.isfinite(got[1, 2:]))
    # a page begun again is a page like any other
    c.lens[:] = 17
    c.dl.upload(c.lens.astype(np.uint32))
    q, k, v, qw, kw = projections(c, 55)
    prologue(c, q, k, v, None, qw, kw)
    c.check_attention(c.attention())


def test_lengths_starts_and_pages_that_do_not_hold(ctx):
    """A sequence shorter than its rows, one longer than max_seq_len, one of length 0, bad page ids, and starts that
    descend, pass num_rows or hold more than max_rows rows."""
    c = Case(ctx, [2, 99, 0, 20, 20, 30], [3, 1, 1, 2, 1, 3], 8, 1, 256, 16, 61, extra_rows=3, max_len=48)
    c.table[3, 1] = c.pages + 5
    c.table[4, 1] = -7
    c.up()
    q, k, v, qw, kw = projections(c, 62)
    prologue(c, q, k, v, None, qw, kw)
    got = c.attention()
    n = c.starts
    assert np.all(got[n[0]:n[3]] == 0)  # nothing to see
    c.lens[:3] = 3
    ok = range(int(n[3]), int(n[6]))
    c.check_attention(got, ok)
    # starts: sequence 1 descends, sequence 3 passes num_rows, sequence 5 holds too many
    starts = np.array([0, 3, 2, 4, 400, 5, 11], np.uint32)
    c.ds.upload(starts)
    c.dl.upload(np.full(6, 40, np.uint32))
    out = ctx.from_numpy(np.full(q.shape[1:], 7.5, np.float32))
    before = c.dk.download(np.int8), c.dv.download(np.int8)
    ws = ctx.alloc(ctx.attn8_workspace_bytes(c.p))
    ctx.pagedAttn8(ctx.from_numpy(c.q), *c.cache, c.dt, c.dl, out, c.p, ws, row_starts=c.ds)
    got = out.download(np.float32).reshape(q.shape[1:])
    assert np.all(got[5:] == 7.5)
    dq = ctx.from_numpy(np.full(q.shape[1:], 3.25, np.float32))
    ctx.pagedAttnPrologue8(ctx.from_numpy(q), ctx.from_numpy(k), ctx.from_numpy(v), 1, ctx.from_numpy(qw),
                           ctx.from_numpy(kw), None, dq, *c.cache, c.dt, c.dl, c.p, row_starts=c.ds)
    assert np.all(dq.download(np.float32).reshape(q.shape[1:])[5:] == 3.25)
    now = c.dk.download(np.int8), c.dv.download(np.int8)
    for s in (3, 4, 5):  # nothing appended for them
        pages = c.table[s][(c.table[s] >= 0) & (c.table[s] < c.pages)]
        for a, b in zip(before, now):
            assert np.array_equal(a.reshape(c.pages, -1)[pages], b.reshape(c.pages, -1)[pages])


@pytest.mark.parametrize("hd,nkh,ps", [(64, 3, 16), (256, 1, 48), (512, 2, 16)])
def test_values(ctx, hd, nkh, ps):
    c = Case(ctx, [5 * ps], [1], nkh, nkh, hd, ps, 71).up()
    pages = np.array([3, 0, 3, -1, c.pages, 5], np.int32)
    n = ps * nkh * hd
    k, v = ctx.empty(len(pages) * n, np.uint16), ctx.empty(len(pages) * n, np.uint16)
    ctx.kv8Values(*c.cache, ctx.from_numpy(pages), len(pages), ps, nkh, hd, c.pages, k, v)
    for pool, out in ((c.k, k), (c.v, v)):
        got = out.download(np.uint16).view(np.float16).reshape(len(pages), ps, nkh, hd)
        want = pool.values()
        for i, pg in enumerate(pages):
            assert np.array_equal(got[i], want[pg].astype(np.float16) if 0 <= pg < c.pages else np.zeros_like(got[i]))


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


@pytest.mark.parametrize("lens,rows,nqh,nkh,hd,ps,window", ATTN)
def test_attention(ctx, lens, rows, nqh, nkh, hd, ps, window):
    c = Case(ctx, lens, rows, nqh, nkh, hd, ps, 81, window=window, scale=0.8,
             extra_rows=0 if set(rows) == {1} else 2).up()
    got = c.attention()
    total = int(c.n.sum())
    rows = range(total) if total < 60 else sorted({*range(0, total, 7), total - 1, total - 2})
    c.check_attention(got, rows)
    assert np.array_equal(c.attention().view(np.uint32), got.view(np.uint32))  # the sums' order is fixed


@pytest.mark.parametrize("nkh,ragged", [(1, False), (3, True)])
def test_attention_of_many_sequences(ctx, nkh, ragged):
    """More sequences than a wave has lanes, some without positions or rows; shares that end inside one."""
    rng = np.random.default_rng(7)
    lens, rows = rng.integers(0, 400, 300), np.ones(300, int)
    lens[60:200] = 0
    if ragged:
        rows = rng.integers(0, 3, 300)
    c = Case(ctx, lens, rows, 4 * nkh, nkh, 128, 32, 86, extra_rows=int(ragged)).up()
    got = c.attention()
    total = int(c.n.sum())
    c.check_attention(got, range(0, total, 3))
    for r in range(total):
        assert np.any(got[r] != 0) == (c.row(r)[1] >= 0), r


@pytest.mark.parametrize("rows", [1, 40])
def test_attention_of_a_long_cache(ctx, rows):
    c = Case(ctx, [20011, 150], [rows, min(rows, 2)], 8, 1, 256, 16, 91).up()
    got = c.attention()
    total = int(c.n.sum())
    c.check_attention(got, sorted({0, rows // 2, rows - 1, total - 1}))


@pytest.mark.parametrize("hd,nkh", [(64, 2), (128, 1), (512, 1)])
@pytest.mark.parametrize("rows", [1, 20])
def test_attention_of_a_long_cache_at_each_head_dim(ctx, rows, hd, nkh):
    """More than 32 workgroups of one sequence; more than one round of a tile's pages."""
    c = Case(ctx, [9003, 31], [rows, 1], 8 * nkh, nkh, hd, 48, 92).up()
    got = c.attention()
    c.check_attention(got, sorted({0, rows // 2, rows - 1, rows}))


@pytest.mark.parametrize("rows", [1, 20])
def test_attention_masks_and_extremes(ctx, rows):
    """Pages outside the window or behind the length may hold anything: NaN scales there stay there. A dominant key
    whose values are 0 leaves the others their share; scales far apart meet in one row."""
    c = Case(ctx, [300, 300], [rows, rows], 8, 1, 256, 16, 101, window=100, max_len=400)
    far = [c.table[s, j] for s in (0, 1) for j in range((300 - rows - 100) // 16)]
    for pool in (c.k, c.v):
        pool.scale[far] = np.nan
        pool.scale[-2:] = np.inf
    for s in (0, 1):
        c.table[s, 19:] = c.pages - 1
    # sequence 1: the V scales of its pages from 2^-30 to 2^20
    c.v.scale[c.table[1, 11:19], 0] = 2.0 ** np.array([-30, -10, -6, 0, 5, 20, -20, -5])
    # sequence 0: position 290 - rows is 18 above the rest (q . k), its values zero
    pg, slot = c.table[0, (290 - rows) // 16], (290 - rows) % 16
    c.v.codes[pg, slot] = 0
    c.q[:rows] *= 0.01
    d = c.rng.normal(size=(1, 1, 256)).astype(np.float32)
    c.q[:rows] += 0.05 * d
    near = c.table[0, 11:19]
    c.k.codes[near] = np.rint(c.k.codes[near] * 0.05)
    c.k.codes[pg, slot, 0] = np.clip(np.rint(d[0, 0] * 40), -127, 127)
    c.k.scale[pg, 0] = 2.0 ** -5
    c.up()
    c.check_attention(c.attention())


@pytest.mark.parametrize("hd,rows,window", [(256, 2, 0), (256, 2, 20), (512, 2, 0), (128, 70, 0), (256, 40, 30),
                                            (512, 40, 0), (64, 300, 0)])
def test_a_page_that_is_not_finite_stays_with_the_rows_that_see_it(ctx, hd, rows, window):
    """The rows before a page's first position do not see it, though their step of positions may hold nothing else."""
    c = Case(ctx, [97 if rows == 2 else 80 + rows], [rows], 8, 1, hd, 16, 111, window=window).up()
    page = 6  # from position 96 on
    for k, v in ((np.nan, 1.0), (1.0, np.nan), (np.nan, np.nan), (1.0, np.inf)):
        ks, vs = c.k.scale.copy(), c.v.scale.copy()
        ks[c.table[0, page]] *= k
        vs[c.table[0, page]] *= v
        c.dks.upload(ks)
        c.dvs.upload(vs)
        got = c.attention()
        pos = c.lens[0] - rows + np.arange(rows)
        sees = (pos >= 16 * page) & ((window == 0) | (pos - window + 1 < 16 * page + 16))
        assert 0 < sees.sum() < rows
        assert not np.isfinite(got[sees]).any()
        c.check_attention(got, np.flatnonzero(~sees), what=(k, v))


@pytest.mark.parametrize("hd,rows", [(256, 1), (512, 1), (64, 90), (128, 90), (256, 90), (512, 90)])
def test_scales_and_q_of_nothing(ctx, hd, rows):
    """Pages of zeros as the append leaves them (2^-64) or never begun (0), next to pages that hold something; q so
    small that every score is 0 in f32, and q of zeros."""
    for what in ("least", "never begun", "all never begun", "small q", "small q, least", "q of zeros"):
        c = Case(ctx, [150], [rows], 8, 1, hd, 16, 121, scale=0.7)
        for pool in (c.k, c.v):
            if "least" in what:
                pool.scale[c.table[0, 2:10]] = 2.0 ** -64
                pool.codes[c.table[0, 2:10]] = 0
            if "never" in what:
                pool.scale[c.table[0, 2 if what[0] == "n" else 0:]] = 0
        c.q *= np.float32(1e-33 if "small" in what else 0.0 if "zeros" in what else 1.0)
        c.up()
        c.check_attention(c.attention(), sorted({0, 5, 63, 64, rows - 1} & set(range(rows))), what=what)


@pytest.mark.parametrize("scale", [-0.9, 0.0, 1e-30])
@pytest.mark.parametrize("hd,rows,window", [(256, 1, 0), (512, 1, 40), (64, 50, 0), (256, 50, 60), (512, 50, 0)])
def test_scale_of_any_sign(ctx, hd, rows, window, scale):
    c = Case(ctx, [170, 60], [rows, rows], 8, 1, hd, 32, 131, window=window, scale=scale).up()
    c.check_attention(c.attention(), sorted({0, 7, 8, rows - 1, rows, 2 * rows - 1} & set(range(2 * rows))))


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
    got = c.attention()
    total = int(c.n.sum())
    short = [r for r in range(total) if c.lens[c.row(r)[0]] < c.n[c.row(r)[0]]]
    assert short and np.all(got[short] == 0)
    c.check_attention(got, sorted((set(range(0, total, 11)) | {total - 1}) - set(short)))


def test_two_graphs_share_a_workspace(ctx):
    """Prompts and steps captured apart into graphs over one workspace, replayed in turn with eager calls between."""
    a = Case(ctx, [300], [120], 8, 1, 256, 16, 151).up()
    b = Case(ctx, [700, 40], [1, 1], 8, 1, 512, 16, 152).up()
    bytes_ = max(ctx.attn8_workspace_bytes(c.p) for c in (a, b))
    ws = ctx.from_numpy(np.full(bytes_, 0xff, np.uint8))
    want = [c.attention() for c in (a, b)]
    runs = []
    for c in (a, b):
        q, out = ctx.from_numpy(c.q), ctx.from_numpy(np.full(c.q.shape, 7.5, np.float32))
        ctx.graph_begin()
        ctx.pagedAttn8(q, *c.cache, c.dt, c.dl, out, c.p, ws, row_starts=c.ds)
        runs.append((ctx.graph_end(), q, out, c))
    for _ in range(4):
        for i in (0, 1, 1, 0):
            g, _, out, c = runs[i]
            out.upload(np.full(c.q.shape, 7.5, np.float32))
            ctx.graph_launch(g)
            got = out.download(np.float32).reshape(c.q.shape)
            assert np.array_equal(got.view(np.uint32), want[i].view(np.uint32))
            eager = runs[1 - i][3]
            assert np.array_equal(eager.attention(ws).view(np.uint32), want[1 - i].view(np.uint32))
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
            c.k.codes[pg, slot], c.k.scale[pg] = 0, 1.0
            c.k.codes[pg, slot, 0, 0] = {a: 100, b: 80}.get(pos, -100)
            c.v.codes[pg, slot] *= np.int8(pos != a)
        c.q[:] = 0
        c.q[..., 0] = -np.log(far) / 20
        c.up()
        c.check_attention(c.attention(), what=(a, b))


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
    ops, out = ctx.from_numpy(np.full(size, 0x5a, np.uint8)), ctx.empty(c.q.size, np.float32)
    ws = ctx.alloc(ctx.attn8_workspace_bytes(c.p))
    ctx.pagedAttn8(ctx.from_numpy(c.q), *c.cache, c.dt, c.dl, out, c.p, ws, row_starts=c.ds, ops=ops)
    y = out.download(np.float32).reshape(c.q.shape)
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
    scaled = want / sc[:, :R, None]
    assert np.all((np.abs(scaled).max(-1) < 2.0 ** 14) & ((np.abs(scaled).max(-1) >= 2.0 ** 13) | (top[..., 0] == 0)))
    sub = scaled.reshape(nblk, R, 8, 32)
    tol = 32 * U * np.abs(sub).sum(-1) + 2.0 ** -24 * 64
    assert (np.abs(p[:, :R].sum(-1) * 64 - sub.sum(-1)) <= tol).all() and np.all(p[:, :R, :, 3] == 0)
    raw = b[:, :main].reshape(nblk, ntv, 8, 2, 4, 16, 16).transpose(0, 1, 5, 2, 3, 4, 6).reshape(nblk, 16 * ntv, -1)
    assert np.all(raw[:, R:] == 0x5a)


def test_attention_of_far_pages(ctx):
    """Pools of more than 4 GiB: page offsets past 32 bits."""
    hd, ps, pages = 512, 16, (1 << 32) // (16 * 512) + 40
    c = Case(ctx, [100, 70], [1, 1], 8, 1, hd, ps, 111)
    small, shift = c.pages, pages - c.pages
    pool_k, pool_v = ctx.alloc(pages * ps * hd), ctx.alloc(pages * ps * hd)
    scales = [ctx.alloc(4 * pages) for _ in range(2)]
    pool_k.offset(shift * ps * hd).upload(c.k.codes)
    pool_v.offset(shift * ps * hd).upload(c.v.codes)
    scales[0].offset(4 * shift).upload(c.k.scale)
    scales[1].offset(4 * shift).upload(c.v.scale)
    c.up()
    host = c.table.copy()
    c.dt.upload(np.where(host >= 0, host + shift, -1).astype(np.int32))
    c.p.num_pages = pages
    c.cache = (pool_k, pool_v, scales[0], scales[1])
    c.check_attention(c.attention())
    q, k, v, qw, kw = projections(c, 112)
    ctx.pagedAttnPrologue8(None, ctx.from_numpy(k), ctx.from_numpy(v), 1, None, ctx.from_numpy(kw), None, None,
                           *c.cache, c.dt, c.dl, c.p)
    cs = table_of(ctx, hd, 100)[1]
    for s, L in enumerate(c.lens):
        c.k.append(K8.rotated(K8.normed(k[0, s:s + 1], kw), cs[L - 1:L]), host[s], int(L) - 1)
        c.v.append(K8.normed(v[0, s:s + 1]), host[s], int(L) - 1)
    got = pool_k.download(np.int8, small * ps * hd, offset=shift * ps * hd)
    assert np.array_equal(got, c.k.codes.reshape(-1))
    c.check_attention(c.attention())
    pages_dev = ctx.from_numpy((host[:, 0] + shift).astype(np.int32))
    out = [ctx.empty(2 * ps * hd, np.uint16) for _ in range(2)]
    ctx.kv8Values(*c.cache, pages_dev, 2, ps, 1, hd, pages, *out)
    assert np.array_equal(out[1].download(np.uint16).view(np.float16).reshape(2, ps, 1, hd),
                          c.v.values()[host[:, 0]].astype(np.float16))


def test_step_prompt_and_replays_together(ctx):
    """A prompt appended and attended to in one call each, then decode steps through a captured graph (two graphs over
    one workspace, replayed in turn) while the host goes on working: every replay against the oracle."""
    c = Case(ctx, [37, 21], [37, 21], 8, 1, 256, 16, 121, max_len=96, spare=8)
    for s in (0, 1):  # room for the steps
        free = [p for p in range(c.pages) if p not in c.table]
        c.table[s, 2 + (s == 0):5] = free[:3 - (s == 0)]
    c.up()
    q, k, v, qw, kw = projections(c, 122)
    table = table_of(ctx, 256, 96)[0]
    c.q = prologue(c, q, k, v, table, qw, kw) * np.float32(0.1)
    c.check_attention(c.attention(), [0, 1, 20, 36, 37, 57])
    # steps: one row each, read from the same buffers
    c.n[:], c.starts, c.one, c.ds = 1, np.array([0, 1, 2], np.uint32), True, None
    c.p = ctx.kv8_params(2, 8, 1, 256, 16, c.width, 96, c.pages)
    bufs = [ctx.empty(2 * 8 * 256, np.float32), ctx.empty(2 * 256, np.float32), ctx.empty(2 * 256, np.float32)]
    w = [ctx.from_numpy(qw), ctx.from_numpy((kw * np.float16(0.1)).astype(np.float16))]
    qo, out = ctx.empty(2 * 8 * 256, np.float32), ctx.empty(2 * 8 * 256, np.float32)
    ws = ctx.alloc(ctx.attn8_workspace_bytes(c.p))
    graphs = []
    for _ in range(2):
        ctx.graph_begin()
        ctx.advanceSeqLens(c.dl, 2, 1)
        ctx.pagedAttnPrologue8(bufs[0], bufs[1], bufs[2], 1, w[0], w[1], None, qo, *c.cache, c.dt, c.dl, c.p,
                               rope_cs=table, rope_rows=96)
        ctx.pagedAttn8(qo, *c.cache, c.dt, c.dl, out, c.p, ws)
        graphs.append(ctx.graph_end())
    host_table = table.download(np.float32).reshape(96, 128, 2)
    for step in range(24):
        q, k, v, _, _ = projections(c, 200 + step)
        for b, x in zip(bufs, (q, k, v)):
            b.upload(x)
        ctx.graph_launch(graphs[step % 2])
        c.lens += 1
        for s, L in enumerate(c.lens):
            cs = host_table[L - 1:L]
            kn = K8.normed(k[0, s:s + 1], (kw * np.float16(0.1)).astype(np.float16))
            c.k.append(K8.rotated(kn, cs), c.table[s], L - 1)
            c.v.append(K8.normed(v[0, s:s + 1]), c.table[s], L - 1)
        c.q = qo.download(np.float32).reshape(2, 8, 256)
        c.check_attention(out.download(np.float32).reshape(2, 8, 256), what=step)
        check_pools(c)
    for g in graphs:
        ctx.graph_destroy(g)


def test_refusals(ctx):
    b = ctx.zeros(1 << 16, np.uint8)
    ws = ctx.zeros(1 << 22, np.uint8)
    good = dict(num_seqs=2, nqh=8, nkh=1, hd=256, page_size=16, max_pages=4, max_seq_len=64, num_pages=9)

    def attn(p, q=b, kp=b, wsp=ws, rs=None):
        ctx.pagedAttn8(q, kp, b, b, b, b, b, b, p, wsp, row_starts=rs)

    def pro(p, q=b, k=b, v=b, parts=1, rope=None, rows=0, rs=None, qo=b, kw=b):
        ctx.pagedAttnPrologue8(q, k, v, parts, b, kw, None, qo, b, b, b, b, b, b, p, row_starts=rs, rope_cs=rope,
                               rope_rows=rows)

    for change in (dict(nqh=7, nkh=2), dict(nqh=17), dict(nqh=65, nkh=65), dict(hd=96), dict(page_size=24),
                   dict(page_size=0), dict(page_size=2048), dict(max_seq_len=65), dict(max_seq_len=0),
                   dict(num_seqs=0), dict(num_rows=3), dict(max_rows=2), dict(num_rows=70000, max_rows=70000),
                   dict(num_pages=0)):
        p = ctx.kv8_params(**{**good, **change})
        for f in (attn, pro):
            with pytest.raises(g4hip.G4Error):
                f(p)
    p = ctx.kv8_params(**good)
    for call in (lambda: attn(p, q=None), lambda: attn(p, q=b.offset(4)), lambda: attn(p, kp=b.offset(8)),
                 lambda: attn(p, wsp=ctx.zeros(1, np.uint8).offset(1)), lambda: pro(p, q=None, k=None, v=None),
                 lambda: pro(p, v=None), lambda: pro(p, k=None), lambda: pro(p, parts=0), lambda: pro(p, parts=2),
                 lambda: pro(p, rope=b, rows=63), lambda: pro(p, rope=b.offset(4), rows=64),
                 lambda: pro(p, qo=None), lambda: pro(p, kw=None), lambda: pro(p, k=b.offset(4)),
                 lambda: ctx.kv8Values(b, b, b, b, b, 1, 24, 1, 256, 4, b, b),
                 lambda: ctx.kv8Values(b, b, b, b, b, 0, 16, 1, 256, 4, b, b),
                 lambda: ctx.kv8Values(b, b, b, b, None, 1, 16, 1, 256, 4, b, b)):
        with pytest.raises(g4hip.G4Error):
            call()


def test_operand_blocks_that_are_refused(ctx):
    b = ctx.zeros(1 << 20, np.uint8)
    ws = ctx.zeros(1 << 24, np.uint8)
    for change in (dict(hd=128), dict(num_seqs=65), dict(num_rows=6, max_rows=3), dict(ops=b.offset(8))):
        ops = change.pop("ops", b)
        p = ctx.kv8_params(**{**dict(num_seqs=2, nqh=8, nkh=1, hd=256, page_size=16, max_pages=4, max_seq_len=64,
                                     num_pages=9), **change})
        with pytest.raises(g4hip.G4Error):
            ctx.pagedAttn8(b, b, b, b, b, b, b, b, p, ws, row_starts=b if p.num_rows != p.num_seqs else None, ops=ops)


def test_starts_that_give_rows_to_many_sequences(ctx):
    """Every other sequence's starts descend, the others hold all rows each: 1024 x 4096 tiles of some 1900 steps are
    more than 32 bits number. Nothing is written, and every wait ends."""
    S, rows, hd, top = 2048, 16384, 64, 1 << 17
    p = ctx.kv8_params(S, 16, 1, hd, 1024, top // 1024, top, 2, num_rows=rows, max_rows=rows)
    assert S // 2 * (rows * 16 // 64) * ((top - rows) // 64) > 2 ** 32
    pool, scale = ctx.zeros(2 * 1024 * hd, np.int8), ctx.from_numpy(np.ones(2, np.float32))
    table, lens = ctx.zeros(S * (top // 1024), np.int32), ctx.from_numpy(np.full(S, top, np.uint32))
    starts = ctx.from_numpy(np.where(np.arange(S + 1) % 2, rows, 0).astype(np.uint32))
    q, out = ctx.zeros(rows * 16 * hd, np.float32), ctx.from_numpy(np.full(rows * 16 * hd, 7.5, np.float32))
    ws = ctx.from_numpy(np.full(ctx.attn8_workspace_bytes(p), 0xff, np.uint8))
    ctx.pagedAttn8(q, pool, pool, scale, scale, table, lens, out, p, ws, row_starts=starts)
    assert np.all(out.download(np.float32) == 7.5)


@pytest.mark.parametrize("hd,theta,divisor", [(64, 1e4, 1), (256, 1e6, 0), (512, 1e6, 1), (128, 5e5, 1)])
def test_prologue_by_theta_and_divisor(ctx, hd, theta, divisor):
    """Angles formed in the launch: of its theta, divided by the frequencies' table where it says so; the same bits as
    from a table, and cos and sin within 2^-22 of the f32 angle's."""
    c = Case(ctx, [61, 300], [9, 40], 8, 2, hd, 32, 181)
    c.p.theta, c.p.apply_divisor = theta, divisor
    rng = np.random.default_rng(182)
    freqs = rng.choice(np.array([1, 2, 8, 0.5], np.float16), hd // 2)
    n = c.p.max_seq_len
    t, df = ctx.empty(n * hd, np.float32), ctx.from_numpy(freqs)
    ctx.ropeTable(theta, divisor, df, hd, n, t)
    f = (1.0 / np.float64(np.float32(theta)) ** (2.0 * np.arange(hd // 2) / hd)).astype(np.float32)
    angle = np.arange(n, dtype=np.float32)[:, None] * (f / freqs.astype(np.float32) if divisor else f)
    host = t.download(np.float32).reshape(n, hd // 2, 2)
    # (theta^x by another library: an angle may be the next f32, 2^-23 of it)
    tol = 2.0 ** -22 * (1 + np.abs(angle.astype(np.float64)))
    for i, fn in enumerate((np.cos, np.sin)):
        assert (np.abs(host[..., i] - fn(angle.astype(np.float64))) <= tol).all()
    q, k, v, qw, kw = projections(c, 183)
    runs = []
    for table in (None, t):
        c.up()
        out = ctx.from_numpy(np.full(q[0].shape, 3.25, np.float32))
        ctx.pagedAttnPrologue8(*(ctx.from_numpy(x) for x in (q, k, v)), 1, ctx.from_numpy(qw), ctx.from_numpy(kw), df,
                               out, *c.cache, c.dt, c.dl, c.p, row_starts=c.ds, rope_cs=table,
                               rope_rows=n if table else 0)
        runs.append([out.download(np.uint32)] + [b.download(np.uint8) for b in c.cache])
    assert all(np.array_equal(a, b) for a, b in zip(*runs))
    got = runs[0][0].view(np.float32).reshape(q[0].shape)
    for s in range(2):
        a, m, L = int(c.starts[s]), int(c.n[s]), int(c.lens[s])
        x = K8.normed(q[0, a:a + m].astype(np.float64), qw)
        half = hd // 2
        mag = np.tile(np.abs(x[..., :half]) + np.abs(x[..., half:]), 2)
        assert (np.abs(got[a:a + m] - K8.rotated(x, host[L - m:L])) <= 11 * U * mag + 1e-30).all()
        c.k.append(K8.rotated(K8.normed(k[0, a:a + m], kw), host[L - m:L]), c.table[s], L - m)
        c.v.append(K8.normed(v[0, a:a + m]), c.table[s], L - m)
    check_pools(c)


@pytest.mark.parametrize("hd,ps", [(64, 256), (128, 1024), (256, 512), (512, 256), (512, 1024)])
def test_large_pages(ctx, hd, ps):
    """Pages of more rows than a workgroup keeps: begun, filled and left within; then steps and their attention."""
    c = Case(ctx, [ps + 700, 300, 2 * ps + 1], [ps + 333, 1, 2], 4, 2, hd, ps, 191, parts=2).up()
    q, k, v, qw, kw = projections(c, 192)
    got = prologue(c, q, k, v, table_of(ctx, hd, c.p.max_seq_len)[0], qw, kw)
    c.q = got * np.float32(0.1)
    total = int(c.n.sum())
    c.check_attention(c.attention(), sorted({0, 63, 64, ps - 1, total - 4, total - 3, total - 2, total - 1}))


def test_rows_taken_back(ctx):
    """Drafted rows whose length is set back: their page keeps the scale that they made grow, the codes before them
    the rounding to it, the next rows are appended under it; a page that they began is begun again."""
    c = Case(ctx, [21, 40], [5, 9], 4, 2, 128, 16, 201, max_len=64, spare=4)
    free = [p for p in range(c.pages) if p not in c.table]
    c.table[0, 2:4], c.table[1, 3] = free[:2], free[2]
    c.up()
    for step, (lens, spread) in enumerate([([21, 40], 1), ([24, 44], 9), ([23, 39], 1), ([28, 48], 1)]):
        c.lens[:] = lens
        c.dl.upload(c.lens.astype(np.uint32))
        q, k, v, qw, kw = projections(c, 202 + step)
        k[..., 3] *= spread  # a spike: the norm leaves a larger element
        v[..., 5] *= spread
        prologue(c, q, k, v, None, qw, kw)
        c.check_attention(c.attention(), what=step)


def test_steps_beside_a_prompt(ctx):
    rng = np.random.default_rng(211)
    lens, rows = rng.integers(1, 900, 65), np.ones(65, int)
    lens[20], rows[20] = 420, 300
    c = Case(ctx, lens, rows, 8, 1, 256, 16, 212, window=512).up()
    got = c.attention()
    total = int(c.n.sum())
    c.check_attention(got, sorted({*range(0, 20), *range(20, 320, 29), 319, *range(320, total)}))
