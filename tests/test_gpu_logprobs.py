"""Log probabilities, entropy and top alternatives on the GPU against float64.

A log probability is a difference of f32 numbers (value - maximum - log Z): its
error is a few roundings of the largest of them, 8 * 2^-24 (|x - m| + log Z + 1).
The entropy's sums add `size` terms in partial sums: the same of what they add
up to. Ids are equal."""
import numpy as np
import pytest

import g4hip
import kv8_oracle as K8

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def call(ctx, x, tokens, ntop, entropy=True):
    rows, size = x.shape
    outs = [ctx.from_numpy(np.full(rows, 9.0, np.float32)) for _ in range(2)]
    ids = ctx.from_numpy(np.full(rows * max(ntop, 1), 77, np.uint32))
    top = ctx.from_numpy(np.full(rows * max(ntop, 1), 9.0, np.float32))
    ws = ctx.from_numpy(np.full(ctx.logprobs_workspace_bytes(size, rows, ntop), 0xff, np.uint8))
    base = ctx.alloc(x.nbytes + 4).upload(x, 4)
    d = base.offset(4)  # rows of any alignment a float has
    ctx.logprobsBatch(d, None if tokens is None else ctx.from_numpy(tokens.astype(np.uint32)), size, rows,
                      None if tokens is None else outs[0], outs[1] if entropy else None, ntop, ids if ntop else None,
                      top if ntop else None, ws)
    got = (outs[0].download(np.float32), outs[1].download(np.float32), ids.download(np.uint32)[:rows * ntop],
           top.download(np.float32)[:rows * ntop])
    return got[0], got[1], got[2].reshape(rows, ntop), got[3].reshape(rows, ntop)


def check(ctx, x, tokens, ntop):
    lp, ent, ids, top = call(ctx, x, tokens, ntop)
    for r in range(len(x)):
        want = K8.logprobs(x[r], int(tokens[r]), ntop)
        assert np.array_equal(ids[r], want[2]), r
        with np.errstate(invalid="ignore"):
            d = x[r].astype(np.float64) - np.fmax.reduce(x[r])
            reach = np.log(x.shape[1]) + 1
        for got, ref, a in [(lp[r], want[0], d[tokens[r]] if 0 <= tokens[r] < x.shape[1] else 0)] + list(
                zip(top[r], want[3], d[ids[r]])):
            with np.errstate(over="ignore"):
                ref = ref if np.isfinite(np.float32(ref)) else np.float32(ref)  # (-6e38 is -Inf in f32)
            if np.isfinite(ref):
                assert abs(got - ref) <= 8 * U * (abs(a) + reach), (r, got, ref)
            else:
                assert np.array_equal(got, np.float32(ref), equal_nan=True), (r, got, ref)
        if np.isfinite(want[1]):
            assert abs(ent[r] - want[1]) <= 32 * U * reach, (r, ent[r], want[1])
        else:
            assert np.isnan(ent[r])
    return lp, ent, ids, top


@pytest.mark.parametrize("rows,size,ntop", [
    (1, 1, 1), (3, 2, 2), (2, 63, 5), (2, 64, 64), (5, 65, 20), (2, 255, 1), (3, 1000, 0), (4, 4095, 20), (3, 4097, 64),
    (2, 8193, 7), (1, 32003, 33), (40, 5000, 3), (1, 262144, 20), (9, 262144, 5), (300, 2049, 20), (2, 100003, 64),
])
def test_rows(ctx, rows, size, ntop):
    rng = np.random.default_rng(rows * 1000 + size)
    x = (30 * np.tanh(rng.normal(-4, 3, (rows, size)) / 30)).astype(np.float32)
    x[:, rng.integers(0, size)] += 12
    tokens = rng.integers(0, size, rows)
    got = check(ctx, x, tokens, ntop)
    again = call(ctx, x, tokens, ntop)
    for a, b in zip(got, again):  # the sums' order is fixed
        assert np.array_equal(a.view(np.uint32), b.view(np.uint32))


def test_ties_go_to_the_lowest_index(ctx):
    rng = np.random.default_rng(5)
    x = np.full((4, 20000), -3.0, np.float32)
    x[0] = np.round(rng.normal(0, 1.5, 20000))      # many equal values
    x[1, rng.integers(0, 20000, 30)] = 2.0
    x[2] = 0.0
    x[2, 1::2] = -0.0                               # equal to 0
    check(ctx, x, np.array([0, 19999, 3, 7]), 64)


def test_peaked_and_flat_rows(ctx):
    x = np.zeros((5, 30001), np.float32)
    x[0, 12345] = 1000.0
    x[1] = 3.0e38
    x[2] = -3.0e38
    x[2, 4] = 3.0e38
    x[3] = np.linspace(-80, 80, 30001)[::-1]
    x[4, 77] = 15.0
    check(ctx, x, np.array([12345, 5, 4, 30000, 77]), 20)


def test_infinities_and_nan(ctx):
    rng = np.random.default_rng(6)
    x = rng.normal(0, 2, (7, 9001)).astype(np.float32)
    x[0, ::3] = -np.inf
    x[1, 8] = np.nan
    x[2, 4000] = np.inf
    x[3] = -np.inf
    x[4] = np.nan
    x[5] = -np.inf
    x[5, 8999] = 1.0
    x[6, :] = np.nan
    x[6, 5000:5003] = [1.0, 2.0, 1.0]
    check(ctx, x, np.array([0, 1, 4000, 5, 6, 8999, 5000]), 8)


def test_values_of_the_lowest_f32(ctx):
    """A mask of the type's lowest value leaves probabilities of 0, not NaN."""
    x = np.full((1, 5000), np.finfo(np.float32).min, np.float32)
    x[0, [7, 4999]] = 1.0
    lp, ent, ids, _ = check(ctx, x, np.array([7]), 3)
    assert ids[0].tolist() == [7, 4999, 0] and abs(lp[0] + np.log(2)) < 1e-6 and abs(ent[0] - np.log(2)) < 1e-6


def test_tokens_outside_and_outputs_left_out(ctx):
    rng = np.random.default_rng(7)
    x = rng.normal(0, 2, (3, 6000)).astype(np.float32)
    lp, ent, _, _ = check(ctx, x, np.array([6000, 0xffffffff, 5999]), 2)
    assert np.isnan(lp[0]) and np.isnan(lp[1]) and np.all(np.isfinite(ent))
    a = call(ctx, x, None, 2)
    assert np.all(a[0] == 9.0) and np.array_equal(a[1], ent)
    b = call(ctx, x, np.array([1, 2, 3]), 0, entropy=False)
    assert np.all(b[1] == 9.0) and np.all(np.isfinite(b[0]))


def test_captured_and_replayed(ctx):
    rng = np.random.default_rng(8)
    rows, size, ntop = 5, 40001, 6
    x = ctx.empty(rows * size, np.float32)
    t = ctx.empty(rows, np.uint32)
    lp, ent = ctx.empty(rows, np.float32), ctx.empty(rows, np.float32)
    ids, top = ctx.empty(rows * ntop, np.uint32), ctx.empty(rows * ntop, np.float32)
    ws = ctx.alloc(ctx.logprobs_workspace_bytes(size, rows, ntop))
    graphs = []
    for _ in range(2):  # two graphs over one workspace
        ctx.graph_begin()
        ctx.logprobsBatch(x, t, size, rows, lp, ent, ntop, ids, top, ws)
        graphs.append(ctx.graph_end())
    for k in range(6):
        h, th = rng.normal(0, 3, (rows, size)).astype(np.float32), rng.integers(0, size, rows)
        x.upload(h)
        t.upload(th.astype(np.uint32))
        ctx.graph_launch(graphs[k % 2])
        got = [b.download(d) for b, d in ((lp, np.float32), (ent, np.float32), (ids, np.uint32), (top, np.float32))]
        want = call(ctx, h, th, ntop)
        for a, b in zip(got, want):
            assert np.array_equal(a.view(np.uint32), b.reshape(-1).view(np.uint32))
    for g in graphs:
        ctx.graph_destroy(g)


def test_refusals(ctx):
    b, ws = ctx.zeros(4096, np.float32), ctx.zeros(1 << 20, np.uint8)
    for args in ((b, b, 0, 1, b, b, 0, None, None, ws), (b, b, 10, 0, b, b, 0, None, None, ws),
                 (b, b, 10, 65536, b, b, 0, None, None, ws), (b, b, 10, 1, b, b, 11, b, b, ws),
                 (b, b, 100, 1, b, b, 65, b, b, ws), (b, None, 10, 1, b, b, 1, b, b, ws),
                 (b, b, 10, 1, None, b, 1, b, b, ws), (None, b, 10, 1, b, b, 1, b, b, ws),
                 (b, b, 10, 1, b, b, 1, None, b, ws), (b, b, 10, 1, b, b, 1, b, None, ws),
                 (b, b, 10, 1, b, b, 1, b, b, ws.offset(4))):
        with pytest.raises(g4hip.G4Error):
            ctx.logprobsBatch(*args)


@pytest.mark.parametrize("low", [-np.inf, np.finfo(np.float32).min])
@pytest.mark.parametrize("rows,size", [(17, 262144), (2, 100003)])
def test_rows_under_a_mask(ctx, rows, size, low):
    """A grammar leaves a few tokens of a large vocabulary: fewer than the alternatives asked for, or in few chunks."""
    rng = np.random.default_rng(9)
    x = np.full((rows, size), low, np.float32)
    tokens = np.zeros(rows, int)
    for r in range(rows):
        kept = rng.choice(size, [1, 3, 19, 20, 21, 2000, size // 3][r % 7], replace=False)
        if r % 2:
            kept = kept // 64  # (one chunk or a few)
        x[r, kept] = rng.normal(-4, 3, kept.size)
        tokens[r] = kept[0] if r % 3 else rng.integers(0, size)
    check(ctx, x, tokens, 20)
