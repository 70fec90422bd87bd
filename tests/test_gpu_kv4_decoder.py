"""The ragged step, batched prefill and scoring over 4-bit pages, with and without a budget of rows.

Every layer's attention is held to float64 over the device's own roped q and the pages' values (tolerances:
test_gpu_kv4's). A row appended to layer 0, whose input does not depend on the cache, is within a step of its scale of the
f16 decoder's row, and 2^-10 of the row's largest value (the f16 rounding, 2^-11 of a value, and the f32 roundings of
the two prologues)."""
import numpy as np
import pytest

import kv4_oracle as K4
from g4hip.decoder import BatchDecoder, E2BShape
from gpu_util import bits_equal
from test_gpu_kv4 import U, slack

pytestmark = pytest.mark.gpu
LENS = [0, 1, 15, 16, 63, 64, 511, 530]


def shape(kind="real"):
    if kind == "uniform":
        return E2BShape(n_layers=2, global_layers=(1,), vocab=4096)
    return E2BShape.real(n_layers=4, n_unshared=2, global_layers=(1, 3), vocab=4096)


def pools(d, il):
    """Layer il's K and V pages, as the device holds them."""
    s, L, src = d.s, d.layers[il], d.s.producer(il)
    n, ps, h, hd = d._pool_rows(il) // d.page_size, d.page_size, s.n_kv_heads, s.hd(il)
    ks, vs = (b.download(np.uint8) for b in d.kv_scales[src])
    k, v = (K4.unpack(b.download(np.uint8).reshape(n, ps, h, hd // 2)) for b in (L.k_cache, L.v_cache))
    return K4.Pool(k, ks.reshape(n, ps, h, hd // 32)), K4.Pool(v, K4.by_row(vs.reshape(n, ps // 16, h, hd // 32, 16)))


def table_of(d, il, seq):
    return d.cut_table_host[seq] if d._is_cut(il) else d.page_table_host[seq]


def check_rows(d, il, q, got, rows):
    """rows: (row, its sequence, its place in the cache)."""
    s = d.s
    k, v = (p.values() for p in pools(d, il))
    q, got = (x.reshape(-1, s.n_q_heads, s.hd(il)) for x in (q, got))
    for r, seq, pos in rows:
        table = table_of(d, il, seq)
        want, mag, reach, _ = K4.attend(q[r], k, v, table, pos, 0 if s.is_global(il) else s.window, 1.0)
        top = np.abs(v[table[:pos // d.page_size + 1]]).max()
        tol = slack(s.hd(il), pos + 1, reach) * mag + 2.0 ** -40 * (pos + 1) * top + 1e-30
        assert (np.abs(got[r] - want) <= tol).all(), (il, r, seq, pos, float((np.abs(got[r] - want) / tol).max()))


@pytest.mark.parametrize("kind,ps", [("real", 16), ("uniform", 64)])
def test_steps(ctx, kind, ps):
    kw = dict(page_size=ps, reserve=8, seed=41, embed=True)
    d = BatchDecoder(ctx, LENS, shape(kind), kv="fp4", **kw)
    f = BatchDecoder(ctx, LENS, shape(kind), **kw)
    d.fill_kv(seed=42)
    s, B = d.s, d.B
    rng = np.random.default_rng(43)
    for step in range(3):
        toks = rng.integers(0, s.vocab, B).astype(np.uint32)
        lens = np.array(LENS) + step
        for x in (d, f):
            x.tokens.upload(toks)
        seen = []

        def probe(stage, il, _):
            if stage == "attn":
                check_rows(d, il, d.q.download(np.float32, B * s.q_dim_of(il)),
                           d.attn.download(np.float32, B * s.q_dim_of(il)), [(b, b, int(lens[b])) for b in range(B)])
                seen.append(il)

        d.step(probe=probe)
        f.step()
        assert seen == list(range(s.n_layers))
        L, kv = f.layers[0], s.kv_dim_of(0)
        for pool, b16 in zip(pools(d, 0), (L.k_cache, L.v_cache)):
            b16, val = b16.download(np.float16).reshape(-1, kv), pool.values()
            for b in range(B):
                at = d.page_table_host[b, lens[b] // ps], lens[b] % ps
                r16 = b16[f.pool_row(b, int(lens[b]))].astype(np.float64)
                unit = np.repeat(2.0 ** (pool.scale[at].reshape(-1).astype(np.float64) - 127), 32)
                assert (np.abs(val[at].reshape(-1) - r16) <= unit + 2.0 ** -10 * np.abs(r16).max()).all(), (step, b)
    assert np.array_equal(d.seq_lens.download(np.uint32), np.array(LENS) + 3)


def test_eager_steps_after_replays_find_room(ctx):
    """The host does not count the replays of a captured step: a step of its own after them evicts where all of its own
    would have."""
    runs = []
    for replays in (0, 6):
        d = BatchDecoder(ctx, LENS, shape(), seed=53, reserve=24, embed=True, kv="fp4", budget=64, slack=8)
        d.fill_kv(seed=54)
        d.tokens.upload(np.arange(d.B, dtype=np.uint32))
        g = d.capture() if replays else None
        got = []
        for i in range(14):
            if i < replays:
                ctx.graph_launch(g)
            else:
                d.step()
            got.append([b.download(np.uint32) for b in (d.tokens, d.logits, d.cut_lens)])
        runs.append(got)
        if g is not None:
            ctx.graph_destroy(g)
    assert max(x[2].max() for x in runs[0]) == 72 and any(x[2].max() == 65 for x in runs[0][1:])
    for step, (a, b) in enumerate(zip(*runs)):
        assert all(np.array_equal(x, y) for x, y in zip(a, b)), step


def test_drafts_taken_back_and_a_sequence_begun_anew(ctx):
    """With caches that hold more than their budget: tokens taken back and decoded again leave the same bits; a sequence
    begun anew leaves the others what they had."""
    d = BatchDecoder(ctx, LENS, shape(), seed=57, reserve=24, embed=True, kv="fp4", budget=64, slack=12)
    d.fill_kv(seed=58)
    s = d.s
    toks = np.random.default_rng(59).integers(0, s.vocab, (8, d.B)).astype(np.uint32)

    def run(first, last):
        got = []
        for t in toks[first:last]:
            d.tokens.upload(t)
            d.step()
            got.append(d.logits.download(np.uint32))
        return got

    once = run(0, 6)
    d.set_lengths(np.array(LENS) + 2)
    cached = np.minimum(LENS, 64) + 2
    assert np.array_equal(d.cut_lens.download(np.uint32), cached)
    assert np.array_equal(run(2, 6), once[2:])
    lens = np.array(LENS) + 6
    lens[6] = 0
    d.set_lengths(lens)
    cached += 4
    cached[6] = 0
    assert np.array_equal(d.cut_lens.download(np.uint32), cached) and np.array_equal(d.seq_lens.download(np.uint32), lens)

    def probe(stage, il, _):
        if stage == "attn":
            at = cached if d._is_cut(il) else lens
            check_rows(d, il, d.q.download(np.float32, d.B * s.q_dim_of(il)),
                       d.attn.download(np.float32, d.B * s.q_dim_of(il)), [(b, b, int(at[b])) for b in range(d.B)])

    d.tokens.upload(toks[6])
    d.step(probe=probe)


def test_replays_past_the_room(ctx):
    """One and two replays too many (63 + 10 and 64 + 10 rows for 72): a step says so and changes nothing, evict() warns and
    cuts to the budget, and the next steps see what the caches hold."""
    d = BatchDecoder(ctx, LENS, shape(), seed=55, reserve=24, embed=True, kv="fp4", budget=64, slack=8)
    d.fill_kv(seed=56)
    d.tokens.upload(np.arange(d.B, dtype=np.uint32))
    g = d.capture()
    for _ in range(10):
        ctx.graph_launch(g)
    with pytest.raises(RuntimeError, match=r"2 rows of sequences \[4, 5, 6, 7\]"):
        d.step()
    assert np.array_equal(d.seq_lens.download(np.uint32), np.array(LENS) + 10)
    assert np.array_equal(d.cut_lens.download(np.uint32), np.minimum(LENS, 64) + 10)
    with pytest.warns(RuntimeWarning, match="2 rows"):
        d.evict()
    want = np.minimum(np.minimum(LENS, 64) + 10, 64)
    assert np.array_equal(d.cut_lens.download(np.uint32), want) and np.array_equal(d.cut_lens_host, want)
    s = d.s

    def probe(stage, il, _):
        if stage == "attn":
            at = want if d._is_cut(il) else np.array(LENS) + 10
            check_rows(d, il, d.q.download(np.float32, d.B * s.q_dim_of(il)),
                       d.attn.download(np.float32, d.B * s.q_dim_of(il)), [(b, b, int(at[b])) for b in range(d.B)])

    d.step(probe=probe)
    ctx.graph_launch(g)
    assert np.array_equal(d.cut_lens.download(np.uint32), want + 2)
    ctx.graph_destroy(g)


@pytest.mark.parametrize("budget", [None, 64])
def test_a_captured_step_equals_eager_ones(ctx, budget):
    runs = []
    for captured in (False, True):
        d = BatchDecoder(ctx, LENS, shape(), seed=51, reserve=24, embed=True, kv="fp4", budget=budget, slack=8)
        d.fill_kv(seed=52)
        d.tokens.upload(np.arange(d.B, dtype=np.uint32))
        g = d.capture() if captured else None
        got = []
        for i in range(20):  # (over a page's end)
            if budget and i % 8 == 0:
                d.evict()
            if captured:
                ctx.graph_launch(g)
            else:
                d.step()
            got.append([b.download(np.uint32) for b in (d.tokens, d.logits)])
        got.append([b.download(np.uint8) for L in d.layers for b in (L.k_cache, L.v_cache)])
        got.append([b.download(np.uint8) for p in d.kv_scales.values() for b in p])
        got.append([b.download(np.uint32) for b in d.mass.values()])
        runs.append(got)
        if captured:
            ctx.graph_destroy(g)
    for step, (a, b) in enumerate(zip(*runs)):
        assert all(np.array_equal(x, y) for x, y in zip(a, b)), step


@pytest.mark.parametrize("kind", ["real", "uniform"])
@pytest.mark.parametrize("T,start", [(1, 0), (5, 0), (16, 0), (20, 0), (21, 40), (3, 37)])
def test_prefill_in_chunks(ctx, kind, T, start):
    d = BatchDecoder(ctx, [0] * 16, shape(kind), seed=61, reserve=start + T + 8, shared_pages=True, embed=True, kv="fp4")
    d.fill_kv(seed=62)
    s, B = d.s, d.B
    chunk = [-1]

    def probe(stage, il, _):
        chunk[0] += stage == "prep" and il == 0
        if stage == "attn":
            n = min(B, T - B * chunk[0])
            q = d.q.download(np.float32, B * s.q_dim_of(il))
            check_rows(d, il, q, d.attn.download(np.float32, B * s.q_dim_of(il)),
                       [(r, 0, start + B * chunk[0] + r) for r in range(n)])

    toks = np.random.default_rng(63).integers(0, s.vocab, T).astype(np.uint32)
    last = d.prefill(toks, start, probe=probe)
    assert chunk[0] == -(-T // B) - 1 and last == (T - 1) % B
    H = d.hidden.download(np.float32).reshape(B, s.hidden)
    assert all(bits_equal(H[r], H[last]) for r in range(last + 1, B))


@pytest.mark.parametrize("kind,B,T,start", [("real", 16, 100, 0), ("real", 64, 700, 0), ("uniform", 64, 201, 100),
                                            ("uniform", 16, 97, 530)])
def test_prefill_many_rows_a_pass(ctx, kind, B, T, start):
    d = BatchDecoder(ctx, [0] * B, shape(kind), seed=71, reserve=start + T + 80, shared_pages=True, embed=True, kv="fp4")
    d.fill_kv(seed=72)
    s, il = d.s, d.s.n_layers - 1
    toks = np.random.default_rng(73).integers(0, s.vocab, T).astype(np.uint32)
    d.prefill(toks, start)
    assert d.wide_cap >= T  # (all rows in one pass)
    n = s.q_dim_of(il) * T
    rows = sorted({0, 1, 15, 16, 63, T // 2, T - 2, T - 1} & set(range(T)))
    check_rows(d, il, d.wide["q"].download(np.float32, n), d.wide["attn"].download(np.float32, n),
               [(r, 0, start + r) for r in rows])


def test_score(ctx):
    d = BatchDecoder(ctx, [0] * 16, shape(), seed=81, reserve=64, shared_pages=True, embed=True, kv="fp4", logprobs=3)
    d.fill_kv(seed=82)
    toks = np.random.default_rng(83).integers(0, d.s.vocab, 22).astype(np.uint32)
    got = d.score(toks, 5)
    for first, n in ((0, 16), (16, 5)):  # the same chunks again, one call each
        d.prefill(toks[first:first + n], 5 + first)
        x = d.logits.download(np.float32).reshape(16, -1)[:n].astype(np.float64)
        want = x[np.arange(n), toks[first + 1:first + n + 1]] - np.log(np.exp(x - x.max(1, keepdims=True)).sum(1)) - x.max(1)
        assert (np.abs(got[first:first + n] - want) <= 8 * U * (2 * np.abs(x).max() + np.log(d.s.vocab) + 1)).all()


@pytest.mark.parametrize("kind", ["real", "uniform"])
def test_steps_within_a_budget(ctx, kind):
    """The layers without a window see what their caches hold: rows appended under their text's positions, weighed by
    every layer that reads them, cut when there is no room; the others are as without a budget."""
    kw = dict(reserve=40, seed=91, embed=True, kv="fp4")
    d = BatchDecoder(ctx, LENS, shape(kind), budget=40, slack=6, sinks=2, recent=8, **kw)
    d.fill_kv(seed=92)
    s, B = d.s, d.B
    lens, cached = np.array(LENS), np.minimum(LENS, 40)
    rng = np.random.default_rng(93)
    cuts = 0
    for step in range(20):
        d.tokens.upload(rng.integers(0, s.vocab, B).astype(np.uint32))
        if cached.max() + 1 > 46:
            cached, cuts = np.minimum(cached, 40), cuts + 1
        before = {}
        more = {il: 0.0 for il in d.mass}

        def probe(stage, il, _):
            if stage == "prep" and il < s.n_layers and d._is_cut(il) and s.is_producer(il):
                before[il] = d.mass[il].download(np.float32).astype(np.float64)
            if stage == "attn":
                cut = d._is_cut(il)
                q, got = (x.download(np.float32, B * s.q_dim_of(il)) for x in (d.q, d.attn))
                rows = [(b, b, int((cached if cut else lens)[b])) for b in range(B)]
                check_rows(d, il, q, got, rows)
                if cut:  # every head of every sequence adds one
                    src = s.producer(il)
                    more[src] += B * s.n_q_heads
                    now = d.mass[src].download(np.float32).astype(np.float64)
                    new = [(d.cut_table_host[b, cached[b] // d.page_size], cached[b] % d.page_size) for b in range(B)]
                    old = before[src].reshape(-1, d.page_size, s.n_kv_heads).copy()
                    for at in new:
                        old[at] = 0  # (the append's)
                    assert abs(now.sum() - old.sum() - more[src]) <= 1e-4 * more[src], (step, il)

        d.step(probe=probe)
        lens, cached = lens + 1, cached + 1
        assert np.array_equal(d.cut_lens_host, cached)
    assert cuts >= 2 and np.array_equal(d.cut_lens.download(np.uint32), cached)
    assert np.array_equal(d.seq_lens.download(np.uint32), lens)
    # an eviction by hand, against the oracle
    pool = {il: pools(d, il) for il in d.mass}
    mass = {il: d.mass[il].download(np.float32).reshape(d.cut_pages, d.page_size, s.n_kv_heads) for il in d.mass}
    d.evict()
    for il in d.mass:
        k, v = pool[il]
        kept, after = K4.evict(k, v, mass[il], d.cut_table_host, cached, 40, 2, 8, d.cut_rows)
        assert np.array_equal(d.kept[il].download(np.int32).reshape(kept.shape), kept)
        now = pools(d, il)
        assert np.array_equal(now[0].codes, k.codes) and np.array_equal(now[1].scale, v.scale)
        assert np.array_equal(d.mass[il].download(np.float32).reshape(mass[il].shape), mass[il])
    assert np.array_equal(d.cut_lens.download(np.uint32), after) and np.array_equal(d.cut_lens_host, after)


@pytest.mark.parametrize("B,T", [(16, 100), (16, 40), (64, 700)])
def test_a_prompt_longer_than_its_budget(ctx, B, T):
    """Passes and chunks of a prompt cut the cache between them; the text goes on token by token, and another begins."""
    d = BatchDecoder(ctx, [0] * B, shape(), seed=95, reserve=T + 60, shared_pages=True, embed=True, kv="fp4", budget=48,
                     slack=80, sinks=3)
    s, il = d.s, 3  # a global layer that reads the cache of layer 1
    assert d.cut["recent"] == 12
    rng = np.random.default_rng(96)
    for turn in range(2):
        toks = rng.integers(0, s.vocab, T).astype(np.uint32)
        last = d.prefill(toks)
        assert d.text == T and np.isfinite(d.logits.download(np.float32)).all()
        cached = int(d.cut_lens.download(np.uint32)[0])
        assert cached == d.cut_lens_host[0] and (cached <= 128 if T > 48 else cached == T)
        for i in range(40):
            seen = []

            def probe(stage, il, _):
                if stage == "attn":
                    at = int(d.cut_lens_host[0]) - 1 if d._is_cut(il) else T + i
                    check_rows(d, il, d.q.download(np.float32, B * s.q_dim_of(il)),
                               d.attn.download(np.float32, B * s.q_dim_of(il)), [(0, 0, at)])
                    seen.append(il)

            d.prefill(d.tokens.download(np.uint32)[last:last + 1], T + i, probe=probe)
            last = 0
            assert len(seen) == s.n_layers
            now = int(d.cut_lens_host[0])
            assert now == (cached + 1 if cached < 128 else 49)
            cached = now
    with pytest.raises(ValueError, match="go on at"):
        d.prefill([1, 2], 5)
    assert d.score(rng.integers(0, s.vocab, 60)).shape == (59,) and d.text == 59


@pytest.mark.parametrize("budget,slack,goes_on", [(200, 64, 40), (24, 24, 56)])
def test_a_prompt_that_fails_half_way(ctx, budget, slack, goes_on):
    """Its second chunk raises between two layers. What is made again leaves every bit as if nothing had failed: from the
    prompt's begin, or from behind the eviction that its second chunk made."""
    toks = np.random.default_rng(97).integers(0, 4096, 80).astype(np.uint32)
    chunks = []

    def fails(stage, il, _):
        if stage == "prep" and il == 0:
            chunks.append(il)
        if stage == "attn" and il == 2 and len(chunks) == 2:
            raise RuntimeError("half way")

    runs = []
    for broken in (False, True):
        d = BatchDecoder(ctx, [0] * 16, shape(), seed=98, reserve=100, shared_pages=True, embed=True, kv="fp4",
                         budget=budget, slack=slack)
        d.prefill(toks[:40], probe=lambda *a: None)
        at = 40
        if broken:
            with pytest.raises(RuntimeError, match="half way"):
                d.prefill(toks[40:], 40, probe=fails)
            at = d.text
            assert at == goes_on and np.array_equal(d.cut_lens.download(np.uint32), d.cut_lens_host)
        for a, b in ((40, goes_on), (goes_on, 80)):
            if at <= a < b:
                d.prefill(toks[a:b], a, probe=lambda *a: None)
        n = int(d.cut_lens_host[0])
        live = (d.cut_table_host[0, np.arange(n) // 16], np.arange(n) % 16)
        runs.append([d.logits.download(np.uint32), d.cut_lens.download(np.uint32)] +
                    [m.download(np.uint32).reshape(d.cut_pages, 16, -1)[live] for m in d.mass.values()] +
                    [x[live] for il in d.mass for p in pools(d, il) for x in (p.codes, p.scale)])
    assert all(np.array_equal(a, b) for a, b in zip(*runs))


def test_refusals(ctx):
    s = shape()
    for kw in (dict(kv="int8", budget=40), dict(budget=40), dict(kv="fp4", budget=0), dict(kv="fp4", budget=40, slack=0),
               dict(kv="fp4", budget=40, sinks=41, recent=0), dict(kv="fp4", budget=40, sinks=10, recent=31),
               dict(kv="fp4", budget=40, sinks=-1), dict(kv="fp4", budget=40, recent=-1),
               dict(kv="fp4", budget=40, slack=15, shared_pages=True)):
        with pytest.raises(ValueError, match="budget|slack"):
            BatchDecoder(ctx, [0] * 16, s, **kw)
    d = BatchDecoder(ctx, [0] * 16, s, reserve=64, shared_pages=True, embed=True, kv="fp4")
    for call in (d.step, d.capture, d.evict, lambda: d.score([1]), lambda: d.prefill([])):
        with pytest.raises(ValueError):
            call()
    assert d.prefill([1, 2, 3]) == 2
