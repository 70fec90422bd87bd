"""The ragged step, batched prefill and scoring over 8-bit pages.

Every layer's attention is held to float64 over the device's own roped q and the
pages' values (tolerances: test_gpu_kv8's). A row appended to layer 0, whose input
does not depend on the cache, is within half a scale of the f16 decoder's row, and
2^-10 of the row's largest value (the f16 rounding, 2^-11 of a value, and the f32
roundings of the two prologues). Log probabilities are held to float64 over the
device's own logits (tolerances: test_gpu_logprobs's)."""
import numpy as np
import pytest

import kv8_oracle as K8
from g4hip.decoder import BatchDecoder, E2BShape
from gpu_util import bits_equal

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
LENS = [0, 1, 15, 16, 63, 64, 511, 530]


def shape(kind="real"):
    if kind == "uniform":
        return E2BShape(n_layers=2, global_layers=(1,), vocab=4096)
    return E2BShape.real(n_layers=4, n_unshared=2, global_layers=(1, 3), vocab=4096)


def pools(d, il):
    """Layer il's K and V values in float64 and V's scales, as the device holds them."""
    s, L = d.s, d.layers[il]
    dims = (d.num_pages, d.page_size, s.n_kv_heads, s.hd(il))
    out = [K8.Pool(b.download(np.int8).reshape(dims), x.download(np.float32).reshape(d.num_pages, s.n_kv_heads))
           for b, x in zip((L.k_cache, L.v_cache), d.kv_scales[s.producer(il)])]
    return out[0].values(), out[1].values(), out[1].scale


def check_rows(d, il, q, got, rows):
    """rows: (row, its sequence, its position)."""
    s = d.s
    k, v, vs = pools(d, il)
    q, got = (x.reshape(-1, s.n_q_heads, s.hd(il)) for x in (q, got))
    for r, seq, pos in rows:
        want, mag, reach = K8.attend(q[r], k, v, d.page_table_host[seq], pos, 0 if s.is_global(il) else s.window, 1.0)
        pages = d.page_table_host[seq][:pos // d.page_size + 1]
        tol = 6 * U * (8 + reach) * mag + 2.0 ** -40 * (pos + 1) * 127 * vs[pages].max() + 1e-30
        assert (np.abs(got[r] - want) <= tol).all(), (il, r, seq, pos, float((np.abs(got[r] - want) / tol).max()))


def check_logprobs(d, rows):
    V, n = d.s.vocab, d.ntop
    x = d.logits.download(np.float32).reshape(d.B, V)
    toks, lp, ent = d.tokens.download(np.uint32), d.token_logprobs.download(np.float32), d.entropy.download(np.float32)
    ids, top = (b.download(t).reshape(d.B, n) for b, t in ((d.top_ids, np.uint32), (d.top_logprobs, np.float32)))
    for r in rows:
        want = K8.logprobs(x[r], int(toks[r]), n)
        m, reach = float(x[r].max()), np.log(V) + 1
        assert np.array_equal(ids[r], want[2]) and toks[r] == ids[r][0], r
        assert abs(lp[r] - want[0]) <= 8 * U * reach and abs(ent[r] - want[1]) <= 32 * U * reach, r
        assert (np.abs(top[r] - want[3]) <= 8 * U * (np.abs(x[r][ids[r]] - m) + reach)).all(), r


@pytest.mark.parametrize("kind,ps", [("real", 16), ("uniform", 64)])
def test_steps(ctx, kind, ps):
    kw = dict(page_size=ps, reserve=8, seed=41, embed=True)
    d = BatchDecoder(ctx, LENS, shape(kind), kv="int8", logprobs=5, **kw)
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
        check_logprobs(d, range(B))
        L, kv = f.layers[0], s.kv_dim_of(0)
        k, v, _ = pools(d, 0)
        scale = [x.download(np.float32) for x in d.kv_scales[0]]
        for val, b16, sc in ((k, L.k_cache, scale[0]), (v, L.v_cache, scale[1])):
            b16 = b16.download(np.float16).reshape(-1, kv)
            for b in range(B):
                page = d.page_table_host[b, lens[b] // ps]
                row, r16 = val[page, lens[b] % ps].reshape(-1), b16[f.pool_row(b, int(lens[b]))].astype(np.float64)
                assert np.abs(row - r16).max() <= 0.5 * sc[page] + 2.0 ** -10 * np.abs(r16).max(), (step, b)
    assert np.array_equal(d.seq_lens.download(np.uint32), np.array(LENS) + 3)


def test_a_captured_step_equals_eager_ones(ctx):
    runs = []
    for captured in (False, True):
        d = BatchDecoder(ctx, LENS, shape(), seed=51, reserve=24, embed=True, kv="int8", logprobs=3)
        d.fill_kv(seed=52)
        d.tokens.upload(np.arange(d.B, dtype=np.uint32))
        g = d.capture() if captured else None
        got = []
        for _ in range(20):  # (over a page's end)
            if captured:
                ctx.graph_launch(g)
            else:
                d.step()
            got.append([b.download(np.uint32) for b in (d.tokens, d.logits, d.token_logprobs, d.entropy, d.top_ids,
                                                        d.top_logprobs)])
        got.append([b.download(np.uint8) for L in d.layers for b in (L.k_cache, L.v_cache)])
        got.append([b.download(np.uint32) for p in d.kv_scales.values() for b in p])
        runs.append(got)
        if captured:
            ctx.graph_destroy(g)
    for step, (a, b) in enumerate(zip(*runs)):
        assert all(np.array_equal(x, y) for x, y in zip(a, b)), step


@pytest.mark.parametrize("kind", ["real", "uniform"])
@pytest.mark.parametrize("T,start", [(1, 0), (5, 0), (16, 0), (20, 0), (21, 40), (3, 37)])
def test_prefill_in_chunks(ctx, kind, T, start):
    d = BatchDecoder(ctx, [0] * 16, shape(kind), seed=61, reserve=start + T + 8, shared_pages=True, embed=True,
                     kv="int8", logprobs=4)
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
    check_logprobs(d, range(B))
    H = d.hidden.download(np.float32).reshape(B, s.hidden)
    assert all(bits_equal(H[r], H[last]) for r in range(last + 1, B))


@pytest.mark.parametrize("T,start", [(5, 0), (16, 3), (20, 40)])
def test_a_short_prompt_leaves_rows_out(ctx, T, start):
    d = BatchDecoder(ctx, [0] * 64, shape(), seed=65, reserve=128, shared_pages=True, embed=True, kv="int8", logprobs=4)
    d.fill_kv(seed=66)
    toks = np.random.default_rng(67).integers(0, d.s.vocab, T).astype(np.uint32)
    assert d.prefill(toks, start) == T - 1
    il, s = d.s.n_layers - 1, d.s
    n = T * s.q_dim_of(il)
    check_rows(d, il, d.q.download(np.float32, n), d.attn.download(np.float32, n),
               [(r, 0, start + r) for r in range(T)])
    check_logprobs(d, range(64))


@pytest.mark.parametrize("kind,B,T,start", [("real", 16, 100, 0), ("real", 64, 700, 0), ("uniform", 64, 201, 100),
                                            ("uniform", 16, 97, 530), ("real", 1, 33, 3)])
def test_prefill_many_rows_a_pass(ctx, kind, B, T, start):
    d = BatchDecoder(ctx, [0] * B, shape(kind), seed=71, reserve=start + T + 80, shared_pages=True, embed=True,
                     kv="int8", logprobs=4)
    d.fill_kv(seed=72)
    s, il = d.s, d.s.n_layers - 1
    toks = np.random.default_rng(73).integers(0, s.vocab, T).astype(np.uint32)
    last = d.prefill(toks, start)
    assert d.wide_cap >= T  # (all rows in one pass)
    n = s.q_dim_of(il) * T
    rows = sorted({0, 1, 15, 16, 63, T // 2, T - 2, T - 1} & set(range(T)))
    check_rows(d, il, d.wide["q"].download(np.float32, n), d.wide["attn"].download(np.float32, n),
               [(r, 0, start + r) for r in rows])
    check_logprobs(d, range(B))
    H = d.hidden.download(np.float32).reshape(B, s.hidden)
    assert all(bits_equal(H[r], H[last]) for r in range(last + 1, B))
    # the next tokens of the same sequence, one at a time
    for i in range(3):
        seen = []

        def probe(stage, il, _):
            if stage == "attn":
                check_rows(d, il, d.q.download(np.float32, B * s.q_dim_of(il)),
                           d.attn.download(np.float32, B * s.q_dim_of(il)), [(0, 0, start + T + i)])
                seen.append(il)

        assert d.prefill(d.tokens.download(np.uint32)[last:last + 1], start + T + i, probe=probe) == 0
        last = 0
        assert len(seen) == s.n_layers


@pytest.mark.parametrize("kv", ["int8", "f16"])
def test_score(ctx, kv):
    d = BatchDecoder(ctx, [0] * 16, shape(), seed=81, reserve=64, shared_pages=True, embed=True, kv=kv)
    d.fill_kv(seed=82)
    toks = np.random.default_rng(83).integers(0, d.s.vocab, 22).astype(np.uint32)
    got = d.score(toks, 5)
    assert got.shape == (21,)
    want = []
    for first, n in ((0, 16), (16, 5)):  # the same chunks again, one call each
        d.prefill(toks[first:first + n], 5 + first)
        want.append(d.logits.download(np.float32).reshape(16, -1)[:n])
    for i, x in enumerate(np.concatenate(want)):
        ref = K8.logprobs(x, int(toks[i + 1]), 0)[0]
        assert abs(got[i] - ref) <= 8 * U * (abs(float(x[toks[i + 1]]) - float(x.max())) + np.log(x.size) + 1), i


def test_log_probabilities_without_alternatives_and_of_a_topk_sample(ctx):
    """A step whose host samples has no token yet: entropy and alternatives only."""
    x = BatchDecoder(ctx, [3, 20], shape(), seed=85, embed=True, kv="int8", logprobs=0)
    y = BatchDecoder(ctx, [3, 20], shape(), seed=85, embed=True, kv="int8", logprobs=6)
    for d in (x, y):
        d.fill_kv(seed=86)
        d.token_logprobs.upload(np.full(2, 7.0, np.float32))
    x.step()
    y.step("topk")
    assert np.all(x.token_logprobs.download(np.float32) < 0) and x.top_ids is None
    assert np.all(y.token_logprobs.download(np.float32) == 7.0)
    assert bits_equal(x.entropy.download(np.float32), y.entropy.download(np.float32))
    assert np.array_equal(y.top_ids.download(np.uint32).reshape(2, 6)[:, 0], x.tokens.download(np.uint32))


def test_refusals(ctx):
    s = shape()
    with pytest.raises(ValueError):
        BatchDecoder(ctx, [0], s, kv="int4")
    with pytest.raises(ValueError):
        BatchDecoder(ctx, [0], s, lm_head=False, logprobs=3)
    d = BatchDecoder(ctx, [0] * 16, s, reserve=64, shared_pages=True, embed=True, kv="int8")
    for call in (d.step, d.capture, lambda: d.score([1]), lambda: d.score(np.zeros(64, np.uint32)),
                 lambda: d.prefill([]), lambda: d.prefill(np.zeros(64, np.uint32))):
        with pytest.raises(ValueError):
            call()
    assert d.prefill([1, 2, 3]) == 2
    with pytest.raises(ValueError):
        d.step()


def test_fewer_rows_than_the_decoder_has_at_a_large_vocabulary(ctx):
    """A short prompt and a text's last rows take the log probabilities of fewer rows, whose launch holds fewer values
    a thread and leaves more partials a row."""
    s = E2BShape.real(n_layers=4, n_unshared=2, global_layers=(1, 3), vocab=128256)
    d = BatchDecoder(ctx, [0] * 40, s, seed=91, reserve=160, shared_pages=True, embed=True, kv="int8", logprobs=4)
    d.fill_kv(seed=92)
    toks = np.random.default_rng(93).integers(0, s.vocab, 61).astype(np.uint32)
    for T in (12, 25):  # 16 and 32 rows of the 40
        assert d.prefill(toks[:T]) == T - 1
        check_logprobs(d, range(40))
    got = d.score(toks, 3)
    assert got.shape == (60,)
    last = d.logits.download(np.float32).reshape(40, -1)[:20]  # what the second pass left
    d.prefill(toks[:40], 3)
    for i, x in enumerate(np.concatenate([d.logits.download(np.float32).reshape(40, -1), last])):
        ref = K8.logprobs(x, int(toks[i + 1]), 0)[0]
        assert abs(got[i] - ref) <= 8 * U * (abs(float(x[toks[i + 1]]) - float(x.max())) + np.log(x.size) + 1), i
