"""The host's part of a budget of rows, without a device: when caches are cut, what their lengths are, and that nothing
is decided while a step is captured."""
import numpy as np
import pytest

from g4hip.decoder import BatchDecoder
from test_kv8_host import Buf, Ctx, decoder


class Lens(Buf):
    def zero(self):
        self.mem[:] = 0


class CutCtx(Ctx):
    def __init__(self):
        super().__init__()
        self.cuts = []

    def kvEvict4(self, k, v, ks, vs, mass, table, lens, p, keep, first, recent, kept, ws):
        self.cuts.append((p, lens.mem.view(np.uint32).tolist()))
        x = lens.mem.view(np.uint32)
        x[:] = np.minimum(x, keep)

    def advanceSeqLens(self, lens, n, by):
        lens.mem.view(np.uint32)[:n] += by


def with_budget(d, lens, shared, budget=8, slack=4):
    d.ctx.__class__ = CutCtx
    d.ctx.cuts = []
    d.shared_pages, d.kv4, d.budget, d.cut_rows = shared, True, budget, budget + slack
    d.cut = dict(keep=budget, first=1, recent=2)
    d.cut_lens_host = np.array(lens, np.uint32)
    d.cut_lens, d.cut_lens_next = (Lens(d.ctx, np.zeros(4 * len(lens), np.uint8)) for _ in "ab")
    d.cut_lens.upload(d.cut_lens_host)
    d.evict_params, d.evict_ws, d.cut_table, d.text = {1: "one", 3: "three"}, None, None, 0
    d.mass, d.kept = ({1: None, 3: None} for _ in "mk")
    d.kv_scales = {1: (None, None), 3: (None, None)}
    d.layers = {i: type("L", (), dict(k_cache=None, v_cache=None)) for i in (1, 3)}
    return d


def lens_of(d):
    got = d.cut_lens.mem.view(np.uint32).tolist()
    assert got == d.cut_lens_host.tolist()
    return got


def test_caches_are_cut_where_a_step_finds_no_room():
    d = with_budget(decoder(), [11, 3], False)
    d._make_room(1)
    assert lens_of(d) == [12, 4] and not d.ctx.cuts
    d._make_room(1)  # (13 rows do not fit): every layer of the same lengths
    assert d.ctx.cuts == [("one", [12, 4]), ("three", [12, 4])] and lens_of(d) == [9, 5]
    for n in (10, 11, 12):
        d._make_room(1)
        assert lens_of(d)[0] == n
    assert len(d.ctx.cuts) == 2


def test_a_captured_step_decides_nothing():
    d = with_budget(decoder(), [12, 3], False)
    d.capturing = True
    d._make_room(1)
    assert not d.ctx.cuts and d.cut_lens_host.tolist() == [12, 3] and d.cut_lens.mem.view(np.uint32).tolist() == [13, 4]
    d.capturing = False
    d.evict()  # what the device holds, whatever the host counted
    assert lens_of(d) == [8, 4]


def test_chunks_of_a_prompt_make_room_for_their_rows():
    d = with_budget(decoder(), [0], True)
    d.prefill(np.arange(100, 118))  # five chunks: 4, 8, 12, cut to 8, 12, cut to 8, 10
    assert [x[1] for x in d.ctx.cuts if x[0] == "one"] == [[12], [12]] and lens_of(d) == [10] and d.text == 18
    d.prefill([1, 2], 18)
    assert lens_of(d) == [12] and d.text == 20
    d.prefill([1, 2, 3])  # another text
    assert lens_of(d) == [3] and d.text == 3
    d.score(np.arange(6), 3)
    assert lens_of(d) == [8] and d.text == 8


@pytest.mark.parametrize("start", [1, 17, 19])
def test_a_text_goes_on_where_it_ended(start):
    d = with_budget(decoder(), [0], True)
    d.prefill(np.arange(18))
    before = lens_of(d), len(d.seen)
    for call in (lambda: d.prefill([1], start), lambda: d.score([1, 2], start)):
        with pytest.raises(ValueError, match="go on at 18"):
            call()
    assert (lens_of(d), len(d.seen)) == before


def test_an_eviction_needs_a_budget():
    with pytest.raises(ValueError, match="budget"):
        decoder().evict()


@pytest.mark.parametrize("kw", [dict(kv="int8", budget=4), dict(budget=4), dict(kv="fp4", budget=0),
                                dict(kv="fp4", budget=4, sinks=3, recent=2), dict(kv="fp4", budget=4, slack=0)])
def test_budgets_that_do_not_hold_are_refused(kw):
    """Before anything is allocated for them."""
    with pytest.raises(ValueError, match="budget"):
        BatchDecoder(None, [3], **kw)


TEXTS = [(0, lambda d, n, start: d.prefill(np.arange(n), start)), (8, lambda d, n, start: d.prefill(np.arange(n), start)),
         (0, lambda d, n, start: d.score(np.arange(n + 1), start))]


def failing(lens, wide_rows, fail_at, **kw):
    """A shared decoder whose step number fail_at raises, and whose steps weigh what is cached."""
    d = with_budget(decoder(wide_rows=wide_rows, fail_at=fail_at), lens, True, **kw)
    mass = Buf(d.ctx, np.zeros(4 * 64, np.uint8))
    d.held_mass = [(Buf(d.ctx, np.zeros(4 * 64, np.uint8)), mass)]
    d.masses = mass.mem.view(np.float32)
    for name in ("step", "_wide_pass"):
        def weighs(*a, run=getattr(d, name), **k):
            d.masses[:int(d.cut_lens_host[0])] += 1
            run(*a, **k)

        setattr(d, name, weighs)
    return d


@pytest.mark.parametrize("wide_rows,call", TEXTS, ids=["chunks", "passes", "text"])
def test_a_prompt_that_fails_leaves_the_caches_as_they_were(wide_rows, call):
    """The rows of its passes so far are gone, what they added to others' masses too; the call can be made again."""
    at = 5 if wide_rows else 3  # (its second pass)
    d = failing([0], wide_rows, at, budget=100)
    call(d, 8, 0)
    while len(d.seen) < at - 1:
        d.seen.append(None)
    want = d.masses[:8].tolist()
    with pytest.raises(RuntimeError, match="fails"):
        call(d, 24, 8)
    assert len(d.seen) == at and d.text == 8 and lens_of(d) == [8] and d.masses[:8].tolist() == want
    with pytest.raises(ValueError, match="go on at 8"):
        call(d, 1, 32)
    d.seen.append(None)
    call(d, 24, 8)
    assert d.text == 32 and lens_of(d) == [32] and d.span_rows == 0


@pytest.mark.parametrize("wide_rows,call", TEXTS, ids=["chunks", "passes", "text"])
def test_a_first_prompt_that_fails_leaves_nothing(wide_rows, call):
    d = failing([0], wide_rows, 1, budget=100)
    with pytest.raises(RuntimeError, match="fails"):
        call(d, 24, 0)
    assert d.text == 0 and lens_of(d) == [0]
    d.seen.append(None)
    call(d, 24, 0)
    assert d.text == 24 and lens_of(d) == [24]


def test_a_prompt_that_fails_behind_an_eviction_goes_on_behind_it():
    """What an eviction took cannot be had back: the passes before it stay."""
    d = failing([0], 0, 4)
    call = TEXTS[0][1]
    call(d, 8, 0)
    with pytest.raises(RuntimeError, match="fails"):
        call(d, 16, 8)  # 12; cut to 8, 12; cut to 8, 12: fails
    assert d.text == 16 and lens_of(d) == [8] and d.masses[:8].tolist() == [4, 4, 4, 4, 3, 3, 3, 3]
    with pytest.raises(ValueError, match="go on at 16"):
        call(d, 1, 8)
    d.seen.append(None)
    call(d, 8, 16)
    assert d.text == 24 and lens_of(d) == [12]


def test_an_eviction_that_fails_leaves_a_text_to_begin_again():
    d = failing([0], 0, None)
    call = TEXTS[0][1]
    call(d, 12, 0)

    def broken(*a):
        raise MemoryError

    d.ctx.kvEvict4 = broken
    with pytest.raises(MemoryError):
        call(d, 4, 12)
    assert d.text == 0 and lens_of(d) == [0]
    with pytest.raises(ValueError, match="go on at 0"):
        call(d, 4, 12)
    del d.ctx.kvEvict4
    call(d, 4, 0)
    assert d.text == 4 and lens_of(d) == [4]


def overrun(lens):
    """A ragged decoder whose captured step was replayed too often; its eviction is the device's: a length past the cache's
    rows stays."""
    d = with_budget(decoder(), lens, False)
    d.launches, d.ctx.launches = 7, 9

    def cut(k, v, ks, vs, mass, table, now, *a):
        x = now.mem.view(np.uint32)
        x[:] = np.where(x > d.cut_rows, x, np.minimum(x, 8))

    d.ctx.kvEvict4 = cut
    return d


@pytest.mark.parametrize("lens,which", [([13, 4], r"1 rows of sequences \[0\]"), ([12, 30], r"18 rows of sequences \[1\]"),
                                        ([14, 13], r"2 rows of sequences \[0, 1\]")])
def test_replays_past_the_room_are_not_hidden(lens, which):
    """A step of the host's raises before it changes anything; evict() says it and leaves caches that have room again."""
    d = overrun(lens)
    before = d.seq_lens.mem.tolist()
    for _ in range(2):
        with pytest.raises(RuntimeError, match=which):
            BatchDecoder.step(d)
        assert d.seq_lens.mem.tolist() == before and d.cut_lens.mem.view(np.uint32).tolist() == lens
    with pytest.warns(RuntimeWarning, match=which):
        d.evict()
    assert lens_of(d) == np.minimum(lens, 8).tolist()
    d._make_room(1)
    assert lens_of(d) == (np.minimum(lens, 8) + 1).tolist()


def test_replays_that_just_fit_are_no_overrun(recwarn):
    d = overrun([12, 3])
    d._make_room(1)
    assert lens_of(d) == [9, 4]
    d = overrun([12, 3])
    d.evict()
    assert lens_of(d) == [8, 3] and not len(recwarn)


def test_lengths_are_read_where_graphs_ran_since():
    """Once after the replays, not at every step for good: a read waits for the device."""
    d = with_budget(decoder(), [3, 2], False)
    d.ctx.launches = 5
    waits = []

    def steps(n):
        for _ in range(n):
            before = d.ctx.waits
            d._make_room(1)
            waits.append(d.ctx.waits - before)

    steps(2)  # (nothing was captured: graphs of others say nothing)
    d.ctx.launches += 1
    steps(1)
    d.ctx.graph_begin = lambda: None
    d.ctx.graph_end = lambda: "graph"
    d.lens_host, d.step = np.zeros(2, np.uint32), lambda sample: d._make_room(1)
    assert d.capture() == "graph"
    d.cut_lens.mem.view(np.uint32)[:] -= np.uint32(1)  # (the capture ran nothing)
    steps(1)
    d.ctx.launches += 2  # two replays
    d.cut_lens.mem.view(np.uint32)[:] += np.uint32(2)
    steps(3)
    assert waits == [0, 0, 0, 0, 1, 0, 0] and lens_of(d) == [12, 11] and not d.ctx.cuts
    steps(1)
    assert waits[-1] == 0 and lens_of(d) == [9, 9] and len(d.ctx.cuts) == 2
    d.ctx.launches += 1
    d.evict()
    steps(1)
    assert waits[-1] == 0


def ragged(lens, budget=8, slack=4):
    d = with_budget(decoder(B=len(lens)), np.minimum(lens, budget), False, budget, slack)
    d.gone = np.array(lens) - d.cut_lens_host
    d.lens_host = np.array(lens, np.uint32)
    return d


def texts(d, n):
    for _ in range(n):
        d._make_room(1)
        d.lens_host = d.lens_host + 1


def test_lengths_set_back_take_the_last_rows_of_the_cut_caches():
    """A sequence that stays keeps what it has, one that loses its last tokens loses their rows, 0 begins another text."""
    d = ragged([5, 8, 20, 3])
    texts(d, 3)  # 8, 11, 23 (11 cached), 6
    d.set_lengths([8, 11, 23, 6])
    assert lens_of(d) == [8, 11, 11, 6] and d.seq_lens.mem.view(np.uint32).tolist() == [8, 11, 23, 6]
    d.set_lengths([6, 9, 21, 0])
    assert lens_of(d) == [6, 9, 9, 0]
    texts(d, 3)
    assert lens_of(d) == [9, 12, 12, 3] and not d.ctx.cuts
    texts(d, 2)  # (cut to 8, 8, 8, 3)
    assert lens_of(d) == [10, 10, 10, 5] and d.ctx.cuts
    d.set_lengths([10, 13, 25, 5])
    assert lens_of(d) == [9, 9, 9, 5]
    d.set_lengths([9, 12, 24, 2])
    assert lens_of(d) == [8, 8, 8, 2]


@pytest.mark.parametrize("lens", [[10, 11, 26, 8], [8, 14, 26, 8], [11, 14, 23, 8], [1, 14, 26, 0]])
def test_lengths_set_back_past_an_eviction_are_refused(lens):
    """Before anything changes: the rows that it left are not those of the shorter text."""
    d = ragged([5, 8, 20, 2])
    texts(d, 6)  # 11, 14, 26 and 8 tokens, of which the evictions took 1, 4, 16 and none
    assert lens_of(d) == [10, 10, 10, 8]
    now = lens_of(d), d.seq_lens.mem.tolist()
    with pytest.raises(ValueError, match="eviction"):
        d.set_lengths(lens)
    assert (lens_of(d), d.seq_lens.mem.tolist()) == now


def test_longer_lengths_count_as_cut():
    d = ragged([5, 20])
    d.set_lengths([7, 100])
    assert lens_of(d) == [7, 8]
    d.set_lengths([9, 0])
    assert lens_of(d) == [8, 0]
    texts(d, 2)
    d.set_lengths([10, 1])
    assert lens_of(d) == [9, 1]


def test_a_steps_bytes_are_those_of_the_rows_it_reads():
    d = ragged([5, 8, 20])
    d.s = type("S", (), dict(n_layers=3, window=6, is_global=lambda self, il: il != 1, kv_dim_of=lambda self, il: 64))()
    row = 2 * 64 * 17 // 32

    def rows():
        assert d.kv_bytes_per_step() % row == 0
        return d.kv_bytes_per_step() // row - sum(min(int(n) + 1, 6) for n in d.lens_host)

    assert rows() == 2 * (6 + 9 + 9)
    texts(d, 3)
    assert rows() == 2 * (9 + 12 + 12)
    texts(d, 1)  # (the next finds no room: each is cut first)
    assert rows() == 2 * (9 + 9 + 9)
    texts(d, 1)
    assert lens_of(d) == [9, 9, 9] and rows() == 2 * (10 + 10 + 10)


def test_a_budget_of_layers_that_all_have_a_window_limits_nothing():
    d = ragged([5, 20])
    d.evict_params, d.launches, d.ctx.launches = {}, 0, 0
    texts(d, 9)
    d.ctx.launches += 9
    texts(d, 9)
    d.evict()
    d.set_lengths([21, 19])
    assert d.seq_lens.mem.view(np.uint32).tolist() == [21, 19] and not d.ctx.cuts
    d = with_budget(decoder(), [0], True)
    d.evict_params = {}
    d.prefill(np.arange(30), 5)
    d.prefill(np.arange(30), 2)
    assert len(d.seen) == 16 and not d.ctx.cuts
