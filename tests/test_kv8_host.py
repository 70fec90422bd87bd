"""The host's part of prompts and texts over 8-bit shared pages, without a device: what each step finds in the
buffers that place it, when the host waits, and what a call that fails leaves."""
from types import SimpleNamespace

import numpy as np
import pytest

from g4hip.decoder import BatchDecoder


class Buf:
    def __init__(self, ctx, mem):
        self.ctx, self.mem, self.nbytes = ctx, mem, mem.size

    def offset(self, n):
        return Buf(self.ctx, self.mem[n:])

    def upload(self, a, offset=0):
        self.ctx.waits += 1  # (an upload waits for the stream)
        a = np.ascontiguousarray(a).view(np.uint8).reshape(-1)
        self.mem[offset:offset + a.size] = a
        return self

    def download(self, dtype, count=None):
        self.ctx.waits += 1
        return self.mem.view(dtype)[:count].copy()

    def free(self):
        pass


class Ctx:
    """A device of host memory; every call that makes the host wait is counted."""

    def __init__(self):
        self.waits = 0

    def alloc(self, n):
        return Buf(self, np.zeros(n, np.uint8))

    def empty(self, n, dtype):
        return self.alloc(n * np.dtype(dtype).itemsize)

    def from_numpy(self, a):
        return self.alloc(a.nbytes).upload(a)

    def copy(self, dst, src, n):
        dst.mem[:n] = src.mem[:n]

    def sync(self):
        self.waits += 1

    def logprobs_workspace_bytes(self, *a):
        return 16

    def logprobsBatch(self, *a, **k):
        pass

    batchPrep = repeatRow = logprobsBatch


def decoder(B=4, wide_rows=0, fail_at=None):
    """Steps note what they find: tokens, lengths, the sequence's length and rows, and the waits so far."""
    d = BatchDecoder.__new__(BatchDecoder)
    c = d.ctx = Ctx()
    d.B, d.kv8, d.shared_pages, d.max_seq, d.wide_rows, d.ntop = B, True, True, 1000, wide_rows, None
    d.s = SimpleNamespace(vocab=10, ple_dim=0, hidden=8, eps=1e-6)
    d.embedding = d.lm_head = d.final_norm = d.xn = d.xops = d.logits = object()
    d.span, d.span_rows = c.alloc(12), 0
    d.tokens, d.seq_lens, d.hidden = c.alloc(4 * B), c.alloc(4 * B), c.alloc(32 * B)
    d.seen = []

    def note(tokens, lens):
        if fail_at == len(d.seen):
            raise RuntimeError("a step that fails")
        d.seen.append((tokens.mem.view(np.uint32).tolist(), lens.mem.view(np.uint32).tolist(),
                       d.span.mem.view(np.uint32).tolist(), d.span_rows, c.waits))

    d._wide_buffers = lambda rows: setattr(d, "wide", {"hidden": c.alloc(32 * wide_rows)})
    d._wide_pass = lambda tokens, lens, n, end: note(tokens.offset(0), lens.offset(0))
    d._head = lambda *a: None
    d.step = lambda *a, **k: note(d.tokens, d.seq_lens)
    return d


def test_chunks_of_a_prompt():
    d = decoder()
    toks = np.arange(100, 111)
    assert d.prefill(toks, 5) == 2
    assert [x[:4] for x in d.seen] == [
        ([100, 101, 102, 103], [5, 6, 7, 8], [9, 0, 4], 4),
        ([104, 105, 106, 107], [9, 10, 11, 12], [13, 0, 4], 4),
        ([108, 109, 110, 110], [13, 14, 15, 15], [16, 0, 3], 3)]
    assert d.span_rows == 0


def test_passes_of_a_long_prompt():
    d = decoder(wide_rows=8)
    assert d.prefill(np.arange(19), 5) == 2
    assert [x[2:4] for x in d.seen] == [([13, 0, 8], 8), ([21, 0, 8], 8), ([24, 0, 3], 3)]
    assert d.span_rows == 0


def test_chunks_of_a_text():
    d = decoder()
    assert d.score(np.arange(100, 111), 5).shape == (10,)
    assert [x[:4] for x in d.seen] == [
        ([100, 101, 102, 103], [5, 6, 7, 8], [9, 0, 4], 4),
        ([104, 105, 106, 107], [9, 10, 11, 12], [13, 0, 4], 4),
        ([108, 109, 109, 109], [13, 14, 14, 14], [15, 0, 2], 2)]
    assert d.span_rows == 0


CALLS = [(0, lambda d: d.prefill(np.arange(11), 5)), (8, lambda d: d.prefill(np.arange(19), 5)),
         (0, lambda d: d.score(np.arange(11), 5))]
NAMES = ["chunks", "passes", "text"]


@pytest.mark.parametrize("wide_rows,call", CALLS, ids=NAMES)
def test_a_step_that_fails_leaves_no_rows_placed(wide_rows, call):
    """A step without placed rows is refused: it would append over the failed one's."""
    d = decoder(wide_rows=wide_rows, fail_at=1)
    with pytest.raises(RuntimeError, match="fails"):
        call(d)
    assert d.span_rows == 0
    with pytest.raises(ValueError, match="shared pages"):
        BatchDecoder.step(d)


@pytest.mark.parametrize("wide_rows,call", CALLS, ids=NAMES)
def test_no_wait_between_steps(wide_rows, call):
    """What places the steps goes up before the first; they run back to back, as over f16 pages."""
    d = decoder(wide_rows=wide_rows)
    call(d)
    assert len(d.seen) == 3 and len({x[4] for x in d.seen}) == 1, [x[4] for x in d.seen]


def test_a_workspace_that_could_not_grow_is_asked_for_again():
    """The old one is given back before the larger one is asked for; without either, the next call gets its own."""
    d, sizes, asked = decoder(), {"long": 100, "short": 40}, []
    d.attn8_ws, d.attn8_cap = d.ctx.alloc(60), 60

    def alloc(n):
        asked.append(n)
        if n == 100:
            raise MemoryError
        return Buf(d.ctx, np.zeros(n, np.uint8))

    d.ctx.alloc, d.ctx.attn8_workspace_bytes = alloc, sizes.get
    with pytest.raises(MemoryError):
        d._attn8_workspace(["long"])
    d._attn8_workspace(["short"])
    assert asked == [100, 40] and d.attn8_ws.nbytes == d.attn8_cap == 40


@pytest.mark.parametrize("n", [-1, 65])
def test_alternatives_that_no_call_gives_are_refused(n):
    """Before anything is allocated for them."""
    with pytest.raises(ValueError, match="logprobs"):
        BatchDecoder(None, [3], kv="int8", logprobs=n)


@pytest.mark.parametrize("wide_rows,call", [(0, lambda d: d.prefill(np.arange(11), -3)),
                                            (8, lambda d: d.prefill(np.arange(19), -1)),
                                            (0, lambda d: d.score(np.arange(11), -3))], ids=NAMES)
def test_positions_before_the_first_are_refused(wide_rows, call):
    d = decoder(wide_rows=wide_rows)
    with pytest.raises(ValueError, match="from -"):
        call(d)
    d.kv8 = False
    with pytest.raises(ValueError, match="from -"):
        call(d)
    assert not d.seen
