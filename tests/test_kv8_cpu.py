"""Shape checks of the 8-bit pool and the log probabilities that need no GPU."""
import ctypes

import pytest

from g4hip import _lib


def size(**change):
    f = dict(num_seqs=2, num_q_heads=8, num_kv_heads=1, head_dim=256, page_size=16, max_pages=4, max_seq_len=64,
             num_pages=9, num_rows=2, max_rows=1, sliding_window=0, scale=1.0, eps=1e-6, theta=1e4, apply_divisor=0)
    n = ctypes.c_size_t()
    rc = _lib.lib().g4_pagedAttn8_workspace_size(_lib.Kv8Params(**{**f, **change}), ctypes.byref(n))
    return rc, n.value


def test_attention_workspace_sizes():
    rc, n = size()
    assert rc == 0 and 0 < n < 1 << 30
    assert size(num_rows=40, max_rows=33)[0] == 0
    assert size(max_seq_len=1, max_pages=1, num_seqs=1, num_rows=1)[0] == 0


@pytest.mark.parametrize("change", [
    dict(num_q_heads=7, num_kv_heads=2), dict(num_q_heads=17), dict(num_q_heads=65, num_kv_heads=65),
    dict(num_q_heads=0), dict(num_kv_heads=0), dict(head_dim=96), dict(head_dim=0), dict(page_size=24),
    dict(page_size=0), dict(page_size=2048), dict(max_seq_len=65), dict(max_seq_len=0), dict(max_pages=0),
    dict(num_seqs=0), dict(num_seqs=65536, num_rows=65536), dict(num_rows=0), dict(max_rows=0),
    dict(num_rows=70000, max_rows=70000), dict(num_rows=2, max_rows=3), dict(num_pages=0),
    dict(num_pages=1 << 31)])
def test_shapes_that_are_refused(change):
    assert size(**change)[0] == -1


def test_logprobs_workspace_sizes():
    n = ctypes.c_size_t()
    f = _lib.lib().g4_logprobsBatch_workspace_size
    assert f(262144, 64, 20, ctypes.byref(n)) == 0 and 0 < n.value < 1 << 28
    for bad in ((0, 1, 0), ((1 << 28) + 1, 1, 0), (10, 0, 0), (10, 65536, 0), (10, 1, 11), (100, 1, 65)):
        assert f(*bad, ctypes.byref(n)) == -1
    assert f(10, 1, 1, None) == -1


def test_a_pool_of_too_many_positions_is_refused():
    big = dict(page_size=1024, max_seq_len=1024, max_pages=1)
    assert size(num_pages=(1 << 26) - 1, **big)[0] == 0
    assert size(num_pages=1 << 26, **big)[0] == -1


@pytest.mark.parametrize("ntop", [0, 5, 64])
@pytest.mark.parametrize("vocab", [64, 4096, 32003, 100003, 128256, 262144])
def test_a_logprobs_workspace_serves_fewer_rows(vocab, ntop):
    """A decoder sizes it for all its rows; a short prompt and a text's last rows are fewer."""
    f, n, most = _lib.lib().g4_logprobsBatch_workspace_size, ctypes.c_size_t(), 0
    for rows in [*range(1, 70), 127, 128, 500, 511, 512, 513, 2000, 65535]:
        assert f(vocab, rows, ntop, ctypes.byref(n)) == 0
        assert n.value >= most, (rows, n.value, most)
        most = n.value
