"""Shape checks of the 4-bit pool, its eviction and the oracle's rounding that need no GPU."""
import ctypes

import numpy as np
import pytest

import kv4_oracle as K4
from g4hip import _lib

GOOD = dict(num_seqs=2, num_q_heads=8, num_kv_heads=1, head_dim=256, page_size=16, max_pages=4, max_seq_len=64,
            num_pages=9, num_rows=2, max_rows=1, sliding_window=0, scale=1.0, eps=1e-6, theta=1e4, apply_divisor=0)


def size(with_mass=0, **change):
    n = ctypes.c_size_t()
    rc = _lib.lib().g4_pagedAttn4_workspace_size(_lib.Kv4Params(**{**GOOD, **change}), with_mass, ctypes.byref(n))
    return rc, n.value


def evict_size(keep, **change):
    n = ctypes.c_size_t()
    rc = _lib.lib().g4_kvEvict4_workspace_size(_lib.Kv4Params(**{**GOOD, **change}), keep, ctypes.byref(n))
    return rc, n.value


def test_attention_workspace_sizes():
    for mass in (0, 1):
        rc, n = size(mass)
        assert rc == 0 and 0 < n < 1 << 30
        assert size(mass, num_rows=40, max_rows=33)[0] == 0
        assert size(mass, max_seq_len=1, max_pages=1, num_seqs=1, num_rows=1)[0] == 0
    assert size(1)[1] >= size(0)[1]


@pytest.mark.parametrize("change", [
    dict(num_q_heads=7, num_kv_heads=2), dict(num_q_heads=17), dict(num_q_heads=65, num_kv_heads=65),
    dict(num_q_heads=0), dict(num_kv_heads=0), dict(head_dim=96), dict(head_dim=0), dict(page_size=24),
    dict(page_size=0), dict(page_size=2048), dict(max_seq_len=65), dict(max_seq_len=0), dict(max_pages=0),
    dict(num_seqs=0), dict(num_seqs=65536, num_rows=65536), dict(num_rows=0), dict(max_rows=0),
    dict(num_rows=70000, max_rows=70000), dict(num_rows=2, max_rows=3), dict(num_pages=0),
    dict(num_pages=1 << 31)])
def test_shapes_that_are_refused(change):
    assert size(0, **change)[0] == -1 and size(1, **change)[0] == -1


def test_weights_of_prompts_that_no_launch_numbers_are_refused():
    """Four threads a position of the longest cache, fewer than 2^32 in all; without weights, or of few rows, 2^30
    positions are taken. Before anything is launched."""
    far = dict(num_seqs=1, page_size=1024, max_pages=1 << 20, num_pages=1 << 20, num_rows=40, max_rows=40)
    assert size(1, **far, max_seq_len=1 << 30)[0] == -1
    assert size(0, **far, max_seq_len=1 << 30)[0] == size(1, **far, max_seq_len=(1 << 30) - 256)[0] == 0
    assert size(1, **far, max_seq_len=1 << 30, sliding_window=1 << 20)[0] == 0
    assert size(1, **{**far, "num_rows": 2, "max_rows": 2}, max_seq_len=1 << 30)[0] == 0


def test_eviction_workspace_sizes():
    rc, n = evict_size(64)
    assert rc == 0 and 0 < n < 1 << 20
    assert evict_size(1)[0] == 0 and evict_size(64, num_rows=0, max_rows=0, num_q_heads=3)[0] == 0
    assert evict_size(0)[0] == evict_size(65)[0] == -1
    for bad in (dict(num_kv_heads=65), dict(num_kv_heads=0), dict(head_dim=96), dict(page_size=24), dict(num_seqs=0)):
        assert evict_size(10, **bad)[0] == -1


def test_the_oracle_rounds_to_the_nearest_code():
    y = np.concatenate([np.linspace(-7, 7, 4001), K4.BORDERS, -K4.BORDERS, K4.LEVELS])
    x = np.zeros((len(y), 32))
    x[:, 0], x[:, 1] = 7, y  # a scale of 1
    codes, scale, _ = K4.encode(x)
    assert np.all(scale == 127)
    got = K4.VALUES[codes[:, 1]]
    best = np.abs(K4.LEVELS[:, None] - np.abs(y)).min(0)
    assert np.array_equal(np.abs(np.abs(got) - np.abs(y)), best) and np.all(got * y >= 0)
    # halves go to the even code
    assert [int(c & 7) for c in codes[4001:4008, 1]] == [0, 2, 2, 4, 4, 6, 6]


@pytest.mark.parametrize("top,byte", [(7.0, 127), (7.0000001, 128), (3.5, 126), (3.6, 127), (6.0, 127), (0.0, 107),
                                      (2.0 ** -40, 107), (7 * 2.0 ** -20, 107), (7.1 * 2.0 ** -20, 108), (8.0, 128)])
def test_the_oracle_takes_the_least_scale(top, byte):
    x = np.zeros((1, 64))
    x[0, 40] = -top
    assert list(K4.encode(x)[1][0]) == [107, byte]
    v = K4.values(*K4.encode(x)[:2])
    assert abs(v[0, 40] + top) <= 2.0 ** (byte - 127)


def test_the_oracle_keeps_the_heaviest_rows_the_first_of_equal_ones():
    m = np.array([5, 0, 1, 1, 9, 1, np.nan, -4, 0], np.float32)
    assert list(K4.chosen(m, 0, 0, 4)) == [0, 2, 3, 4]
    assert list(K4.chosen(m, 2, 1, 5)) == [0, 1, 2, 4, 8]
    assert list(K4.chosen(m, 0, 0, 8)) == [0, 1, 2, 3, 4, 5, 6, 7]
    assert list(K4.chosen(m, 3, 3, 6)) == [0, 1, 2, 6, 7, 8]
