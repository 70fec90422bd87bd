"""The layout of the eviction's keys in LDS (csrc/kv4_keys.hpp), listed by a host program: a group's candidates are each
some wave's, in order, and no wave's keys of any group lie where another's of any group do, so that a wave may fetch the
next group's while others still read the last one's."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gemma4-webgpu_amd", "csrc")
PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "kv4_keys.hpp"
int main(int argc, char** argv) {
  for (int i = 1; i < argc; ++i) {
    const g4kv4::Keys k{(uint32_t)strtoul(argv[i], nullptr, 10)};
    for (uint32_t g = 0; g < k.groups(); ++g)
      for (uint32_t w = 0; w < k.THREADS / 64; ++w)
        printf("%u %u %u %u %u %u %u\n", k.n, g, w, k.rows(g), k.first(g, w), k.place(w), 64 * k.each(g));
  }
}
"""
COUNTS = [1, 63, 1024, 1025, 32767, 32768, 32769, 33000, 33792, 33995, 40000, 60000, 65536, 69997, 98305, 1000003]


@pytest.fixture(scope="module")
def layout(tmp_path_factory):
    d = tmp_path_factory.mktemp("keys")
    (d / "keys.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-I", CSRC, str(d / "keys.cpp"), "-o", str(d / "keys")], check=True)
    out = subprocess.run([str(d / "keys"), *map(str, COUNTS)], check=True, capture_output=True, text=True).stdout
    got = {n: [] for n in COUNTS}
    for line in out.splitlines():
        n, *rest = map(int, line.split())
        got[n].append(rest)
    return got


@pytest.mark.parametrize("n", COUNTS)
def test_every_candidate_is_in_one_group_and_wave(layout, n):
    groups = {}
    for g, w, rows, first, _, count in layout[n]:
        assert first == groups.setdefault(g, [0, rows])[0] and w == first // max(count, 1)
        groups[g][0] += count
    assert sorted(groups) == list(range(-(-n // 32768))) and sum(rows for _, rows in groups.values()) == n
    assert all(upto >= rows for upto, rows in groups.values())


@pytest.mark.parametrize("n", COUNTS)
def test_no_wave_has_keys_where_another_has(layout, n):
    """Between the groups of a selection nothing waits for the other waves."""
    for _, wave, _, _, place, count in layout[n]:
        assert place + count <= 32768  # (the array's)
        for _, other, _, _, at, many in layout[n]:
            assert wave == other or place + count <= at or at + many <= place, (wave, other)
