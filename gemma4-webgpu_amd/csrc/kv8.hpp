// kv8.hpp — what the kernels of the 8-bit paged K/V pool share: a call's rows
// by sequence (g4_kv8_params in g4hip.h).
#pragma once
#include "g4_internal.hpp"

namespace g4kv8 {

// The rows of a call: which are sequence s's, and where they stand in it.
struct Rows {
  const uint32_t* seq_lens;
  const uint32_t* row_starts;  // or null: row s is sequence s's only one
  uint32_t num_seqs, num_rows, max_rows, max_seq_len;
};
struct Seq {
  uint32_t first, n;  // its rows: first .. first + n - 1 (n = 0: none, or starts that do not hold)
  uint32_t base;      // position of its first row
  uint32_t len;       // its length; 0 where the rows do not fit into it
};
__device__ __forceinline__ Seq seq_rows(const Rows& r, uint32_t s) {
  Seq q{s, 1, 0, 0};
  const uint32_t L = r.seq_lens[s];  // (all three on their way at once)
  if (r.row_starts) {
    const uint32_t a = r.row_starts[s], b = r.row_starts[s + 1];
    q.first = a;
    q.n = b >= a && b <= r.num_rows && b - a <= r.max_rows ? b - a : 0u;
  }
  if (q.n > 0 && L >= q.n && L <= r.max_seq_len) {
    q.len = L;
    q.base = L - q.n;
  }
  return q;
}
// The sequence that holds row r (num_seqs: none).
__device__ __forceinline__ uint32_t seq_of_row(const Rows& r, uint32_t row) {
  if (!r.row_starts) return row;
  uint32_t lo = 0, hi = r.num_seqs;  // the last s with row_starts[s] <= row
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (r.row_starts[mid] <= row) lo = mid;
    else hi = mid;
  }
  return r.row_starts[lo] <= row && row < r.row_starts[lo + 1] ? lo : r.num_seqs;
}

}  // namespace g4kv8

// Checks of the pool's and the rows' shape (k_kv8.hip).
int g4_internal_kv8_check(const char* fn, const g4_kv8_params& p, const uint32_t* row_starts);
