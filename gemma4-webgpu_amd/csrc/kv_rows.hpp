// kv_rows.hpp — a call's new rows of q, k and v as the appends to the 8-bit and
// the 4-bit paged K/V pool form them: split-K parts added up, norm, rotation.
// The norms and the rotation of k and v are in f64 (a value near the border of
// two codes then gets the same code as in exact arithmetic, whatever the order of
// the sums), q's in f32.
#pragma once
#include "kv8.hpp"
#include "mqf_core.hpp"

namespace g4kv8 {

struct RowArgs {
  const float *q, *k, *v;
  uint32_t nparts;
  const uint16_t *q_w, *k_w;
  const uint16_t* rope_freqs;
  const float2* rope_cs;
  float* q_out;
  const int32_t* page_table;
  Rows rows;
  uint32_t nqh, nkh, page_size, max_pages, num_pages;
  float eps, theta;
  uint32_t apply_divisor;
  const uint32_t* positions;  // or null: rows stand in the cache where they stand in the text
  uint32_t most_position;     // that the rotation has
};

// Where a sequence's first new row stands in its text, of which positions[s]
// tokens are known; false where that does not hold its rows or is past the table.
__device__ __forceinline__ bool moved_to(const RowArgs& a, uint32_t s, const Seq& q, uint32_t& first) {
  const uint32_t n = a.positions[s];
  first = n - q.n;
  return n >= q.n && n <= a.most_position;
}

// A lane's share of a row: PP neighbouring pairs (i, i + HD / 2).
template <int HD>
struct Row {
  static constexpr int HALF = HD / 2, PP = HALF >= 64 ? HALF / 64 : 1, ACT = HALF / PP;
};

// Parts added in order, in T; four of them on their way.
template <int HD, typename T>
__device__ __forceinline__ void load_row(const float* p, size_t stride, uint32_t nparts, int lane, T* lo, T* hi) {
  constexpr int PP = Row<HD>::PP, HALF = Row<HD>::HALF;
  typedef float vec __attribute__((ext_vector_type(PP == 1 ? 2 : PP)));  // (PP 1: the second is not used)
#pragma unroll
  for (int i = 0; i < PP; ++i) lo[i] = hi[i] = 0;
  if (lane >= Row<HD>::ACT) return;
  const float* b = p + PP * lane;
#pragma nounroll
  for (uint32_t c = 0; c < nparts; c += 4) {
    vec x[4], y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {  // (past the last one: that one again, not added)
      const float* r = b + (size_t)min(c + k, nparts - 1) * stride;
      if constexpr (PP == 1) {
        x[k][0] = r[0];
        y[k][0] = r[HALF];
      } else {
        x[k] = *(const vec*)r;
        y[k] = *(const vec*)(r + HALF);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < PP; ++i) {
        lo[i] += c + k < nparts ? (T)x[k][i] : (T)-0.0;
        hi[i] += c + k < nparts ? (T)y[k][i] : (T)-0.0;
      }
  }
}

// Cos and sin of a lane's pairs at a position, and a norm's weights at them (1 without one).
template <int HD>
struct Turn {
  static constexpr int PP = Row<HD>::PP;
  float2 cs[PP];
};
template <int HD, bool TABLE>
__device__ __forceinline__ void load_turn(const RowArgs& a, uint32_t pos, int lane, Turn<HD>& t) {
  constexpr int PP = Row<HD>::PP, HALF = Row<HD>::HALF;
#pragma unroll
  for (int i = 0; i < PP; ++i) {
    const int k = min(PP * lane + i, HALF - 1);
    t.cs[i] = TABLE ? a.rope_cs[(size_t)pos * HALF + k]
                    : g4mqf::rope_cos_sin(a.theta, a.apply_divisor, a.rope_freqs[k], k, HD, pos);
  }
}
template <int HD>
struct Weights {
  static constexpr int PP = Row<HD>::PP;
  float lo[PP], hi[PP];
};
template <int HD>
__device__ __forceinline__ void load_weights(const uint16_t* w, int lane, Weights<HD>& t) {
  constexpr int PP = Row<HD>::PP, HALF = Row<HD>::HALF;
#pragma unroll
  for (int i = 0; i < PP; ++i) {
    const int k = min(PP * lane + i, HALF - 1);
    t.lo[i] = g4d::f16_bits_to_f32(w[k]);
    t.hi[i] = g4d::f16_bits_to_f32(w[k + HALF]);
  }
}
template <int HD, typename T>
__device__ __forceinline__ void rotate(const Weights<HD>& w, const Turn<HD>& t, T* lo, T* hi) {
#pragma unroll
  for (int i = 0; i < Row<HD>::PP; ++i) {
    const T x0 = lo[i] * (T)w.lo[i], x1 = hi[i] * (T)w.hi[i];
    lo[i] = x0 * (T)t.cs[i].x - x1 * (T)t.cs[i].y;
    hi[i] = x0 * (T)t.cs[i].y + x1 * (T)t.cs[i].x;
  }
}

// The heads of a row QH at a time, a wave each.
template <int HD, int NT, int QH, bool TABLE, bool MOVED>
__device__ __forceinline__ void q_row(const RowArgs& a, uint32_t block) {
  constexpr int PP = Row<HD>::PP, HALF = Row<HD>::HALF, NW = NT / 64;
  const int lane = threadIdx.x & 63;
  const uint32_t groups = (a.nqh + QH - 1) / QH;
  const uint64_t i = (uint64_t)block * NW + (threadIdx.x >> 6);
  if (i >= (uint64_t)a.rows.num_rows * groups) return;
  const uint32_t row = (uint32_t)(i / groups), h0 = (uint32_t)(i % groups) * QH;
  const size_t at = ((size_t)row * a.nqh + h0) * HD, stride = (size_t)a.rows.num_rows * a.nqh * HD;
  Weights<HD> w;
  load_weights<HD>(a.q_w, lane, w);
  float lo[QH][PP], hi[QH][PP];
#pragma unroll
  for (int h = 0; h < QH; ++h)
    load_row<HD>(a.q + at + min((uint32_t)h, a.nqh - 1 - h0) * HD, stride, a.nparts, lane, lo[h], hi[h]);
  const uint32_t s = seq_of_row(a.rows, row);
  if (s >= a.rows.num_seqs) return;
  const Seq q = seq_rows(a.rows, s);
  uint32_t p0 = q.base;
  if (!q.len || (MOVED && !moved_to(a, s, q, p0))) return;
  Turn<HD> t;
  load_turn<HD, TABLE>(a, p0 + (row - q.first), lane, t);
#pragma unroll
  for (int h = 0; h < QH; ++h) {
    if (h0 + h >= a.nqh) return;
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < PP; ++e) ss += lo[h][e] * lo[h][e] + hi[h][e] * hi[h][e];
    ss = g4d::wave_sum_dpp(ss);
    const float inv = 1.0f / sqrtf(ss * (1.0f / (float)HD) + a.eps);
#pragma unroll
    for (int e = 0; e < PP; ++e) {
      lo[h][e] *= inv;
      hi[h][e] *= inv;
    }
    rotate<HD>(w, t, lo[h], hi[h]);
    if (lane < Row<HD>::ACT) {
      float* o = a.q_out + at + h * HD + PP * lane;
      if constexpr (PP == 1) {
        o[0] = lo[h][0];
        o[HALF] = hi[h][0];
      } else {
        typedef float vec __attribute__((ext_vector_type(PP)));
        vec x, y;
#pragma unroll
        for (int e = 0; e < PP; ++e) {
          x[e] = lo[h][e];
          y[e] = hi[h][e];
        }
        *(vec*)o = x;
        *(vec*)(o + HALF) = y;
      }
    }
  }
}

__device__ __forceinline__ uint64_t magnitude(double x) { return __builtin_bit_cast(uint64_t, x) & ~(1ull << 63); }
// 1 / sqrt(x), from the hardware's estimate by two steps of Newton's iteration.
__device__ __forceinline__ double rsqrt64(double x) {
  double y = __builtin_amdgcn_rsq(x);
#pragma unroll
  for (int i = 0; i < 2; ++i) y = fma(y * 0.5, fma(-x * y, y, 1.0), y);
  return y;
}

}  // namespace g4kv8
