// attn_paged.hpp — what attention over the 8-bit and the 4-bit paged K/V pool
// share: a call's rows as columns of query heads, its pages as tiles of 16 rows,
// its work dealt to workgroups, and the output as operand blocks.
#pragma once
#include "kv8.hpp"
#include "mm_operand.hpp"

namespace g4kv8 {

using g4mm::f4;

struct PagedArgs {
  const float* q;
  const int32_t* page_table;
  Rows rows;
  uint32_t nqh, nkh, G, g_magic, g_same, page_tiles, page_magic, page_same, max_pages, num_pages, window;
  float scale;
  float* out;
  uint8_t* ops;    // few rows, or null: the output as operand blocks, in ntv tiles of 16 rows
  int ntv;
  uint32_t wgs;    // workgroups that share the work
  uint2* meta;     // per sequence and KV head: the workgroups that hold its partials
  float* part;     // their partials
  uint32_t tiles;  // many rows: column tiles of the longest sequence
};
inline PagedArgs paged_args(const g4_kv8_params& p, const float* q, const int32_t* page_table, const uint32_t* seq_lens,
                            const uint32_t* row_starts, float* out, void* ops) {
  const uint32_t tiles = p.page_size / 16, G = p.num_q_heads / p.num_kv_heads;
  auto magic = [](uint32_t d) { return d == 1 ? 0u : (uint32_t)(((1ull << 32) + d - 1) / d); };
  PagedArgs a{};
  a.q = q;
  a.page_table = page_table;
  a.rows = {seq_lens, row_starts, p.num_seqs, p.num_rows, p.max_rows, p.max_seq_len};
  a.nqh = p.num_q_heads;
  a.nkh = p.num_kv_heads;
  a.G = G;
  a.g_magic = magic(G);
  a.g_same = G == 1 ? ~0u : 0u;
  a.page_tiles = tiles;
  a.page_magic = magic(tiles);
  a.page_same = tiles == 1 ? ~0u : 0u;
  a.max_pages = p.max_pages;
  a.num_pages = p.num_pages;
  a.window = p.sliding_window;
  a.scale = p.scale;
  a.out = out;
  a.ops = (uint8_t*)ops;
  a.ntv = (int)(g4d::pad_batch(p.num_rows) / 16);
  return a;
}

__device__ __forceinline__ float exp2_h(float x) { return __builtin_amdgcn_exp2f(x); }

// Wave-uniform values into scalar registers.
__device__ __forceinline__ uint32_t uni(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int32_t uni_i(int32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint64_t uni(uint64_t x) {
  return (uint64_t)uni((uint32_t)(x >> 32)) << 32 | uni((uint32_t)x);
}

// x / G for x < 2^28 (G <= 16: x times the rounded-up 2^32 / G is off by less than 1 / G; a G of 1: a magic of 0 and
// all of x).
__device__ __forceinline__ uint32_t div_g(const PagedArgs& a, uint32_t x) { return __umulhi(x, a.g_magic) + (x & a.g_same); }
// Row of q and of the output (of nqh heads a row) that is a sequence's column of a KV head.
__device__ __forceinline__ size_t row_of(const PagedArgs& a, uint32_t first, uint32_t kvh, uint32_t col) {
  return (size_t)first * a.nqh + kvh * a.G + (size_t)div_g(a, col) * (a.nqh - a.G) + col;
}

// Page (of the sequence's list) that holds tile t: t < 2^26, at most 64 tiles
// a page, so t times the rounded-up 2^32 / tiles is off by less than a tile
// (one tile a page: a magic of 0 and all of t).
__device__ __forceinline__ uint32_t page_of(const PagedArgs& a, uint32_t t) {
  return __umulhi(t, a.page_magic) + (t & a.page_same);
}
__device__ __forceinline__ uint32_t clamp_page(const PagedArgs& a, int32_t pg) {
  return pg < 0 ? 0u : min((uint32_t)pg, a.num_pages - 1);
}

// First position (of a whole tile) that any row of the sequence sees.
__device__ __forceinline__ uint32_t first_seen(const PagedArgs& a, const Seq& q) {
  return a.window && q.base + 1 > a.window ? (q.base + 1 - a.window) & ~15u : 0u;
}

// T units dealt to W workgroups: the first T % W get one more.
struct Share {
  uint32_t T, W;
  __device__ uint32_t first(uint32_t wg) const { return wg * (T / W) + min(wg, T % W); }
  __device__ uint32_t owner(uint32_t unit) const {
    const uint32_t q = T / W, r = T % W, big = r * (q + 1);
    return unit < big ? unit / (q + 1) : r + (unit - big) / q;
  }
};

// Inclusive sums over the lanes: within rows of 16, then the rows' last values
// broadcast to the rows behind.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  int v = (int)x;
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return (uint32_t)v;
}
__device__ __forceinline__ uint32_t pick(uint32_t v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// The output's super-block kb of a row, lane l holding its values 4 l .. + 3, as
// an operand block of the o projection (g4d::Ops), what the batch's norms write of
// the same values.
__device__ __forceinline__ void write_ops(const PagedArgs& a, uint32_t row, uint32_t kb, int l, const f4& y) {
  typedef _Float16 h4 __attribute__((ext_vector_type(4)));
  const float am = g4d::wave_max_dpp(fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3]))));
  float inverse;
  const float up = g4d::f16_pair_scale(am, inverse);
  const uint32_t t = row >> 4, c = row & 15u, s = l >> 3, q = (l >> 1) & 3, j = 4 * (l & 1);
  uint8_t* base = a.ops + (size_t)kb * g4d::Ops::bytes(a.ntv);
  h4 hi, lo;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = y[i] * up;
    hi[i] = (_Float16)x;
    lo[i] = (_Float16)(x - (float)hi[i]);
    sum += x;
  }
  uint8_t* mp = base + t * g4d::Ops::MAIN_T + s * 2048 + (c + 16 * q) * 16 + j * 2;
  *(h4*)mp = hi;
  *(h4*)(mp + 1024) = lo;
  sum = g4d::sum8(sum) * 0.015625f;  // of the sub-block, in three parts
  if ((l & 7) == 0) {
    h4 p;
    p[0] = (_Float16)sum;
    const float r = sum - (float)p[0];
    p[1] = (_Float16)r;
    p[2] = (_Float16)(r - (float)p[1]);
    p[3] = (_Float16)0.f;
    *(h4*)(base + g4d::Ops::sums_off(a.ntv) + t * 1024 + (c + 16 * (s >> 1)) * 16 + (s & 1) * 8) = p;
  }
  if (l == 0) *(float*)(base + g4d::Ops::scale_off(a.ntv) + t * 64 + c * 4) = inverse;
}

}  // namespace g4kv8
