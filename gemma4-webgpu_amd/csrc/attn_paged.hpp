// attn_paged.hpp — what attention over the 8-bit and the 4-bit paged K/V pool
// share: a call's rows as columns of query heads, its pages as tiles of 16 rows,
// its work dealt to workgroups, and the output as operand blocks.
#pragma once
#include <algorithm>

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

// ---- many rows a sequence: tiles of 64 columns, steps of 64 positions ----

constexpr int TC = 64, TP = 64;  // columns of a workgroup, positions of a step
constexpr float kTileP = 32768.f;
constexpr uint32_t kTileCost = 3, kLeast = 4;  // cost of a tile besides its steps; least cost of a share

// Columns [64 ct, + 64) of a sequence and KV head: rows r0 .. r1, which see positions lo .. end - 1.
struct Tile {
  uint32_t lo, end, steps;
};
__device__ __forceinline__ Tile tile_of(const PagedArgs& a, const Seq& q, uint32_t ct) {
  const uint32_t r0 = div_g(a, ct * TC), r1 = min(q.n - 1, div_g(a, ct * TC + TC - 1));
  Tile t;
  t.lo = a.window && q.base + r0 + 1 > a.window ? (q.base + r0 + 1 - a.window) & ~15u : 0u;
  t.end = q.base + r1 + 1;
  t.steps = (t.end - t.lo + TP - 1) / TP;
  return t;
}
// Cost of column tile j % tiles of sequence j / tiles: kTileCost, then its steps (0: there is none).
__device__ __forceinline__ uint32_t cost_of(const PagedArgs& a, uint32_t j) {
  const Seq q = seq_rows(a.rows, j / a.tiles);
  const uint32_t ct = j % a.tiles;
  return q.len && ct * TC < q.n * a.G ? kTileCost + tile_of(a, q, ct).steps : 0u;
}

// A workgroup's share of the whole cost, which is dealt in equal parts: the steps of all column tiles, and kTileCost
// more for each. A thread numbers a run of tiles.
template <int NTH>
struct WalkLds {
  uint32_t upto[NTH + 1], sum[NTH / 64], at[2];  // upto: units before each thread's run
  float all[NTH / 64];
};
struct Part {  // steps st0 .. st1 - 1 of the `steps` of a tile
  Seq q;
  Tile t;
  uint32_t s, ct, kvh, st0, st1, slot;
  uint2 meta;  // what to note of the tile, by the one that begins it
};
template <int NTH>
struct Walk {
  const PagedArgs& a;
  WalkLds<NTH>& m;
  uint32_t pairs, run, pair, before, used, u, ue;
  Share sh;

  // The column tile of a unit, by the thread whose run holds it.
  __device__ __forceinline__ void locate(uint32_t unit) {
    const uint32_t tid = threadIdx.x;
    if (m.upto[tid] <= unit && m.upto[tid + 1] > unit) {
      uint32_t j = tid * run, at = m.upto[tid];
      if (run > 1)  // (a run of one is that tile)
        for (uint32_t n; at + (n = cost_of(a, j) * a.nkh) <= unit; ++j) at += n;
      m.at[0] = j;
      m.at[1] = at;
    }
    __syncthreads();
    pair = uni(m.at[0]);
    before = uni(m.at[1]);
    __syncthreads();
  }
  // False, and every tile noted as without partials, where the costs are past what 32 bits number: rows that are one
  // sequence's each cost less than 2^31 (checked by the host), but starts that descend in between may give rows to many
  // sequences. Nothing is written then.
  __device__ __forceinline__ bool begin() {
    const uint32_t tid = threadIdx.x, l = tid & 63, w = tid >> 6, wg = blockIdx.x;
    pairs = a.rows.num_seqs * a.tiles;
    run = (pairs + NTH - 1) / NTH;
    const uint32_t j0 = min(tid * run, pairs), j1 = min(j0 + run, pairs);
    uint64_t mine = 0;
    for (uint32_t j = j0; j < j1; ++j) mine += (uint64_t)cost_of(a, j) * a.nkh;
    uint32_t upto = wave_scan((uint32_t)mine);
    const float wave_all = g4d::wave_sum_dpp((float)mine);
    if (l == 63) {
      m.sum[w] = upto;
      m.all[w] = wave_all;
    }
    __syncthreads();
    uint32_t total = 0;
    float all = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < NTH / 64; ++i) {
      if (i < w) upto += m.sum[i];
      total += m.sum[i];
      all += m.all[i];
    }
    if (all > 3e9f) {  // (uniform)
      for (uint64_t i = (uint64_t)wg * NTH + tid; i < (uint64_t)pairs * a.nkh; i += (uint64_t)gridDim.x * NTH)
        a.meta[i] = make_uint2(0, 0);
      return false;
    }
    total = uni(total);
    m.upto[tid + 1] = upto;
    if (tid == 0) m.upto[0] = 0;
    __syncthreads();
    sh = Share{total, min(a.wgs, (total + kLeast - 1) / kLeast)};
    pair = before = used = 0;  // column tile at hand, the units before it; partials written
    u = wg < sh.W ? sh.first(wg) : 0u;
    ue = wg < sh.W ? sh.first(wg + 1) : 0u;
    if (u < ue) locate(u);
    return true;
  }
  __device__ __forceinline__ bool next(Part& p) {
    while (u < ue) {
      p.s = pair / a.tiles;
      p.ct = pair % a.tiles;
      const Seq q = seq_rows(a.rows, p.s);
      p.q = Seq{uni(q.first), uni(q.n), uni(q.base), uni(q.len)};
      if (!p.q.len || p.ct * TC >= p.q.n * a.G) {  // behind the sequence's last tile
        locate(u);
        continue;
      }
      const Tile t = tile_of(a, p.q, p.ct);
      p.t = Tile{uni(t.lo), uni(t.end), uni(t.steps)};
      const uint32_t cost = kTileCost + p.t.steps;
      if (u >= before + cost * a.nkh) {
        before += cost * a.nkh;
        ++pair;
        if (pair >= pairs) locate(u);
        continue;
      }
      p.kvh = a.nkh == 1 ? 0u : uni((u - before) / cost);
      const uint32_t seg = before + p.kvh * cost, stop = min(seg + cost, ue);  // the tile's first unit, the last here
      const uint32_t seg0 = seg + kTileCost;
      p.st0 = max(u, seg0) - seg0;
      p.st1 = max(stop, seg0) - seg0;
      u = stop;
      if (p.st0 == p.st1) continue;  // (the share ends before the tile's first step)
      p.slot = 2 * blockIdx.x + used;  // (0 for a tile begun by another workgroup: it comes first)
      used = 1;
      p.meta = make_uint2(p.slot, sh.owner(seg + cost - 1));
      return true;
    }
    return false;
  }
  __device__ __forceinline__ size_t tile_index(const Part& p) const { return (size_t)(p.s * a.tiles + p.ct) * a.nkh + p.kvh; }
};
// Rows that see nothing.
template <int HD, int NTH>
__device__ __forceinline__ void clear_rows(const PagedArgs& a) {
  const uint32_t pairs = a.rows.num_seqs * a.tiles;
  for (uint32_t j = blockIdx.x; j < pairs; j += gridDim.x) {
    const Seq q = seq_rows(a.rows, j / a.tiles);
    const uint32_t g0 = j % a.tiles * TC, ncols = q.n * a.G;
    if (q.len || g0 >= ncols) continue;
    for (uint32_t i = threadIdx.x; i < min((uint32_t)TC, ncols - g0) * a.nkh * HD; i += NTH) {
      const uint32_t g = g0 + i / HD / a.nkh, kvh = i / HD % a.nkh;
      a.out[row_of(a, q.first, kvh, g) * HD + i % HD] = 0.f;
    }
  }
}

// Column tiles of the longest sequence; cost of all tiles (at most).
inline uint32_t tiles_of(const g4_kv8_params& p) {
  return ceil_div((uint64_t)p.max_rows * (p.num_q_heads / p.num_kv_heads), TC);
}
inline uint64_t all_cost(const g4_kv8_params& p) {
  const uint64_t G = p.num_q_heads / p.num_kv_heads, rows = TC / G + 2;  // of a tile
  const uint64_t tiles =
      std::min<uint64_t>(ceil_div(p.num_rows * G, TC) + p.num_seqs, (uint64_t)tiles_of(p) * p.num_seqs);
  uint64_t span = p.max_seq_len;
  if (p.sliding_window) span = std::min<uint64_t>(span, p.sliding_window + rows + 15);
  return tiles * p.num_kv_heads * (kTileCost + ceil_div(span, TP));
}

}  // namespace g4kv8
