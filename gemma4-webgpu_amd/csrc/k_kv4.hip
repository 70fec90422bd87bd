// k_kv4.hip — appending to the 4-bit paged K/V pool, reading its values, and
// evicting rows by their attention weight (no counterpart in the reference).
//
// A value is an e2m1 code times 2^e, one e per 32 dims of a row and head: the
// least with |x| <= 7 * 2^e. Between 6 and 7 the nearest of 6 and the 8 that a
// wider code would have is 6, so every element is within 2^e of its code, and of
// the bounds from 6 to 8 this one has the least error for normal values: a root
// mean square of 0.112 of their deviation, against 0.115 at 6 and at 8. Each row has its
// own scales: nothing is ever rounded again, whatever comes after it or moves it.
#include <algorithm>

#include "attn_paged.hpp"
#include "kv4.hpp"
#include "kv4_keys.hpp"
#include "kv_rows.hpp"

namespace {

using namespace g4kv8;
using g4kv4::BAD;
using g4kv4::BLOCK;
using g4kv4::Keys;

constexpr int PT = 256;    // threads of the append
constexpr int QH = 2;      // q heads of a wave
constexpr int VT = 256;    // of the values kernel
constexpr int ST = Keys::THREADS;  // of the selection and the moves (of more than Keys::GROUP candidates the selection
                                   // reads the masses again for each round)

struct ProArgs : RowArgs {
  g4kv4::Pool pool;
  uint32_t kv_blocks;
};

// The least e >= -20 with x <= 7 * 2^e = 1.75 * 2^(e + 2), of a double's magnitude bits; kBad where it is not finite.
constexpr int kBad = 1000, kLeast = -20;
__device__ __forceinline__ int exponent_of(uint64_t bits) {
  constexpr uint64_t carry = (1ull << 50) - 1;  // takes a fraction above 0.75 to the next exponent
  return bits >= 0x7ffull << 52 ? kBad : max((int)((bits + carry) >> 52) - 1023 - 2, kLeast);
}
// Code of x * up, halves to the even code: steps of 0.5 below 2, of 1 below 4, of 2 from there.
__device__ __forceinline__ uint32_t code_of(double x, double up) {
  const double y = fabs(x * up);
  const double step = y < 2.0 ? 2.0 : y < 4.0 ? 1.0 : 0.5;
  const int c = min((int)rint(y * step) + (y < 2.0 ? 0 : y < 4.0 ? 2 : 4), 7);
  return (uint32_t)c | (uint32_t)(__builtin_bit_cast(uint64_t, x) >> 63) << 3;
}
template <int RG>
__device__ __forceinline__ float group_max(float a) {
  a = g4d::max8(a);
  if constexpr (RG >= 16) a = fmaxf(a, g4d::dpp<g4d::kDppMirror>(a));
  if constexpr (RG >= 32) a = g4d::xmax16(a);
  return a;
}

// A wave a row and head of K or of V (a scale's dims are neighbouring lanes, so that
// no wave waits for another); other workgroups take q's rows. One row each of 64
// sequences at head dim 256 and three parts: 3.8 us, a chain of three loads behind a
// launch. 1900 rows of 8 + 2 heads at 512: 17.8 us for 72 MB, 4.0 TB/s.
template <int HD, bool TABLE, bool MOVED>
__global__ __launch_bounds__(PT, 4) void kv4_prologue_kernel(ProArgs a) {
  constexpr int PP = Row<HD>::PP, NB = HD / BLOCK, GL = BLOCK / PP;
  if (blockIdx.x >= a.kv_blocks) {
    q_row<HD, PT, QH, TABLE, MOVED>(a, blockIdx.x - a.kv_blocks);
    return;
  }
  const int lane = threadIdx.x & 63;
  uint64_t i = (uint64_t)blockIdx.x * (PT / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool is_v = i & 1;
  i >>= 1;
  if (i >= (uint64_t)a.rows.num_rows * a.nkh) return;
  const uint32_t row = (uint32_t)(i / a.nkh), h = (uint32_t)(i % a.nkh);
  double lo[PP], hi[PP];
  Weights<HD> wt;
  if (!is_v) load_weights<HD>(a.k_w, lane, wt);
  load_row<HD>((is_v ? a.v : a.k) + ((size_t)row * a.nkh + h) * HD, (size_t)a.rows.num_rows * a.nkh * HD, a.nparts,
               lane, lo, hi);
  const uint32_t s = seq_of_row(a.rows, row);
  if (s >= a.rows.num_seqs) return;
  const Seq q = seq_rows(a.rows, s);
  uint32_t p0 = q.base;
  if (!q.len || (MOVED && !moved_to(a, s, q, p0))) return;
  const uint32_t t = q.base + (row - q.first), slot = t % a.page_size;
  const int32_t pg = a.page_table[(size_t)s * a.max_pages + t / a.page_size];
  if (pg < 0 || pg >= (int32_t)a.num_pages) return;
  Turn<HD> turn;
  if (!is_v) load_turn<HD, TABLE>(a, p0 + (row - q.first), lane, turn);

  double ss = 0.0;
#pragma unroll
  for (int e = 0; e < PP; ++e) ss = fma(lo[e], lo[e], fma(hi[e], hi[e], ss));
  const double inv = rsqrt64(g4d::wave_sum_dpp(ss) * (1.0 / HD) + (double)a.eps);
#pragma unroll
  for (int e = 0; e < PP; ++e) {
    lo[e] *= inv;
    hi[e] *= inv;
  }
  if (!is_v) rotate<HD>(wt, turn, lo, hi);

  // the lane's dims are of block PP * lane / 32 and, half a row on, of that + NB / 2
  int el = kLeast, eh = kLeast;
#pragma unroll
  for (int e = 0; e < PP; ++e) {
    el = max(el, exponent_of(magnitude(lo[e])));
    eh = max(eh, exponent_of(magnitude(hi[e])));
  }
  const bool poison = __ballot(max(el, eh) == kBad) != 0;
  el = (int)group_max<GL>((float)el);
  eh = (int)group_max<GL>((float)eh);
  const double ul = __builtin_bit_cast(double, (uint64_t)(1023 - el) << 52);
  const double uh = __builtin_bit_cast(double, (uint64_t)(1023 - eh) << 52);
  uint32_t x = 0, y = 0;
#pragma unroll
  for (int e = 0; e < PP; ++e) {
    x |= (poison ? 0u : code_of(lo[e], ul)) << (4 * e);
    y |= (poison ? 0u : code_of(hi[e], uh)) << (4 * e);
  }
  const g4kv4::Shape sh{a.page_size, a.nkh, HD};
  uint8_t* d = (is_v ? a.pool.v : a.pool.k) + sh.code((uint32_t)pg, slot, h);
  if constexpr (PP == 1) {  // (the neighbour has the byte's other half)
    x |= (uint32_t)g4d::dppi<g4d::kDppXor1>((int)x) << 4;
    y |= (uint32_t)g4d::dppi<g4d::kDppXor1>((int)y) << 4;
    if (lane < Row<HD>::ACT && lane % 2 == 0) {
      d[lane / 2] = (uint8_t)x;
      d[lane / 2 + HD / 4] = (uint8_t)y;
    }
  } else if constexpr (PP == 2) {
    d[lane] = (uint8_t)x;
    d[lane + HD / 4] = (uint8_t)y;
  } else {
    *(uint16_t*)(d + 2 * lane) = (uint16_t)x;
    *(uint16_t*)(d + 2 * lane + HD / 4) = (uint16_t)y;
  }
  if (lane % GL == 0 && lane < Row<HD>::ACT) {
    const uint32_t b = lane / GL;
    const uint8_t bl = (uint8_t)(poison ? BAD : (uint32_t)(min(el, 127) + 127));
    const uint8_t bh = (uint8_t)(poison ? BAD : (uint32_t)(min(eh, 127) + 127));
    if (is_v) {
      a.pool.vs[sh.v_scale((uint32_t)pg, slot, h, b)] = bl;
      a.pool.vs[sh.v_scale((uint32_t)pg, slot, h, b + NB / 2)] = bh;
    } else {
      a.pool.ks[sh.k_scale((uint32_t)pg, slot, h, b)] = bl;
      a.pool.ks[sh.k_scale((uint32_t)pg, slot, h, b + NB / 2)] = bh;
    }
  }
  if (!is_v && lane == 0 && a.pool.mass) a.pool.mass[sh.row((uint32_t)pg, slot, h)] = 0.f;
}

struct ValArgs {
  const uint8_t* pool[2];
  const uint8_t* scale[2];
  uint16_t* out[2];
  const int32_t* pages;
  g4kv4::Shape sh;
  uint32_t num_pages;
};

// 16 codes a thread: 8 bytes read and 32 written, so the writes bound it (76 MB of
// 64 sequences' 1024 rows 20.5 us).
__global__ __launch_bounds__(VT) void kv4_values_kernel(ValArgs a) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const uint32_t values = a.sh.page_size * a.sh.nkh * a.sh.hd;  // of a page
  const uint32_t i = (blockIdx.y * VT + threadIdx.x) * 16;
  if (i >= values) return;
  const uint32_t which = blockIdx.z, block = i % a.sh.hd / BLOCK, row = i / a.sh.hd;
  const int32_t pg = a.pages[blockIdx.x];
  const bool in = pg >= 0 && pg < (int32_t)a.num_pages;
  const uint32_t page = in ? (uint32_t)pg : 0u, slot = row / a.sh.nkh, h = row % a.sh.nkh;
  const uint2 x = *(const uint2*)(a.pool[which] + ((size_t)page * values + i) / 2);
  const float sc = g4kv4::scale_of(
      a.scale[which][which ? a.sh.v_scale(page, slot, h, block) : a.sh.k_scale(page, slot, h, block)]);
  u32x4 y[2];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t b = (e < 4 ? x.x : x.y) >> (8 * (e & 3));
    y[e / 4][e % 4] = (uint32_t)g4d::f32_to_f16_bits(g4kv4::value_of(b) * sc) |
                      (uint32_t)g4d::f32_to_f16_bits(g4kv4::value_of(b >> 4) * sc) << 16;
  }
  u32x4* o = (u32x4*)(a.out[which] + (size_t)blockIdx.x * values + i);
  o[0] = in ? y[0] : u32x4{0, 0, 0, 0};
  o[1] = in ? y[1] : u32x4{0, 0, 0, 0};
}

// ---------------------------------------------------------------------------
// eviction
// ---------------------------------------------------------------------------
//
// kv4_select_kernel, a workgroup a sequence and KV head: the order of masses is
// that of their bits (they are above 0, or count 0), so the bound of the largest
// is found by three rounds of bins, from the top 11 bits down; then the rows above
// it and the first of those at it are listed in order. The keys stay in LDS between
// the rounds (in registers the loops over them unroll, and their conditions spill:
// 33 us where this is 27). 2304 rows of one sequence: 7.7 us, a chain of six loads
// (2.2), of the rounds' barriers (1 each) and of the list's; 32000 rows 27, 7 of them
// the masses of one CU, 4 bytes of a line each, 10 the rounds and 7 the list. More
// than Keys::GROUP candidates are read again for each round and the list: 40000 rows
// cut with their moves 71 us where 32000 are in 41.
// kv4_move_kernel moves the rows: 8.6 us for one sequence of 2048 rows of head dim
// 512 (places 0.6, pages 0.4, rows 3.2, stores 1.4 and the launch), 8.0 for 64 of
// 1024 at 256, 14.9 for 8 of 4000 and two heads at 128.
struct EvictArgs {
  g4kv4::Pool pool;
  g4kv4::Shape sh;
  const int32_t* page_table;
  uint32_t* seq_lens;
  uint32_t num_seqs, max_pages, num_pages, max_seq_len, keep, first, recent;
  int32_t* kept;
  uint32_t* cut;  // per sequence: whether it is cut
  uint32_t some;  // pieces of a row that a workgroup moves
  uint32_t tiles, magic, same;  // of 16 rows a page, the rounded-up 2^32 / tiles (0 for one tile: `same` takes all of t)
  // (exact as in the attention: t / 16 < 2^26, at most 64 tiles a page)
  __device__ __forceinline__ uint32_t page_of(uint32_t t) const { return __umulhi(t / 16, magic) + (t / 16 & same); }
  __device__ __forceinline__ uint32_t slot_of(uint32_t t) const { return t - page_of(t) * sh.page_size; }
};

__device__ __forceinline__ uint32_t key_of(float x) { return x > 0.f ? __float_as_uint(x) : 0u; }

__global__ __launch_bounds__(ST) void kv4_select_kernel(EvictArgs a) {
  constexpr uint32_t NW = ST / 64, BINS = 2 * ST, GROUP = Keys::GROUP;
  __shared__ uint32_t s_key[GROUP];
  __shared__ uint32_t s_bin[BINS], s_sum[2 * NW], s_found[3];
  const uint32_t tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t s = blockIdx.x / a.sh.nkh, h = blockIdx.x % a.sh.nkh;
  const uint32_t L = a.seq_lens[s];
  int32_t* kept = a.kept + (size_t)blockIdx.x * a.keep;
  const bool cut = L > a.keep && L <= a.max_seq_len;
  if (h == 0 && tid == 0) a.cut[s] = cut;
  if (!cut) {
    for (uint32_t i = tid; i < a.keep; i += ST) kept[i] = L <= a.max_seq_len && i < L ? (int32_t)i : -1;
    return;
  }
  for (uint32_t i = tid; i < a.first; i += ST) kept[i] = (int32_t)i;
  for (uint32_t i = tid; i < a.recent; i += ST) kept[a.keep - a.recent + i] = (int32_t)(L - a.recent + i);
  const uint32_t n = L - a.first - a.recent, m = a.keep - a.first - a.recent;  // of n candidates m are kept, m < n
  if (m == 0) return;  // (uniform)
  const Keys keys{n};
  const uint32_t groups = keys.groups();
  const int32_t* list = a.page_table + (size_t)s * a.max_pages;
  const uint32_t page_rows = a.sh.page_size * a.sh.nkh, last_page = (L - 1) / a.sh.page_size;
  const uint32_t pages_on = 64 / a.sh.page_size, rows_on = 64 % a.sh.page_size * a.sh.nkh;  // from a key to the next
  uint32_t* const my_key = s_key + Keys::place(w) + lane;  // [64 * j]: of candidate mine(g) + 64 * j of the group
  auto mine = [&](uint32_t g) { return keys.first(g, w) + lane; };
  // Eight at a time: their page ids, then their masses and the next eight's ids, are on their way together. Past the last
  // candidate they are 0, which no round counts and which, behind all others in order, no place is left for.
  auto fetch = [&](uint32_t g) {
    const uint32_t rows = keys.rows(g), count = keys.each(g), i0 = mine(g), t0 = a.first + g * GROUP + i0;
    uint32_t page = a.page_of(t0), row = (t0 - page * a.sh.page_size) * a.sh.nkh + h;
    auto on = [&](uint32_t& p, uint32_t& r) {
      r += rows_on;
      const bool over = r >= page_rows;
      r -= over ? page_rows : 0u;
      p += pages_on + (over ? 1u : 0u);
    };
    int32_t id[8], next[8];
    uint32_t at[8], p = page, r = row;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j, on(p, r)) next[j] = list[min(p, last_page)];
    for (uint32_t j0 = 0; j0 < count; j0 += 8) {
      float x[8];
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j, on(page, row)) {
        id[j] = next[j] < (int32_t)a.num_pages ? next[j] : -1;
        at[j] = row;
      }
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) x[j] = a.pool.mass[(size_t)(uint32_t)max(id[j], 0) * page_rows + at[j]];
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j, on(p, r)) next[j] = list[min(p, last_page)];
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        const uint32_t i = i0 + (j0 + j) * 64;
        if (j0 + j < count) my_key[(j0 + j) * 64] = id[j] >= 0 && i < rows ? key_of(x[j]) : 0u;  // (uniform)
      }
    }
  };
  fetch(0);
  uint32_t bound = 0, left = m;  // the m-th largest key so far; how many of those that share its bits are kept
  uint32_t share = n;            // how many share them
  for (int pass = 0; pass < 3; ++pass) {
    // 11, 11 and 10 bits. The least bin has those that no other has: rows without weight, often many, are not counted
    // one by one.
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t from = bound + (1u << shift), range = (pass == 0 ? 1u << 31 : pass == 1 ? 1u << 21 : 1u << 10) - (1u << shift);
    s_bin[2 * tid] = s_bin[2 * tid + 1] = 0;
    __syncthreads();
    for (uint32_t g = 0; g < groups; ++g) {
      if (groups > 1 && (pass || g)) fetch(g);
      const uint32_t count = keys.each(g);
#pragma unroll 8
      for (uint32_t j = 0; j < count; ++j) {
        const uint32_t d = my_key[64 * j] - from;
        if (d < range) atomicAdd(&s_bin[(d >> shift) + 1], 1u);
      }
    }
    __syncthreads();
    // counts from the largest bin down: two bins a thread, summed over its wave, then over the waves
    uint32_t hi = s_bin[BINS - 1 - 2 * tid], lo = s_bin[BINS - 2 - 2 * tid];
    const uint32_t upto = wave_scan(hi + lo);
    if (lane == 63) s_sum[w] = upto;
    __syncthreads();
    const uint32_t sums = wave_scan(s_sum[lane % NW]);  // (in its first NW lanes)
    const uint32_t above = upto - hi - lo + (w ? pick(sums, w - 1) : 0u);
    if (tid == ST - 1) lo = share - above - hi;
    if (above < left && above + hi + lo >= left) {  // (one thread's)
      const bool one = above + hi >= left;
      s_found[0] = BINS - 1 - 2 * tid - (one ? 0 : 1);
      s_found[1] = above + (one ? 0 : hi);
      s_found[2] = one ? hi : lo;
    }
    __syncthreads();
    bound |= s_found[0] << shift;
    left -= s_found[1];
    share = s_found[2];
  }
  // the rows above the bound and the first `left` at it, in order: how many each wave has, then each row's place
  uint32_t above = 0, at = 0;  // of the groups before
  for (uint32_t g = 0; g < groups; ++g) {
    if (groups > 1) fetch(g);
    const uint32_t count = keys.each(g);
    uint32_t na = 0, ne = 0;
    for (uint32_t j = 0; j < count; ++j) {
      const uint32_t k = my_key[64 * j];
      na += __popcll(__ballot(k > bound));
      ne += __popcll(__ballot(k == bound));
    }
    __syncthreads();  // (the last group's sums, or the last round's, are read)
    if (lane == 0) {
      s_sum[w] = na;
      s_sum[NW + w] = ne;
    }
    __syncthreads();
    const uint32_t sa = wave_scan(s_sum[lane % NW]), se = wave_scan(s_sum[NW + lane % NW]);
    uint32_t wa = above + (w ? pick(sa, w - 1) : 0u), we = at + (w ? pick(se, w - 1) : 0u);
    above += pick(sa, NW - 1);
    at += pick(se, NW - 1);
    auto before = [&](uint64_t lanes, uint32_t x) {  // x more than there are of them below this one
      return __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, x));
    };
    int32_t* to = kept + a.first;
    const uint32_t t0 = a.first + g * GROUP + mine(g);
    for (uint32_t j = 0; j < count; ++j) {
      const uint32_t k = my_key[64 * j];
      const uint64_t ma = __ballot(k > bound), me = __ballot(k == bound);
      if (me == 0) {  // (uniform, and the rule)
        const uint32_t i = before(ma, wa + min(we, left));
        if (k > bound) to[i] = (int32_t)(t0 + 64 * j);
      } else {
        const uint32_t ra = before(ma, wa), re = before(me, we);
        if (k > bound || (k == bound && re < left)) to[ra + min(re, left)] = (int32_t)(t0 + 64 * j);
      }
      wa += __popcll(ma);
      we += __popcll(me);
    }
  }
}

// A workgroup the same `some` pieces of 16 bytes of every row that moves, with their scales; with K's first one also the
// masses. A row moves down only (kept[i] >= i), so a set of rows that is read before any of it is written overwrites
// none that a later set reads: the rows move in place, a set after the other, one barrier between.
constexpr int SETS = 4;  // rows of a thread that move at once
__global__ __launch_bounds__(ST) void kv4_move_kernel(EvictArgs a) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  // (the workgroups of a sequence and KV head have numbers that differ by multiples of 8: they are on one XCD, whose L2
  // has a row's line for all of them)
  const uint32_t some = a.some, parts = a.sh.hd / 32 / some, pairs = a.num_seqs * a.sh.nkh;
  const uint32_t pair = blockIdx.x / (16 * parts) * 8 + blockIdx.x % 8, part = blockIdx.x / 8 % (2 * parts);
  if (pair >= pairs) return;
  const uint32_t s = pair / a.sh.nkh, h = pair % a.sh.nkh;
  const uint32_t cut = a.cut[s];  // (on its way with the first places)
  const bool is_v = part >= parts;
  const uint32_t b = part % parts * some + threadIdx.x % some, per = ST / some, r = threadIdx.x / some;
  const int32_t *kept = a.kept + (size_t)pair * a.keep, *list = a.page_table + (size_t)s * a.max_pages;
  uint8_t *codes = (is_v ? a.pool.v : a.pool.k) + 16 * b, *scales = is_v ? a.pool.vs : a.pool.ks;
  const bool has_mass = part == 0 && threadIdx.x % some == 0;
  // of the set at hand, the next and the one after it: where its rows are, their pages. One wait for memory a set: the
  // rows of this one, the page ids of the next and the places of the one after it are on their way together.
  uint32_t from[SETS], from1[SETS] = {};
  int32_t src[SETS], dst[SETS];
  auto row_of_set = [&](uint32_t i0, int k) { return min(i0 + k * per + r, a.keep - 1); };  // (past the last: that one)
  auto places = [&](uint32_t i0, uint32_t* f) {
#pragma unroll
    for (int k = 0; k < SETS; ++k) f[k] = (uint32_t)kept[row_of_set(i0, k)];
  };
  auto pages = [&](uint32_t i0, const uint32_t* f) {
#pragma unroll
    for (int k = 0; k < SETS; ++k) {
      src[k] = list[a.page_of(f[k])];
      dst[k] = list[a.page_of(row_of_set(i0, k))];
    }
  };
  auto scale_at = [&](uint32_t page, uint32_t slot) {
    return is_v ? a.sh.v_scale(page, slot, h, b) : a.sh.k_scale(page, slot, h, b);
  };
  const uint32_t rows = SETS * per;
  places(0, from);
  if (rows < a.keep) places(rows, from1);
  if (!cut) return;
  if (h == 0 && part == 0 && threadIdx.x == 0) a.seq_lens[s] = a.keep;
  pages(0, from);
  for (uint32_t i0 = 0; i0 < a.keep; i0 += rows) {
    u32x4 x[SETS];
    uint8_t z[SETS];
    float m[SETS];
    int32_t to[SETS];  // page, or -1: it stays where it is
#pragma unroll
    for (int k = 0; k < SETS; ++k) {
      const uint32_t page = src[k] < 0 ? 0u : min((uint32_t)src[k], a.num_pages - 1), slot = a.slot_of(from[k]);
      x[k] = *(const u32x4*)(codes + a.sh.code(page, slot, h));
      z[k] = scales[scale_at(page, slot)];
      m[k] = has_mass && (uint32_t)src[k] < a.num_pages ? a.pool.mass[a.sh.row(page, slot, h)] : 0.f;
      const uint32_t i = i0 + k * per + r;
      to[k] = i < a.keep && from[k] != i && (uint32_t)dst[k] < a.num_pages ? dst[k] : -1;
      from[k] = from1[k];
    }
    if (i0 + rows < a.keep) {  // (uniform)
      pages(i0 + rows, from);
      places(i0 + 2 * rows, from1);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (this wave's rows are here, then every wave's are)
    __syncthreads();
#pragma unroll
    for (int k = 0; k < SETS; ++k) {
      if (to[k] < 0) continue;
      const uint32_t slot = a.slot_of(row_of_set(i0, k));
      *(u32x4*)(codes + a.sh.code((uint32_t)to[k], slot, h)) = x[k];
      scales[scale_at((uint32_t)to[k], slot)] = z[k];
      if (has_mass) a.pool.mass[a.sh.row((uint32_t)to[k], slot, h)] = m[k];
    }
  }
}

int evict_check(const char* fn, g4_kv4_params& p, uint32_t keep) {
  p.num_rows = p.num_seqs;
  p.max_rows = 1;
  p.num_q_heads = p.num_kv_heads;
  int rc = g4_internal_kv8_check(fn, p, nullptr);
  if (rc) return rc;
  G4_REQUIRE(keep > 0 && keep <= p.max_seq_len, "%s: keep %u not in 1..max_seq_len (%u)", fn, keep, p.max_seq_len);
  G4_REQUIRE((uint64_t)p.num_seqs * p.num_kv_heads * keep < 1ull << 40, "%s: %u sequences of %u heads and %u rows", fn,
             p.num_seqs, p.num_kv_heads, keep);
  return G4_OK;
}

template <int HD>
void prologue(g4_ctx* ctx, dim3 grid, const ProArgs& a) {
  const bool table = a.rope_cs, moved = a.positions;
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(PT), 0, ctx->stream, a); };
  if (table && moved) go(kv4_prologue_kernel<HD, true, true>);
  else if (table) go(kv4_prologue_kernel<HD, true, false>);
  else if (moved) go(kv4_prologue_kernel<HD, false, true>);
  else go(kv4_prologue_kernel<HD, false, false>);
}

}  // namespace

extern "C" {

int g4_pagedAttnPrologue4(g4_ctx* ctx, const float* q_parts, const float* k_parts, const float* v_parts,
                          uint32_t nparts, const uint16_t* q_norm_w, const uint16_t* k_norm_w,
                          const uint16_t* rope_freqs, float* q_out, uint8_t* k_pool, uint8_t* v_pool,
                          uint8_t* k_scale, uint8_t* v_scale, const int32_t* page_table, const uint32_t* seq_lens,
                          const uint32_t* row_starts, const uint32_t* positions, float* mass, g4_kv4_params p,
                          const float* rope_cs, uint32_t rope_rows) {
  G4_ENTER(ctx);
  int rc = g4_internal_kv8_check(__func__, p, row_starts);
  if (rc) return rc;
  const bool q = q_parts != nullptr, kv = k_parts != nullptr;
  G4_REQUIRE((q || kv) && nparts >= 1 && seq_lens, "g4_pagedAttnPrologue4: no rows, no parts or null seq_lens");
  G4_REQUIRE(!q || (q_norm_w && q_out), "g4_pagedAttnPrologue4: q_parts, q_norm_w and q_out go together");
  G4_REQUIRE(!q || q_out != q_parts || nparts == 1, "g4_pagedAttnPrologue4: q_out over q_parts needs one part");
  G4_REQUIRE(kv ? (v_parts && k_norm_w && k_pool && v_pool && k_scale && v_scale && page_table) : !v_parts,
             "g4_pagedAttnPrologue4: k_parts, v_parts, k_norm_w, the pools, their scales and the page table go together");
  G4_REQUIRE((((uintptr_t)q_parts | (uintptr_t)k_parts | (uintptr_t)v_parts | (uintptr_t)q_out) & 15) == 0 &&
                 (!kv || (((uintptr_t)k_pool | (uintptr_t)v_pool) & 15) == 0),
             "g4_pagedAttnPrologue4: rows and pools must be 16-byte aligned");
  G4_REQUIRE(!rope_cs || (((positions && rope_rows) || rope_rows >= p.max_seq_len) && ((uintptr_t)rope_cs & 7) == 0),
             "g4_pagedAttnPrologue4: RoPE table of %u rows < max_seq_len %u, or not 8-byte aligned", rope_rows,
             p.max_seq_len);
  G4_REQUIRE(!p.apply_divisor || rope_freqs || rope_cs, "g4_pagedAttnPrologue4: apply_divisor needs rope_freqs");
  ProArgs a{};
  a.q = q_parts;
  a.k = k_parts;
  a.v = v_parts;
  a.nparts = nparts;
  a.q_w = q_norm_w;
  a.k_w = k_norm_w;
  a.rope_freqs = rope_freqs ? rope_freqs : (q ? q_norm_w : k_norm_w);  // read, used only with the divisor
  a.rope_cs = (const float2*)rope_cs;
  a.q_out = q_out;
  a.page_table = page_table;
  a.rows = {seq_lens, row_starts, p.num_seqs, p.num_rows, p.max_rows, p.max_seq_len};
  a.nqh = p.num_q_heads;
  a.nkh = p.num_kv_heads;
  a.page_size = p.page_size;
  a.max_pages = p.max_pages;
  a.num_pages = p.num_pages;
  a.eps = p.eps;
  a.theta = p.theta;
  a.apply_divisor = p.apply_divisor;
  a.positions = positions;
  a.most_position = rope_cs ? rope_rows : ~0u;
  a.pool = {k_pool, v_pool, k_scale, v_scale, kv ? mass : nullptr};
  const uint64_t kv_blocks = kv ? ceil_div(2ull * p.num_rows * p.num_kv_heads, PT / 64) : 0u;
  const uint64_t q_waves = q ? (uint64_t)p.num_rows * ceil_div(p.num_q_heads, QH) : 0ull;
  a.kv_blocks = (uint32_t)kv_blocks;
  const dim3 grid((unsigned)(kv_blocks + ceil_div(q_waves, PT / 64)));  // (at most 65535 rows of 2^11 waves)
  switch (p.head_dim) {
    case 64: prologue<64>(ctx, grid, a); break;
    case 128: prologue<128>(ctx, grid, a); break;
    case 256: prologue<256>(ctx, grid, a); break;
    default: prologue<512>(ctx, grid, a); break;
  }
  G4_LAUNCHED(ctx, "kv4_prologue");
  return G4_OK;
}

int g4_kvEvict4_workspace_size(g4_kv4_params p, uint32_t keep, size_t* bytes) {
  G4_REQUIRE(bytes, "g4_kvEvict4_workspace_size: null out");
  int rc = evict_check(__func__, p, keep);
  if (rc) return rc;
  *bytes = ((size_t)p.num_seqs * sizeof(uint32_t) + 15) / 16 * 16;
  return G4_OK;
}

int g4_kvEvict4(g4_ctx* ctx, uint8_t* k_pool, uint8_t* v_pool, uint8_t* k_scale, uint8_t* v_scale, float* mass,
                const int32_t* page_table, uint32_t* seq_lens, g4_kv4_params p, uint32_t keep, uint32_t first,
                uint32_t recent, int32_t* kept, void* workspace, size_t workspace_bytes) {
  G4_ENTER(ctx);
  G4_REQUIRE(k_pool && v_pool && k_scale && v_scale && mass && page_table && seq_lens && kept && workspace,
             "g4_kvEvict4: null buffer");
  int rc = evict_check(__func__, p, keep);
  if (rc) return rc;
  G4_REQUIRE(first <= keep && recent <= keep - first, "g4_kvEvict4: first %u and recent %u are more than keep %u",
             first, recent, keep);
  G4_REQUIRE((((uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)workspace) & 15) == 0,
             "g4_kvEvict4: pools and workspace must be 16-byte aligned");
  size_t need = 0;
  rc = g4_kvEvict4_workspace_size(p, keep, &need);
  if (rc) return rc;
  G4_REQUIRE(workspace_bytes >= need, "g4_kvEvict4: workspace %zu bytes < %zu required", workspace_bytes, need);
  const uint64_t pairs = (uint64_t)p.num_seqs * p.num_kv_heads;
  G4_REQUIRE(pairs <= 65535, "g4_kvEvict4: %u sequences of %u KV heads in one call", p.num_seqs, p.num_kv_heads);
  // As few pieces a workgroup as fill the device: one CU's address units bound a workgroup (one sequence of 2048 rows at
  // head dim 512 in 8 workgroups 9.3 us, 8 of 4000 rows and two heads at 128 in 32 of them 19).
  uint32_t some = std::min(p.head_dim / 32, 4u);
  while (some > 1 && pairs * 2 * (p.head_dim / 32 / some) < 256) some /= 2;
  const uint32_t tiles = p.page_size / 16;
  const EvictArgs a{{k_pool, v_pool, k_scale, v_scale, mass},
                    {p.page_size, p.num_kv_heads, p.head_dim},
                    page_table, seq_lens, p.num_seqs, p.max_pages, p.num_pages, p.max_seq_len, keep, first, recent,
                    kept, (uint32_t*)workspace, some, tiles, tiles == 1 ? 0u : (uint32_t)(((1ull << 32) + tiles - 1) / tiles),
                    tiles == 1 ? ~0u : 0u};
  hipLaunchKernelGGL(kv4_select_kernel, dim3((unsigned)pairs), dim3(ST), 0, ctx->stream, a);
  G4_LAUNCHED(ctx, "kv4_select");
  const dim3 moves((unsigned)((pairs + 7) / 8 * 8) * 2 * (p.head_dim / 32 / some));
  hipLaunchKernelGGL(kv4_move_kernel, moves, dim3(ST), 0, ctx->stream, a);
  G4_LAUNCHED(ctx, "kv4_move");
  return G4_OK;
}

int g4_kv4Values(g4_ctx* ctx, const uint8_t* k_pool, const uint8_t* v_pool, const uint8_t* k_scale,
                 const uint8_t* v_scale, const int32_t* pages, uint32_t count, uint32_t page_size,
                 uint32_t num_kv_heads, uint32_t head_dim, uint32_t num_pages, uint16_t* k_out, uint16_t* v_out) {
  G4_ENTER(ctx);
  G4_REQUIRE(k_pool && v_pool && k_scale && v_scale && pages && k_out && v_out, "g4_kv4Values: null buffer");
  G4_REQUIRE((((uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0,
             "g4_kv4Values: pools and outputs must be 16-byte aligned");
  g4_kv4_params p{};
  p.num_seqs = p.num_rows = p.max_rows = p.max_pages = p.max_seq_len = 1;
  p.num_q_heads = p.num_kv_heads = num_kv_heads;
  p.head_dim = head_dim;
  p.page_size = page_size;
  p.num_pages = num_pages;
  int rc = g4_internal_kv8_check(__func__, p, nullptr);
  if (rc) return rc;
  G4_REQUIRE(count > 0 && count < (1ull << 32) / VT, "g4_kv4Values: %u pages", count);
  const ValArgs a{{k_pool, v_pool}, {k_scale, v_scale}, {k_out, v_out}, pages, {page_size, num_kv_heads, head_dim},
                  num_pages};
  const dim3 grid(count, ceil_div((uint64_t)page_size * num_kv_heads * head_dim, 16 * VT), 2);
  hipLaunchKernelGGL(kv4_values_kernel, grid, dim3(VT), 0, ctx->stream, a);
  G4_LAUNCHED(ctx, "kv4_values");
  return G4_OK;
}

}  // extern "C"
