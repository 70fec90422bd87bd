// k_kv4.hip — appending to the 4-bit paged K/V pool, reading its values, and
// evicting rows by their attention weight (no counterpart in the reference).
//
// A value is an e2m1 code times 2^e, one e per 32 dims of a row and head: the
// least with |x| <= 7 * 2^e. Between 6 and 7 the nearest of 6 and the 8 that a
// wider code would have is 6, so every element is within 2^e of its code, and of
// the bounds from 6 to 8 this one has the least mean square error for normal
// values: 0.112 of their deviation, against 0.115 at 6 and at 8. Each row has its
// own scales: nothing is ever rounded again, whatever comes after it or moves it.
#include <algorithm>

#include "attn_paged.hpp"
#include "kv4.hpp"
#include "kv_rows.hpp"

namespace {

using namespace g4kv8;
using g4kv4::BAD;
using g4kv4::BLOCK;

constexpr int PT = 256;    // threads of the append
constexpr int QH = 2;      // q heads of a wave
constexpr int VT = 256;    // of the values kernel
constexpr int ST = 1024;   // of the selection
constexpr int MT = 256;    // of the moves
constexpr uint32_t CACHED = 32768;  // candidates whose masses are held in LDS

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

// A wave a row and head of K or of V; other workgroups take q's rows.
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

// 16 codes a thread.
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
// it and the first of those at it are listed in order. kv4_gather_kernel copies
// the rows that move to the workspace, kv4_scatter_kernel to their places: a row
// moves down only, so its place may be where another comes from.
struct EvictArgs {
  g4kv4::Pool pool;
  g4kv4::Shape sh;
  const int32_t* page_table;
  uint32_t* seq_lens;
  uint32_t num_seqs, max_pages, num_pages, max_seq_len, keep, first, recent;
  int32_t* kept;
  uint32_t* cut;   // per sequence: whether it is cut
  uint8_t* rows;   // what moves: codes [num_seqs][nkh][keep][hd], then scales [..][hd / 16], then masses
  uint8_t* scales;
  float* mass;
};

__device__ __forceinline__ uint32_t key_of(float x) { return x > 0.f ? __float_as_uint(x) : 0u; }

__global__ __launch_bounds__(ST) void kv4_select_kernel(EvictArgs a) {
  constexpr int NW = ST / 64, BINS = 2 * ST, FAR = 8;  // FAR: masses on their way
  __shared__ uint32_t s_key[CACHED];
  __shared__ uint32_t s_bin[BINS], s_above[NW], s_at[NW], s_found[2];
  const uint32_t tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
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
  const int32_t* list = a.page_table + (size_t)s * a.max_pages;
  auto fetch = [&](uint32_t i) -> uint32_t {
    const uint32_t t = a.first + i;
    const int32_t pg = list[t / a.sh.page_size];
    const float x = a.pool.mass[a.sh.row(pg < 0 ? 0u : min((uint32_t)pg, a.num_pages - 1), t % a.sh.page_size, h)];
    return pg >= 0 && pg < (int32_t)a.num_pages ? key_of(x) : 0u;
  };
  for (uint32_t i0 = tid; i0 < min(n, CACHED); i0 += FAR * ST) {
    uint32_t k[FAR];
#pragma unroll
    for (int j = 0; j < FAR; ++j) k[j] = fetch(min(i0 + j * ST, n - 1));
#pragma unroll
    for (int j = 0; j < FAR; ++j)
      if (i0 + j * ST < min(n, CACHED)) s_key[i0 + j * ST] = k[j];
  }
  auto key = [&](uint32_t i) -> uint32_t { return i < CACHED ? s_key[i] : fetch(i); };
  uint32_t bound = 0, left = m;  // the m-th largest key so far; how many of those that share its bits are kept
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;  // 11, 11 and 10 bits
    s_bin[2 * tid] = s_bin[2 * tid + 1] = 0;
    __syncthreads();
    for (uint32_t i0 = 0; i0 < n; i0 += ST) {  // (every lane: the first one's bin is counted by one of them)
      const uint32_t i = i0 + tid, k = i < n ? key(i) : 0u;
      const bool in = i < n && (pass == 0 || (k ^ bound) >> (pass == 1 ? 21 : 10) == 0);
      const uint32_t b = k >> shift & (pass == 2 ? 1023u : 2047u);
      const uint64_t some = __ballot(in);
      if (!some) continue;
      const int one = __ffsll((unsigned long long)some) - 1;
      const uint32_t b1 = __builtin_amdgcn_readlane(b, one);
      const uint64_t same = __ballot(in && b == b1);
      if (lane == (uint32_t)one) atomicAdd(&s_bin[b1], (uint32_t)__popcll(same));
      else if (in && b != b1) atomicAdd(&s_bin[b], 1u);
    }
    __syncthreads();
    // counts from the largest bin down: two bins a thread, summed over its wave, then over the waves
    const uint32_t hi = s_bin[BINS - 1 - 2 * tid], lo = s_bin[BINS - 2 - 2 * tid];
    const uint32_t upto = wave_scan(hi + lo);
    if (lane == 63) s_above[w] = upto;
    __syncthreads();
    uint32_t above = upto - hi - lo;
    for (uint32_t i = 0; i < w; ++i) above += s_above[i];
    if (above < left && above + hi + lo >= left) {  // (one thread's)
      const bool first = above + hi >= left;
      s_found[0] = BINS - 1 - 2 * tid - (first ? 0 : 1);
      s_found[1] = above + (first ? 0 : hi);
    }
    __syncthreads();
    bound |= s_found[0] << shift;
    left -= s_found[1];
  }
  // the rows above the bound and the first `left` at it, in order: each wave counts those of its run of candidates
  const uint32_t run = ((n + NW - 1) / NW + 63) / 64 * 64, i0 = min(w * run, n), i1 = min(i0 + run, n);
  uint32_t above = 0, at = 0;
  for (uint32_t i = i0; i < i1; i += 64) {
    const uint32_t k = i + lane < i1 ? key(i + lane) : 0u;
    above += __popcll(__ballot(i + lane < i1 && k > bound));
    at += __popcll(__ballot(i + lane < i1 && k == bound));
  }
  __syncthreads();  // (s_above's counts of the last pass are done with)
  if (lane == 0) {
    s_above[w] = above;
    s_at[w] = at;
  }
  __syncthreads();
  above = at = 0;
  for (uint32_t i = 0; i < w; ++i) {
    above += s_above[i];
    at += s_at[i];
  }
  const uint64_t below = (1ull << lane) - 1;
  for (uint32_t i = i0; i < i1; i += 64) {
    const bool in = i + lane < i1;
    const uint32_t k = in ? key(i + lane) : 0u;
    const uint64_t ma = __ballot(in && k > bound), me = __ballot(in && k == bound);
    const uint32_t ra = above + __popcll(ma & below), re = at + __popcll(me & below);
    if (in && (k > bound || (k == bound && re < left)))
      kept[a.first + ra + min(re, left)] = (int32_t)(a.first + i + lane);
    above += __popcll(ma);
    at += __popcll(me);
  }
}

// A thread 16 bytes of codes (K's, then V's) and one scale of a row; the row's first also its mass.
template <bool BACK>
__global__ __launch_bounds__(MT) void kv4_move_kernel(EvictArgs a) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const uint32_t pieces = a.sh.hd / 16, half = pieces / 2, per = MT / pieces;
  const uint32_t s = blockIdx.y / a.sh.nkh, h = blockIdx.y % a.sh.nkh;
  if (!a.cut[s]) return;
  const uint32_t i = blockIdx.x * per + threadIdx.x / pieces, piece = threadIdx.x % pieces;
  if (!BACK && i == 0 && threadIdx.x == 0 && h == 0) a.seq_lens[s] = a.keep;
  if (i >= a.keep) return;
  const size_t at = (size_t)blockIdx.y * a.keep + i;
  const uint32_t from = (uint32_t)a.kept[at];
  if (from == i) return;
  const uint32_t t = BACK ? i : from;
  const int32_t id = a.page_table[(size_t)s * a.max_pages + t / a.sh.page_size];
  const bool in = id >= 0 && id < (int32_t)a.num_pages;
  if (BACK && !in) return;
  const uint32_t pg = id < 0 ? 0u : min((uint32_t)id, a.num_pages - 1), slot = t % a.sh.page_size;
  const bool is_v = piece >= half;
  const uint32_t b = is_v ? piece - half : piece;
  u32x4* code = (u32x4*)((is_v ? a.pool.v : a.pool.k) + a.sh.code(pg, slot, h) + 16 * b);
  uint8_t* scale = is_v ? a.pool.vs + a.sh.v_scale(pg, slot, h, b) : a.pool.ks + a.sh.k_scale(pg, slot, h, b);
  u32x4* code_w = (u32x4*)(a.rows + at * a.sh.hd + 16 * piece);
  uint8_t* scale_w = a.scales + at * pieces + piece;
  float* mass = a.pool.mass + a.sh.row(pg, slot, h);
  if (BACK) {
    *code = *code_w;
    *scale = *scale_w;
    if (piece == 0) *mass = a.mass[at];
  } else {
    *code_w = *code;
    *scale_w = *scale;
    if (piece == 0) a.mass[at] = in ? *mass : 0.f;
  }
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }
struct EvictSizes {
  size_t cut, rows, scales, mass;
  size_t all() const { return cut + rows + scales + mass; }
};
EvictSizes evict_sizes(const g4_kv4_params& p, uint32_t keep) {
  const size_t n = (size_t)p.num_seqs * p.num_kv_heads * keep;
  return {up256(p.num_seqs * 4ull), up256(n * p.head_dim), up256(n * (p.head_dim / 16)), up256(n * 4)};
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
  *bytes = evict_sizes(p, keep).all();
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
  const EvictSizes z = evict_sizes(p, keep);
  G4_REQUIRE(workspace_bytes >= z.all(), "g4_kvEvict4: workspace %zu bytes < %zu required", workspace_bytes, z.all());
  const uint64_t pairs = (uint64_t)p.num_seqs * p.num_kv_heads;
  G4_REQUIRE(pairs <= 65535, "g4_kvEvict4: %u sequences of %u KV heads in one call", p.num_seqs, p.num_kv_heads);
  uint8_t* w = (uint8_t*)workspace;
  const EvictArgs a{{k_pool, v_pool, k_scale, v_scale, mass},
                    {p.page_size, p.num_kv_heads, p.head_dim},
                    page_table, seq_lens, p.num_seqs, p.max_pages, p.num_pages, p.max_seq_len, keep, first, recent,
                    kept, (uint32_t*)w, w + z.cut, w + z.cut + z.rows, (float*)(w + z.cut + z.rows + z.scales)};
  hipLaunchKernelGGL(kv4_select_kernel, dim3((unsigned)pairs), dim3(ST), 0, ctx->stream, a);
  G4_LAUNCHED(ctx, "kv4_select");
  const dim3 grid(ceil_div(keep, MT / (p.head_dim / 16)), (unsigned)pairs);
  hipLaunchKernelGGL(kv4_move_kernel<false>, grid, dim3(MT), 0, ctx->stream, a);
  G4_LAUNCHED(ctx, "kv4_gather");
  hipLaunchKernelGGL(kv4_move_kernel<true>, grid, dim3(MT), 0, ctx->stream, a);
  G4_LAUNCHED(ctx, "kv4_scatter");
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
