// k_kv8.hip — appending to the 8-bit paged K/V pool, and reading its values
// (the f16 pool's prologue is attn_prologue_kernel of k_attn.hip; the
// reference appends f32 rows, shaders/kv_cache_store.wgsl).
//
// A value is code * 2^e with one e per page and KV head. Powers of two: a value
// divided by the scale is exact, so the code is the correctly rounded one, and
// when a later row makes the scale grow, the codes already there are shifted
// and rounded once, to at most half a step of the new scale. After the norms a
// page's largest element stays within an octave, so growth is rare; the price
// is up to one bit against a scale of amax / 127.
//
// kv8_prologue_kernel: every page of a KV head that a call touches belongs to
// one workgroup (K and V apart), which forms its rows' largest element before
// it stores any code; other workgroups take the query rows, a wave some heads of
// one. Norms, rotation and rounding of K and V are in f64: a value near the
// border of two codes then gets the same code as in exact arithmetic, whatever
// the order of the sums (the f64 units are idle otherwise). q is f32. The rows a
// wave keeps stay in registers between the two steps; where a page has more they
// are formed again for the second.
//
// A step's append is bound by latency, and much of that by instructions, which a
// launch finds in no cache: 27 KB of code (loops unrolled, the rotation without a
// table in line, library square root, division and frexp, maxima in f64 through
// LDS) took 8.3 us for 64 sequences, the same steps in 8 KB 4.0. A prompt of 1900
// rows at head dim 512 (72 MB, 15 us at a copy's rate) takes 18.1 to 18.7.
#include "kv8.hpp"
#include "mqf_core.hpp"

namespace {

using namespace g4kv8;

constexpr int VT = 256;  // threads of the values kernel

struct ProArgs {
  const float *q, *k, *v;
  uint32_t nparts;
  const uint16_t *q_w, *k_w;
  const uint16_t* rope_freqs;
  const float2* rope_cs;
  float* q_out;
  int8_t *kp, *vp;
  float *ks, *vs;
  const int32_t* page_table;
  Rows rows;
  uint32_t nqh, nkh, page_size, max_pages, num_pages;
  uint32_t kv_blocks, seq_pages;  // workgroups of the pages; pages a sequence's rows may touch
  float eps, theta;
  uint32_t apply_divisor;
};

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
__device__ __forceinline__ void load_turn(const ProArgs& a, uint32_t pos, int lane, Turn<HD>& t) {
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
template <int HD, int NT, int QH, bool TABLE>
__device__ __forceinline__ void q_row(const ProArgs& a, uint32_t block) {
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
  if (!q.len) return;
  Turn<HD> t;
  load_turn<HD, TABLE>(a, q.base + (row - q.first), lane, t);
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

// The least e >= -64 with x <= 127 * 2^e, of a double's magnitude bits: the binary
// exponent less 7, one more where the fraction passes that of 127 / 128. kBad
// where it is not finite.
constexpr int kBad = 1000;
__device__ __forceinline__ int exponent_of(uint64_t bits) {
  constexpr uint64_t carry = (1ull << 52) - 1 - 0xfc00000000000ull;
  return bits >= 0x7ffull << 52 ? kBad : max((int)((bits + carry) >> 52) - 1022 - 7, -64);
}
__device__ __forceinline__ uint64_t magnitude(double x) { return __builtin_bit_cast(uint64_t, x) & ~(1ull << 63); }
// 1 / sqrt(x), from the hardware's estimate by two steps of Newton's iteration.
__device__ __forceinline__ double rsqrt64(double x) {
  double y = __builtin_amdgcn_rsq(x);
#pragma unroll
  for (int i = 0; i < 2; ++i) y = fma(y * 0.5, fma(-x * y, y, 1.0), y);
  return y;
}

// KEEP rows a wave; 1 where no sequence of the call has more than there are waves.
template <int HD, int NT, int KEEP, int QH, bool TABLE>
__global__ __launch_bounds__(NT, 4) void kv8_prologue_kernel(ProArgs a) {
  constexpr int PP = Row<HD>::PP, HALF = Row<HD>::HALF, NW = NT / 64;
  __shared__ float s_e[NW];
  if (blockIdx.x >= a.kv_blocks) {  // (the pages, which take longer, start first)
    q_row<HD, NT, QH, TABLE>(a, blockIdx.x - a.kv_blocks);
    return;
  }
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  uint32_t b = blockIdx.x;
  const bool is_v = b & 1;
  b >>= 1;
  const uint32_t kvh = b % a.nkh;
  b /= a.nkh;
  const uint32_t j = b % a.seq_pages, s = b / a.seq_pages;
  const Seq q = seq_rows(a.rows, s);
  const uint32_t pi = q.base / a.page_size + j;
  if (!q.len || pi > (q.len - 1) / a.page_size) return;  // (uniform)
  const int32_t pg = a.page_table[(size_t)s * a.max_pages + pi];
  const uint32_t start = pi * a.page_size;
  const uint32_t p0 = max(q.base, start), p1 = min(q.len, start + a.page_size), m = p1 - p0;
  const float* src = (is_v ? a.v : a.k);
  const size_t stride = (size_t)a.rows.num_rows * a.nkh * HD;

  double lo[KEEP][PP], hi[KEEP][PP];
  Weights<HD> wt;
  Turn<HD> turn[KEEP];
  if (!is_v) load_weights<HD>(a.k_w, lane, wt);
  auto load = [&](uint32_t at) {  // the wave's rows p0 + at + w, + NW, ... (past the last: 0)
#pragma unroll
    for (int r = 0; r < KEEP; ++r) {
      const uint32_t i = at + w + NW * r;
      if (i < m) {  // (uniform over the wave)
        load_row<HD>(src + ((size_t)(q.first + (p0 - q.base) + i) * a.nkh + kvh) * HD, stride, a.nparts, lane, lo[r],
                     hi[r]);
        if (!is_v) load_turn<HD, TABLE>(a, p0 + i, lane, turn[r]);
      } else {
#pragma unroll
        for (int e = 0; e < PP; ++e) lo[r][e] = hi[r][e] = 0.0;
      }
    }
  };
  auto form = [&](uint32_t at) {
    double ss[KEEP];
#pragma unroll
    for (int r = 0; r < KEEP; ++r) {
      ss[r] = 0.0;
#pragma unroll
      for (int e = 0; e < PP; ++e) ss[r] = fma(lo[r][e], lo[r][e], fma(hi[r][e], hi[r][e], ss[r]));
    }
#pragma unroll
    for (int r = 0; r < KEEP; ++r) ss[r] = g4d::wave_sum_dpp(ss[r]);
#pragma unroll
    for (int r = 0; r < KEEP; ++r) {
      if (at + w + NW * r >= m) continue;
      const double inv = rsqrt64(ss[r] * (1.0 / HD) + (double)a.eps);
#pragma unroll
      for (int e = 0; e < PP; ++e) {
        lo[r][e] *= inv;
        hi[r][e] *= inv;
      }
      if (!is_v) rotate<HD>(wt, turn[r], lo[r], hi[r]);
    }
  };
  load(0);
  if (pg < 0 || pg >= (int32_t)a.num_pages) return;
  float* sp = (is_v ? a.vs : a.ks) + (size_t)pg * a.nkh + kvh;
  const uint32_t before = p0 - start;  // codes of earlier calls
  const float old = before ? *sp : 0.f;
  uint64_t am = 0;  // the lane's largest magnitude (an infinity and a NaN are larger than any number)
  for (uint32_t at = 0; at < m; at += KEEP * NW) {
    if (KEEP > 1 && at) load(at);
    form(at);
#pragma unroll
    for (int r = 0; r < KEEP; ++r)
#pragma unroll
      for (int e = 0; e < PP; ++e) am = max(am, max(magnitude(lo[r][e]), magnitude(hi[r][e])));
    if (KEEP == 1) break;
  }
  const float ew = g4d::wave_max_dpp((float)exponent_of(am));
  if (lane == 0) s_e[w] = ew;
  __syncthreads();  // (and every thread has read the scale)
  float ex = s_e[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) ex = fmaxf(ex, s_e[i]);
  const bool poison = ex == (float)kBad || old != old;
  const float sc = poison ? __builtin_nanf("") : fmaxf(old, __uint_as_float((uint32_t)(min((int)ex, 127) + 127) << 23));
  if (threadIdx.x == 0) *sp = sc;
  int8_t* page = (is_v ? a.vp : a.kp) + ((size_t)pg * a.page_size * a.nkh + kvh) * HD;
  const size_t rs = (size_t)a.nkh * HD;  // from one position's row to the next

  if (before && sc != old && !poison) {  // (uniform) round the codes before to the grown scale
    const float ratio = old / sc;
    for (uint32_t i = threadIdx.x; i < before * (HD / 4); i += NT) {
      uint32_t* d = (uint32_t*)(page + (size_t)(i / (HD / 4)) * rs + i % (HD / 4) * 4);
      const uint32_t x = *d;
      uint32_t y = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float c = rintf((float)(int8_t)(x >> (8 * e)) * ratio);
        y |= ((uint32_t)(int)fminf(fmaxf(c, -127.f), 127.f) & 0xffu) << (8 * e);
      }
      *d = y;
    }
  }
  const double up = (double)__uint_as_float(0x7f000000u - __float_as_uint(sc));  // 1 / sc
  for (uint32_t at = 0; at < m; at += KEEP * NW) {
    if (KEEP > 1 && m > KEEP * NW) {
      load(at);
      form(at);
    }
#pragma unroll
    for (int r = 0; r < KEEP; ++r) {
      const uint32_t i = at + w + NW * r;
      if (i >= m || lane >= Row<HD>::ACT) continue;
      int8_t* d = page + (size_t)(before + i) * rs + PP * lane;
      uint32_t x = 0, y = 0;
#pragma unroll
      for (int e = 0; e < PP; ++e) {
        x |= (poison ? 0u : (uint32_t)(int)rint(lo[r][e] * up) & 0xffu) << (8 * e);
        y |= (poison ? 0u : (uint32_t)(int)rint(hi[r][e] * up) & 0xffu) << (8 * e);
      }
      if constexpr (PP == 1) {
        d[0] = (int8_t)x;
        d[HALF] = (int8_t)y;
      } else if constexpr (PP == 2) {
        *(uint16_t*)d = (uint16_t)x;
        *(uint16_t*)(d + HALF) = (uint16_t)y;
      } else {
        *(uint32_t*)d = x;
        *(uint32_t*)(d + HALF) = y;
      }
    }
    if (KEEP == 1) break;
  }
}

struct ValArgs {
  const int8_t* pool[2];
  const float* scale[2];
  uint16_t* out[2];
  const int32_t* pages;
  uint32_t page_size, nkh, hd, num_pages;
};

// 16 codes a thread. A code times its scale has 7 bits: exact in f16 from
// 2^-24 to 65504.
__global__ __launch_bounds__(VT) void kv8_values_kernel(ValArgs a) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const uint32_t bytes = a.page_size * a.nkh * a.hd;  // of a page
  const uint32_t i = (blockIdx.y * VT + threadIdx.x) * 16;
  if (i >= bytes) return;
  const uint32_t which = blockIdx.z;
  const int32_t pg = a.pages[blockIdx.x];
  const bool in = pg >= 0 && pg < (int32_t)a.num_pages;
  const size_t at = (size_t)(in ? pg : 0) * bytes + i;
  const u32x4 x = *(const u32x4*)(a.pool[which] + at);
  const float sc = in ? a.scale[which][(size_t)pg * a.nkh + i / a.hd % a.nkh] : 0.f;
  u32x4 y[2];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t b = x[e / 2] >> (16 * (e & 1));
    y[e / 4][e % 4] = (uint32_t)g4d::f32_to_f16_bits((float)(int8_t)b * sc) |
                      (uint32_t)g4d::f32_to_f16_bits((float)(int8_t)(b >> 8) * sc) << 16;
  }
  u32x4* o = (u32x4*)(a.out[which] + (size_t)blockIdx.x * bytes + i);
  o[0] = in ? y[0] : u32x4{0, 0, 0, 0};
  o[1] = in ? y[1] : u32x4{0, 0, 0, 0};
}

// The launch: few rows (at most four a sequence), a row and two of q's heads a
// wave (64 sequences 3.9 us, with four heads 4.3); more rows, KEEP of them and four
// heads (1900 rows 18.1 to 18.6 us, with two heads 18.5), in workgroups of four waves
// where a page is 16 rows (chunks of seven prompts at head dim 128 6.6 us, with
// eight waves 7.7; at 256 7.7 and 8.0; 1900 rows alike; 300 rows at 512 alone 10.8
// and 6.8) and eight where it is more (the chunks in pages of 32 7.4 us, four waves
// 12.8; 1900 rows at 256 12.8 and 18.0, in pages of 64 at 512 27.2 and 36.8).
struct Shape {
  int threads, heads;
  bool few;
};
Shape shape_of(const g4_kv8_params& p) {
  if (p.max_rows <= 4) return {256, 2, true};
  return {p.page_size <= 16 ? 256 : 512, 4, false};
}
template <int HD, bool TABLE>
void prologue_of(g4_ctx* ctx, const Shape& s, dim3 grid, const ProArgs& a) {
  constexpr int KEEP = HD == 512 ? 2 : 4;  // (four spill)
  if (s.few) hipLaunchKernelGGL((kv8_prologue_kernel<HD, 256, 1, 2, TABLE>), grid, dim3(256), 0, ctx->stream, a);
  else if (s.threads == 256)
    hipLaunchKernelGGL((kv8_prologue_kernel<HD, 256, KEEP, 4, TABLE>), grid, dim3(256), 0, ctx->stream, a);
  else hipLaunchKernelGGL((kv8_prologue_kernel<HD, 512, KEEP, 4, TABLE>), grid, dim3(512), 0, ctx->stream, a);
}
template <int HD>
void prologue(g4_ctx* ctx, const Shape& s, dim3 grid, const ProArgs& a) {
  if (a.rope_cs) prologue_of<HD, true>(ctx, s, grid, a);
  else prologue_of<HD, false>(ctx, s, grid, a);
}

}  // namespace

int g4_internal_kv8_check(const char* fn, const g4_kv8_params& p, const uint32_t* row_starts) {
  G4_REQUIRE(p.num_seqs > 0 && p.num_seqs <= 65535 && p.num_rows > 0 && p.num_rows <= 65535 && p.max_rows > 0 &&
                 p.max_rows <= p.num_rows,
             "%s: 1..65535 sequences and rows, max_rows (%u) from 1 to num_rows (%u)", fn, p.max_rows, p.num_rows);
  G4_REQUIRE(row_starts || (p.max_rows == 1 && p.num_rows == p.num_seqs),
             "%s: without row_starts every sequence has one row (num_rows = num_seqs, max_rows 1)", fn);
  G4_REQUIRE(p.num_kv_heads > 0 && p.num_q_heads > 0 && p.num_q_heads % p.num_kv_heads == 0 &&
                 p.num_q_heads / p.num_kv_heads <= 16 && p.num_kv_heads <= 64,
             "%s: num_q_heads %u must be a multiple (<= 16x) of num_kv_heads %u (<= 64)", fn, p.num_q_heads,
             p.num_kv_heads);
  G4_REQUIRE(p.head_dim == 64 || p.head_dim == 128 || p.head_dim == 256 || p.head_dim == 512,
             "%s: head_dim %u not in {64, 128, 256, 512}", fn, p.head_dim);
  G4_REQUIRE(p.page_size > 0 && p.page_size % 16 == 0 && p.page_size <= 1024,
             "%s: page_size %u is not a multiple of 16 up to 1024", fn, p.page_size);
  G4_REQUIRE(p.max_pages > 0 && p.num_pages > 0 && p.num_pages <= 0x7fffffffu && p.max_seq_len > 0 &&
                 p.max_seq_len <= (1u << 30) && (uint64_t)p.max_seq_len <= (uint64_t)p.page_size * p.max_pages,
             "%s: max_seq_len %u exceeds the page table (%u x %u) or 2^30", fn, p.max_seq_len, p.max_pages,
             p.page_size);
  G4_REQUIRE((uint64_t)p.num_pages * (p.page_size / 16) < 1ull << 32, "%s: %u pages of %u: 2^36 positions or more", fn,
             p.num_pages, p.page_size);
  return G4_OK;
}

extern "C" {

int g4_pagedAttnPrologue8(g4_ctx* ctx, const float* q_parts, const float* k_parts, const float* v_parts,
                          uint32_t nparts, const uint16_t* q_norm_w, const uint16_t* k_norm_w,
                          const uint16_t* rope_freqs, float* q_out, int8_t* k_pool, int8_t* v_pool, float* k_scale,
                          float* v_scale, const int32_t* page_table, const uint32_t* seq_lens,
                          const uint32_t* row_starts, g4_kv8_params p, const float* rope_cs, uint32_t rope_rows) {
  G4_ENTER(ctx);
  int rc = g4_internal_kv8_check(__func__, p, row_starts);
  if (rc) return rc;
  const bool q = q_parts != nullptr, kv = k_parts != nullptr;
  G4_REQUIRE((q || kv) && nparts >= 1 && seq_lens, "g4_pagedAttnPrologue8: no rows, no parts or null seq_lens");
  G4_REQUIRE(!q || (q_norm_w && q_out), "g4_pagedAttnPrologue8: q_parts, q_norm_w and q_out go together");
  G4_REQUIRE(!q || q_out != q_parts || nparts == 1, "g4_pagedAttnPrologue8: q_out over q_parts needs one part");
  G4_REQUIRE(kv ? (v_parts && k_norm_w && k_pool && v_pool && k_scale && v_scale && page_table) : !v_parts,
             "g4_pagedAttnPrologue8: k_parts, v_parts, k_norm_w, the pools, their scales and the page table go together");
  G4_REQUIRE((((uintptr_t)q_parts | (uintptr_t)k_parts | (uintptr_t)v_parts | (uintptr_t)q_out) & 15) == 0 &&
                 (!kv || (((uintptr_t)k_pool | (uintptr_t)v_pool) & 15) == 0),
             "g4_pagedAttnPrologue8: rows and pools must be 16-byte aligned");
  G4_REQUIRE(!rope_cs || (rope_rows >= p.max_seq_len && ((uintptr_t)rope_cs & 7) == 0),
             "g4_pagedAttnPrologue8: RoPE table of %u rows < max_seq_len %u, or not 8-byte aligned", rope_rows,
             p.max_seq_len);
  G4_REQUIRE(!p.apply_divisor || rope_freqs || rope_cs, "g4_pagedAttnPrologue8: apply_divisor needs rope_freqs");
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
  a.kp = k_pool;
  a.vp = v_pool;
  a.ks = k_scale;
  a.vs = v_scale;
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
  a.seq_pages = ceil_div(p.max_rows - 1, p.page_size) + 1;
  const Shape s = shape_of(p);
  const uint64_t kv_blocks = kv ? 2ull * p.num_seqs * a.seq_pages * p.num_kv_heads : 0ull;
  const uint64_t q_waves = q ? (uint64_t)p.num_rows * ceil_div(p.num_q_heads, s.heads) : 0ull;
  const uint64_t blocks = kv_blocks + ceil_div(q_waves, s.threads / 64);
  G4_REQUIRE(blocks < (1ull << 32) / s.threads,
             "g4_pagedAttnPrologue8: %u sequences of up to %u rows of %u and %u heads in one call", p.num_seqs,
             p.max_rows, p.num_q_heads, p.num_kv_heads);
  a.kv_blocks = (uint32_t)kv_blocks;
  const dim3 grid((unsigned)blocks);
  switch (p.head_dim) {
    case 64: prologue<64>(ctx, s, grid, a); break;
    case 128: prologue<128>(ctx, s, grid, a); break;
    case 256: prologue<256>(ctx, s, grid, a); break;
    default: prologue<512>(ctx, s, grid, a); break;
  }
  G4_LAUNCHED(ctx, "kv8_prologue");
  return G4_OK;
}

int g4_kv8Values(g4_ctx* ctx, const int8_t* k_pool, const int8_t* v_pool, const float* k_scale, const float* v_scale,
                 const int32_t* pages, uint32_t count, uint32_t page_size, uint32_t num_kv_heads, uint32_t head_dim,
                 uint32_t num_pages, uint16_t* k_out, uint16_t* v_out) {
  G4_ENTER(ctx);
  G4_REQUIRE(k_pool && v_pool && k_scale && v_scale && pages && k_out && v_out, "g4_kv8Values: null buffer");
  G4_REQUIRE((((uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0,
             "g4_kv8Values: pools and outputs must be 16-byte aligned");
  g4_kv8_params p{};
  p.num_seqs = p.num_rows = p.max_rows = p.max_pages = p.max_seq_len = 1;
  p.num_q_heads = p.num_kv_heads = num_kv_heads;
  p.head_dim = head_dim;
  p.page_size = page_size;
  p.num_pages = num_pages;
  int rc = g4_internal_kv8_check(__func__, p, nullptr);
  if (rc) return rc;
  G4_REQUIRE(count > 0 && count < (1ull << 32) / VT, "g4_kv8Values: %u pages", count);
  const ValArgs a{{k_pool, v_pool}, {k_scale, v_scale}, {k_out, v_out}, pages, page_size, num_kv_heads, head_dim,
                  num_pages};
  const dim3 grid(count, ceil_div((uint64_t)page_size * num_kv_heads * head_dim, 16 * VT), 2);
  hipLaunchKernelGGL(kv8_values_kernel, grid, dim3(VT), 0, ctx->stream, a);
  G4_LAUNCHED(ctx, "kv8_values");
  return G4_OK;
}

}  // extern "C"
