// k_attn8.hip — attention over the 8-bit paged K/V pool (k_kv8.hip writes it)
// on the gfx950 matrix cores.
//
//   S[pos][col] = scale * scale_k[page] * (code_k[pos] . q[col]),
//   out[col] = sum P[pos][col] * scale_v[page] * code_v[pos] / sum P,  P = softmax of S,
//
// a column being one query row and head of a KV head. Both products read the
// codes as they are stored or as exact f16:
//  * scores: v_mfma_i32_16x16x64_i8 of 16 K rows by 64 dims straight from the
//    pool's bytes. q is a 24-bit integer per element (times a power of two of
//    its column) in three signed 8-bit digits, so a score is exact integer
//    arithmetic, rounded to f32 when its three sums are joined: no conversion
//    of K, and q keeps 24 bits below its largest element.
//  * P V: v_mfma_f32_16x16x32_f16, P * 2^15 as f16 hi and, times 2^11 more, its
//    rest lo, in products of their own: 22 bits of every P down to 2^-40 of the
//    row's largest (one pair in one sum, lo not scaled, has them down to 2^-16
//    only: a far key's share is then 1e-3 off where the near ones' values are 0).
//    The V codes are exact in f16. P also carries its page's scale relative to
//    the larger of the step's two pages, which scales the f32 sum.
// Sums over steps are f32. Pages hold whole 16-row tiles, so a tile has one
// page id and one scale, and its rows are in the pool whatever the length.
#include <algorithm>
#include <type_traits>

#include "mm_operand.hpp"

#include "kv8.hpp"

namespace {

using namespace g4kv8;

using g4mm::f4;
using g4mm::h2;
using g4mm::h8;
using g4mm::static_for;
typedef int i4 __attribute__((ext_vector_type(4)));

constexpr int COLS = 16;                 // columns of a matrix product
constexpr float kLog2e = 1.44269504f;    // the softmax works in powers of two
constexpr float kPScale = 32768.f, kLoScale = 2048.f;

struct Args {
  const float* q;
  const int8_t *kp, *vp;
  const float *ks, *vs;
  const int32_t* page_table;
  Rows rows;
  uint32_t nqh, nkh, G, page_tiles, page_magic, page_same, max_pages, num_pages, window;
  float scale;
  float* out;
  uint32_t wgs;   // workgroups that share the work
  uint2* meta;    // per sequence and KV head: the workgroups that hold its partials
  float* part;    // their partials
};

__device__ __forceinline__ float exp2_h(float x) { return __builtin_amdgcn_exp2f(x); }

// Wave-uniform values into scalar registers.
__device__ __forceinline__ uint32_t uni(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint64_t uni(uint64_t x) {
  return (uint64_t)uni((uint32_t)(x >> 32)) << 32 | uni((uint32_t)x);
}

// Page (of the sequence's list) that holds tile t: t < 2^26, at most 64 tiles
// a page, so t times the rounded-up 2^32 / tiles is off by less than a tile
// (one tile a page: a magic of 0 and all of t).
__device__ __forceinline__ uint32_t page_of(const Args& a, uint32_t t) {
  return __umulhi(t, a.page_magic) + (t & a.page_same);
}
// A wave-uniform word that no kernel of the launch writes, by a scalar load:
// it does not queue behind the vector loads in flight.
template <typename T>
__device__ __forceinline__ T scalar_load(const T* p) {
  return *(const __attribute__((address_space(4))) T*)(uintptr_t)p;
}
__device__ __forceinline__ uint32_t clamp_page(const Args& a, int32_t pg) {
  return pg < 0 ? 0u : min((uint32_t)pg, a.num_pages - 1);
}
__device__ __forceinline__ uint32_t page_id(const Args& a, uint32_t s, uint32_t index) {
  return clamp_page(a, a.page_table[(size_t)s * a.max_pages + index]);
}

// First position (of a whole tile) that any row of the sequence sees.
__device__ __forceinline__ uint32_t first_seen(const Args& a, const Seq& q) {
  return a.window && q.base + 1 > a.window ? (q.base + 1 - a.window) & ~15u : 0u;
}

// The power of two that makes the largest |q| of a column a 24-bit integer of
// at most 0x7f7f7f (three signed digits), and its inverse; NaN where it is not finite.
__device__ __forceinline__ float digit_scale(float am, float& inverse) {
  int ex = 0;
  const float m = frexpf(am, &ex);
  const int k = am > 0.f ? min(max((m > 0.99f ? 22 : 23) - ex, -120), 120) : 0;
  const bool fin = am < INFINITY;
  inverse = fin ? ldexpf(1.0f, -k) : __builtin_nanf("");
  return fin ? ldexpf(1.0f, k) : 0.f;
}
// x as its three signed digits, one a byte (the top byte 0): x + 0x808080 has
// the digits plus 128 as its bytes.
__device__ __forceinline__ uint32_t digits(float x) {
  return ((uint32_t)(int)rintf(x) + 0x808080u) ^ 0x808080u;
}
// Bytes `d` of four such words as one.
template <int D>
__device__ __forceinline__ uint32_t plane(uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3) {
  constexpr uint32_t sel = 0x0c0c0000u | (D << 8) | (4 + D);
  const uint32_t lo = __builtin_amdgcn_perm(x0, x1, sel), hi = __builtin_amdgcn_perm(x2, x3, sel);
  return lo | (hi << 16);
}
// Codes (byte B of two words) as f16: 0x6400 | (code + 128) is 1152 + code.
template <int B>
__device__ __forceinline__ h2 two_codes(uint32_t x0, uint32_t x1) {
  const uint32_t x = __builtin_amdgcn_perm(x1, x0, 0x0c000c00u | ((4 + B) << 16) | B) ^ 0x64806480u;
  return __builtin_bit_cast(h2, x) + h2{(_Float16)-1152.f, (_Float16)-1152.f};
}

// ---------------------------------------------------------------------------
// few rows a sequence (a decode step): rows * query heads per KV head <= 16
// ---------------------------------------------------------------------------
//
// HBM bounds it: every K and V byte goes from the pool to a wave's registers
// once, in the matrix operands' order (no LDS): a lane's 16 bytes of a K row
// are its A operand, and its HD / 16 neighbouring dims of 8 V rows become the
// B operands of HD / 16 products, dim HD / 16 * c + e in product e.
//
// The positions of all sequences, in units of 128, are dealt to the workgroups
// in equal shares whatever the lengths (a share may end in one sequence and go
// on in the next), 32 positions at a time to each of the four waves. A sequence
// held by one workgroup is written by it; else its workgroups leave partials
// (max, sum, o), which attn8_merge_kernel adds in order.
constexpr int NT = 256, UNIT = 128;
template <int HD>
struct StepShape {
  static constexpr uint32_t WGS = HD == 512 ? 256 : 512;  // one or two per CU (registers)
  static constexpr uint32_t SLOT = COLS * (HD + 2);       // floats of a partial: max, sum [16], o [16][HD]
};

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

template <int HD>
__global__ __launch_bounds__(NT, HD == 512 ? 1 : 2) void attn8_step_kernel(Args a) {
  constexpr int VB = HD / 16, KJ = HD / 64;
  __shared__ __align__(16) uint32_t s_q[3 * KJ * 64 * 4];  // digits as B operands: [digit][64 dims][lane] 16 B
  __shared__ __align__(16) float s_o[4 * COLS * HD];
  __shared__ float s_m[4 * COLS], s_l[4 * COLS], s_un[COLS];
  const int tid = threadIdx.x, l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), qd = l >> 4, c = l & 15;
  const uint32_t S = a.rows.num_seqs, wg = blockIdx.x;

  // The sequences 64 at a time, one a lane (in every wave alike): their units
  // summed up, T in all; then those that hold this workgroup's share.
  Seq mine{};
  uint32_t c0 = 0, mine_units = 0, incl = 0, total = 0;
  auto load_chunk = [&](uint32_t first) {
    c0 = first;
    mine = first + l < S ? seq_rows(a.rows, first + l) : Seq{0, 0, 0, 0};
    mine_units = mine.len ? (mine.len - first_seen(a, mine) + UNIT - 1) / UNIT : 0u;
    incl = wave_scan(mine_units * a.nkh);
    total = __builtin_amdgcn_readlane(incl, 63);
  };
  uint32_t T = 0;
  for (uint32_t first = 0; first < S; first += 64) {
    load_chunk(first);
    T += total;
  }
  const Share sh{T, min(a.wgs, T)};
  const uint32_t ub = wg < sh.W ? sh.first(wg) : 0u, ue = wg < sh.W ? sh.first(wg + 1) : 0u;
  uint32_t before = 0;  // units before the chunk
  if (S > 64 && ub < ue) {
    for (load_chunk(0); before + total <= ub; load_chunk(c0 + 64)) before += total;
  }

  uint32_t u = ub;
  while (u < ue) {
    while (before + total <= u) {  // (u < T: a later chunk holds it)
      before += total;
      load_chunk(c0 + 64);
    }
    const int at = __ffsll((unsigned long long)__ballot(before + incl > u)) - 1;
    const uint32_t s = c0 + at;
    const Seq sq{pick(mine.first, at), pick(mine.n, at), pick(mine.base, at), pick(mine.len, at)};
    const uint32_t units = pick(mine_units, at), seq0 = before + pick(incl, at) - units * a.nkh;
    const uint32_t lo = first_seen(a, sq), end = sq.len;
    const uint32_t kvh = a.nkh == 1 ? 0u : uni((u - seq0) / units);
    const uint32_t seg = seq0 + kvh * units;  // its first unit
    const uint32_t off = u - seg, take = min(units - off, ue - u);
    const uint32_t ncols = sq.n * a.G;
    const size_t rs = (size_t)a.nkh * HD;

    i4 K[2][KJ];
    uint32_t V[8][VB / 4];
    float ks[2], vs[2];
    // page ids of the next step and, on their way, of the one after it
    int32_t pg[2], pg_far[2];
    const uint32_t st1 = 4 * (off + take), tiles = (end - lo + 15) / 16, t0 = lo / 16;
    const uint32_t k_at = c * (uint32_t)rs + 16 * qd, v_at = 4 * qd * (uint32_t)rs + VB * c;
    const int32_t* list = a.page_table + (size_t)s * a.max_pages;
    auto pages = [&](uint32_t st, int32_t* to) {
#pragma unroll
      for (int p = 0; p < 2; ++p) to[p] = scalar_load(list + page_of(a, t0 + min(2 * st + p, tiles - 1)));
    };
    auto tile_at = [&](const int8_t* pool, uint32_t st, int p) -> const int8_t* {  // the tile's first row
      const uint32_t t = t0 + min(2 * st + p, tiles - 1), slot = (t - page_of(a, t) * a.page_tiles) * 16;
      return (const int8_t*)uni(
          (uint64_t)(pool + ((size_t)clamp_page(a, pg[p]) * (a.page_tiles * 16) + slot) * rs + kvh * HD));
    };
    auto load_k = [&](uint32_t st) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int8_t* base = tile_at(a.kp, st, p);
#pragma unroll
        for (int j = 0; j < KJ; ++j) K[p][j] = *(const i4*)(base + k_at + 64 * j);
        ks[p] = scalar_load(a.ks + (size_t)clamp_page(a, pg[p]) * a.nkh + kvh);
      }
    };
    auto load_v = [&](uint32_t st) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int8_t* base = tile_at(a.vp, st, p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t* r = (const uint32_t*)(base + i * rs + v_at);
          if constexpr (VB >= 16) {
#pragma unroll
            for (int k = 0; k < VB / 16; ++k) {
              const i4 x = *(const i4*)(r + 4 * k);
#pragma unroll
              for (int e = 0; e < 4; ++e) V[4 * p + i][4 * k + e] = (uint32_t)x[e];
            }
          } else {
#pragma unroll
            for (int e = 0; e < VB / 4; ++e) V[4 * p + i][e] = r[e];
          }
        }
        vs[p] = scalar_load(a.vs + (size_t)clamp_page(a, pg[p]) * a.nkh + kvh);
      }
    };

    uint32_t st = 4 * off + w;
    const uint32_t steps = min(st1, (tiles + 1) / 2);  // (the last unit may be short)
    if (st < steps) {
      pages(st, pg);
      load_k(st);
      load_v(st);
      pages(min(st + 4, steps - 1), pg);
    }
    // ---- q's digits: 16 threads a column ----
    __syncthreads();  // the previous sequence's are done with
    {
      constexpr int E = HD / 16;
      const uint32_t col = tid >> 4, part = tid & 15, cc = min(col, ncols - 1);
      const float* qg = a.q + ((size_t)(sq.first + cc / a.G) * a.nqh + kvh * a.G + cc % a.G) * HD + part * E;
      float x[E], am = 0.f;
      bool nan = false;
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        const f4 y = *(const f4*)(qg + e);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[e + i] = y[i];
          am = fmaxf(am, fabsf(y[i]));
          nan |= y[i] != y[i];
        }
      }
      am = g4d::max16(nan ? INFINITY : am);
      float un;
      const float up = digit_scale(am, un);
      if (part == 0) s_un[col] = un;
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        uint32_t d[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = digits(up > 0.f ? x[e + i] * up : 0.f);
        const uint32_t dim = part * E + e;
        uint32_t* dst = s_q + (((dim / 64) * 64 + dim % 64 / 16 * 16 + col) * 4 + dim % 16 / 4);
        dst[0] = plane<0>(d[0], d[1], d[2], d[3]);
        dst[KJ * 256] = plane<1>(d[0], d[1], d[2], d[3]);
        dst[2 * KJ * 256] = plane<2>(d[0], d[1], d[2], d[3]);
      }
    }
    __syncthreads();
    // this lane's column: positions clo .. clo + width - 1
    const float s_scale = s_un[c] * (a.scale * kLog2e);
    const uint32_t cpos = sq.base + c / a.G;
    const uint32_t clo = a.window && cpos + 1 > a.window ? cpos + 1 - a.window : 0u;
    const uint32_t width = (uint32_t)c < ncols ? cpos + 1 - clo : 0u;
    f4 O[VB];
#pragma unroll
    for (int e = 0; e < VB; ++e) O[e] = f4{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.f;  // of column c
    for (; st < steps; st += 4) {
      const uint32_t next = min(st + 4, steps - 1);  // (past the end: its own last rows again, not used)
      asm volatile("" ::: "memory");  // q's digits stay in LDS (in registers they would spill)
      // ---- scores ----
      i4 D[2][3];
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int d = 0; d < 3; ++d) D[p][d] = i4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < KJ; ++j)
#pragma unroll
        for (int d = 0; d < 3; ++d) {
          const i4 B = *(const i4*)(s_q + ((d * KJ + j) * 64 + l) * 4);
#pragma unroll
          for (int p = 0; p < 2; ++p) D[p][d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(K[p][j], B, D[p][d], 0, 0, 0);
        }
      const float sc[2] = {s_scale * ks[0], s_scale * ks[1]};
      pages(min(st + 8, steps - 1), pg_far);
      load_k(next);
      // ---- softmax over the step's 32 positions ----
      const uint32_t pb = lo + 32 * st + 4 * qd;
      float x[8], mx = -INFINITY;
      auto live = [&](int k) { return pb + 16 * (k / 4) + k % 4 - clo < width; };
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = fmaf((float)((D[p][2][i] << 8) + D[p][1][i]), 256.f, (float)D[p][0][i]);
          x[4 * p + i] = v;
          mx = fmaxf(mx, live(4 * p + i) ? v * sc[p] : -INFINITY);
        }
      mx = g4d::xmax32(g4d::xmax16(mx));
      const float m_new = fmaxf(m_run, mx), m_fin = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = exp2_h(m_run - m_fin);
      const float vmax = fmaxf(vs[0], vs[1]);
      const float vr[2] = {vs[0] / vmax * kPScale, vs[1] / vmax * kPScale};
      float ps = 0.f;
      h8 ph, pl;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float e = live(k) ? exp2_h(fmaf(x[k], sc[k / 4], -m_fin)) : 0.f;
        ps += e;
        const float es = live(k) ? e * vr[k / 4] : 0.f;
        ph[k] = (_Float16)es;
        pl[k] = (_Float16)((es - (float)ph[k]) * kLoScale);
      }
      ps = g4d::xsum32(g4d::xsum16(ps));
      l_run = l_run * alpha + ps;
      m_run = m_new;
      if (__ballot(alpha != 1.f)) {
        float ar[4];  // O's rows are columns 4 qd + i
#pragma unroll
        for (int i = 0; i < 4; ++i) ar[i] = __shfl(alpha, 4 * qd + i, 64);
#pragma unroll
        for (int e = 0; e < VB; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) O[e][i] *= ar[i];
      }
      // ---- P V ----
      const float back = vmax * (1.f / kPScale), back_lo = back * (1.f / kLoScale);
      auto product = [&](auto e) __attribute__((always_inline)) {
        constexpr int b = decltype(e)::value % 4, k = decltype(e)::value / 4;
        h8 B;
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const h2 y = two_codes<b>(V[j][k], V[j + 1][k]);
          B[j] = y[0];
          B[j + 1] = y[1];
        }
        const f4 zero = f4{0.f, 0.f, 0.f, 0.f};
        const f4 lo = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, B, zero, 0, 0, 0);
        const f4 hi = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, B, zero, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          O[decltype(e)::value][i] = fmaf(hi[i], back, fmaf(lo[i], back_lo, O[decltype(e)::value][i]));
        if constexpr (decltype(e)::value % 2 == 1) __builtin_amdgcn_sched_barrier(0);
      };
      static_for<VB>(product);
      load_v(next);
#pragma unroll
      for (int p = 0; p < 2; ++p) pg[p] = pg_far[p];
    }

    // ---- the four waves' sums, in their order ----
    if (qd == 0) {
      s_m[w * COLS + c] = m_run;
      s_l[w * COLS + c] = l_run;
    }
    // O of column 4 qd + i, dims VB c .. + VB - 1: groups of four dims turned by c, so that the 16 lanes meet
    // different banks
    constexpr int QG = VB / 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (4u * qd + i < ncols) {
        float* o = s_o + (w * COLS + 4 * qd + i) * HD + VB * c;
#pragma unroll
        for (int e = 0; e < QG; ++e)
          *(f4*)(o + 4 * ((e + c) % QG)) = f4{O[4 * e][i], O[4 * e + 1][i], O[4 * e + 2][i], O[4 * e + 3][i]};
      }
    }
    __syncthreads();
    const bool whole = take == units;
    const uint32_t slot = 2 * wg + (u == ub ? 0u : 1u);
    float* part = a.part + (size_t)slot * StepShape<HD>::SLOT;
    for (uint32_t i = tid; i < ncols * (HD / 4); i += NT) {
      const uint32_t col = i / (HD / 4), d = i % (HD / 4) * 4;
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) M = fmaxf(M, s_m[k * COLS + col]);
      f4 y = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float m = s_m[k * COLS + col];
        const float f = m == -INFINITY ? 1.f : exp2_h(m - M);  // (-Inf: sums of 0, or NaN)
        L += s_l[k * COLS + col] * f;
        y += *(const f4*)(s_o + (k * COLS + col) * HD + d / VB * VB + 4 * ((d % VB / 4 + d / VB) % QG)) * f;
      }
      float* o = whole ? a.out + ((size_t)(sq.first + col / a.G) * a.nqh + kvh * a.G + col % a.G) * HD
                       : part + 2 * COLS + col * HD;
      *(f4*)(o + d) = whole ? y * (1.0f / L) : y;
      if (!whole && d == 0) {
        part[col] = M;
        part[COLS + col] = L;
      }
    }
    if (off == 0 && tid == 0) a.meta[(size_t)s * a.nkh + kvh] = make_uint2(slot, sh.owner(seg + units - 1));
    u += take;
  }
  // rows that see nothing
  for (uint32_t i = wg; i < S * a.nkh; i += gridDim.x) {
    const Seq q = seq_rows(a.rows, i / a.nkh);
    if (q.len || !q.n) continue;
    for (uint32_t d = tid; d < q.n * a.G * HD; d += NT)
      a.out[((size_t)(q.first + d / (a.G * HD)) * a.nqh + i % a.nkh * a.G) * HD + d % (a.G * HD)] = 0.f;
  }
}

// Adds the partials of one column: those of workgroup meta.x / 2 (slot meta.x)
// and of the ones up to meta.y (slot 0 of each), in this order over groups of
// threads: group g takes every NG-th, then the groups are added in order.
template <int HD, int MT>
__global__ __launch_bounds__(MT) void attn8_merge_kernel(Args a) {
  constexpr int TG = HD / 4, NG = MT / TG, MS = 4;  // threads a partial row, groups, loads in flight of each
  __shared__ float s_m[NG], s_l[NG];
  __shared__ __align__(16) float s_o[NG * HD];
  const uint32_t cols = a.rows.max_rows * a.G, col = blockIdx.x % cols;
  const uint32_t sh = blockIdx.x / cols, s = sh / a.nkh, kvh = sh % a.nkh;
  const Seq q = seq_rows(a.rows, s);
  if (!q.len || col >= q.n * a.G) return;
  const uint2 mt = a.meta[sh];
  const uint32_t w0 = mt.x / 2, n = mt.y - w0 + 1;
  if (n == 1) return;  // written by its workgroup
  const uint32_t g = threadIdx.x / TG, d = threadIdx.x % TG * 4;
  auto slot = [&](uint32_t i) -> const float* {
    return a.part + (size_t)(i ? 2 * (w0 + i) : mt.x) * StepShape<HD>::SLOT;
  };
  float m = -INFINITY, l = 0.f;
  f4 o = f4{0.f, 0.f, 0.f, 0.f};
  for (uint32_t i0 = g; i0 < n; i0 += NG * MS) {
    float pm[MS], pl[MS];
    f4 po[MS];
#pragma unroll
    for (int k = 0; k < MS; ++k) {
      const float* p = slot(min(i0 + NG * k, n - 1));
      pm[k] = p[col];
      pl[k] = p[COLS + col];
      po[k] = *(const f4*)(p + 2 * COLS + col * HD + d);
    }
    float mn = m;
#pragma unroll
    for (int k = 0; k < MS; ++k) mn = fmaxf(mn, i0 + NG * k < n ? pm[k] : -INFINITY);
    const float mf = mn == -INFINITY ? 0.f : mn, al = exp2_h(m - mf);
    l *= al;
    o *= al;
#pragma unroll
    for (int k = 0; k < MS; ++k) {
      if (i0 + NG * k >= n) continue;
      const float f = pm[k] == -INFINITY ? 1.f : exp2_h(pm[k] - mf);  // (-Inf: sums of 0, or NaN)
      l += f * pl[k];
      o += f * po[k];
    }
    m = mn;
  }
  if (d == 0) {
    s_m[g] = m;
    s_l[g] = l;
  }
  *(f4*)(s_o + g * HD + d) = o;
  __syncthreads();
  if (g) return;
  float M = -INFINITY, L = 0.f;
  for (int i = 0; i < NG; ++i) M = fmaxf(M, s_m[i]);
  f4 y = f4{0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < NG; ++i) {
    const float f = s_m[i] == -INFINITY ? 1.f : exp2_h(s_m[i] - M);
    L += f * s_l[i];
    y += f * *(const f4*)(s_o + i * HD + d);
  }
  const float inv = 1.0f / L;
  *(f4*)(a.out + ((size_t)(q.first + col / a.G) * a.nqh + kvh * a.G + col % a.G) * HD + d) = y * inv;
}

// One workgroup per row and query head: 256 positions at a time, one score a
// thread, then one or two output dims a thread.
template <int HD>
__global__ __launch_bounds__(NT) void attn8_kernel(Args a) {
  __shared__ float s_q[512], s_p[NT], s_red[8];
  __shared__ int s_pg[NT];
  const uint32_t row = blockIdx.y, head = blockIdx.x, kvh = head / a.G, t = threadIdx.x, ps_ = a.page_tiles * 16;
  const uint32_t s = seq_of_row(a.rows, row);
  if (s >= a.rows.num_seqs) return;
  const Seq sq = seq_rows(a.rows, s);
  if (!sq.n) return;
  float* out = a.out + ((size_t)row * a.nqh + head) * HD;
  const uint32_t end = sq.len ? sq.base + (row - sq.first) + 1 : 0u;
  const uint32_t lo = a.window && end > a.window ? end - a.window : 0u;
  for (uint32_t d = t; d < HD; d += NT) s_q[d] = a.q[((size_t)row * a.nqh + head) * HD + d];
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (uint32_t p0 = lo; p0 < end; p0 += NT) {
    const uint32_t pos = min(p0 + t, end - 1);
    const uint32_t pg = page_id(a, s, pos / ps_);
    __syncthreads();
    s_pg[t] = pg;
    const int8_t* k = a.kp + (((size_t)pg * ps_ + pos % ps_) * a.nkh + kvh) * HD;
    float x = 0.f;
    for (uint32_t d = 0; d < HD; ++d) x = fmaf(s_q[d], (float)k[d], x);
    x = p0 + t < end ? x * a.scale * a.ks[(size_t)pg * a.nkh + kvh] : -INFINITY;
    const float mx = g4d::wave_max(x);
    if ((t & 63) == 0) s_red[t >> 6] = mx;
    __syncthreads();
    float mn = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    mn = fmaxf(m, mn);
    const float al = m == mn ? 1.f : expf(m - mn);
    const float p = p0 + t < end ? expf(x - mn) : 0.f;
    s_p[t] = p;
    const float ps = g4d::wave_sum(p);
    if ((t & 63) == 0) s_red[4 + (t >> 6)] = ps;
    __syncthreads();
    l = l * al + ((s_red[4] + s_red[5]) + (s_red[6] + s_red[7]));
    m = mn;
    o0 *= al;
    o1 *= al;
    const uint32_t n = min((uint32_t)NT, end - p0);
    for (uint32_t i = 0; i < n; ++i) {
      const int32_t g = s_pg[i];
      const int8_t* v = a.vp + (((size_t)g * ps_ + (p0 + i) % ps_) * a.nkh + kvh) * HD;
      const float w = s_p[i] * a.vs[(size_t)g * a.nkh + kvh];
      if (t < HD) o0 = fmaf(w, (float)v[t], o0);
      if (t + NT < HD) o1 = fmaf(w, (float)v[t + NT], o1);
    }
  }
  if (t < HD) out[t] = end ? o0 / l : 0.f;
  if (t + NT < HD) out[t + NT] = end ? o1 / l : 0.f;
}

bool step_fits(const g4_kv8_params& p) {
  return (uint64_t)p.max_rows * (p.num_q_heads / p.num_kv_heads) <= COLS;
}
// Units a sequence may have (a window of several rows spans max_rows - 1 more positions, and up to 15 of its first tile).
uint64_t most_units(const g4_kv8_params& p) {
  uint64_t span = p.max_seq_len;
  if (p.sliding_window) span = std::min<uint64_t>(span, (uint64_t)p.sliding_window + p.max_rows - 1 + 15);
  return (span + UNIT - 1) / UNIT;
}
size_t meta_bytes(const g4_kv8_params& p) {
  return ((size_t)p.num_seqs * p.num_kv_heads * sizeof(uint2) + 255) / 256 * 256;
}
template <int HD>
uint32_t step_wgs(const g4_kv8_params& p) {
  return (uint32_t)std::min<uint64_t>(StepShape<HD>::WGS, most_units(p) * p.num_seqs * p.num_kv_heads);
}
template <int HD>
size_t step_bytes(const g4_kv8_params& p) {
  return meta_bytes(p) + 2ull * step_wgs<HD>(p) * StepShape<HD>::SLOT * sizeof(float);
}

template <int HD>
int attend(g4_ctx* ctx, const g4_kv8_params& p, Args a, void* workspace) {
  if (step_fits(p)) {
    G4_REQUIRE(most_units(p) * p.num_seqs * p.num_kv_heads < (1ull << 31),
               "g4_pagedAttn8: %u sequences of up to %u positions and %u KV heads in one call", p.num_seqs,
               p.max_seq_len, p.num_kv_heads);
    a.wgs = step_wgs<HD>(p);
    a.meta = (uint2*)workspace;
    a.part = (float*)((uint8_t*)workspace + meta_bytes(p));
    hipLaunchKernelGGL(attn8_step_kernel<HD>, dim3(a.wgs), dim3(NT), 0, ctx->stream, a);
    G4_LAUNCHED(ctx, "attn8_step");
    const uint64_t units = most_units(p);
    if (units == 1) return G4_OK;  // no sequence has partials
    const dim3 grid(p.num_seqs * p.num_kv_heads * p.max_rows * a.G);
    if (std::min<uint64_t>(units, a.wgs) <= 32)
      hipLaunchKernelGGL((attn8_merge_kernel<HD, 256>), grid, dim3(256), 0, ctx->stream, a);
    else
      hipLaunchKernelGGL((attn8_merge_kernel<HD, 1024>), grid, dim3(1024), 0, ctx->stream, a);
    G4_LAUNCHED(ctx, "attn8_merge");
    return G4_OK;
  }
  hipLaunchKernelGGL(attn8_kernel<HD>, dim3(p.num_q_heads, p.num_rows), dim3(NT), 0, ctx->stream, a);
  G4_LAUNCHED(ctx, "attn8");
  return G4_OK;
}

}  // namespace

extern "C" {

int g4_pagedAttn8_workspace_size(g4_kv8_params p, size_t* bytes) {
  G4_REQUIRE(bytes, "g4_pagedAttn8_workspace_size: null out");
  int rc = g4_internal_kv8_check(__func__, p, p.max_rows == 1 && p.num_rows == p.num_seqs ? nullptr : &p.num_rows);
  if (rc) return rc;
  *bytes = 256;
  if (step_fits(p))
    *bytes = p.head_dim == 64 ? step_bytes<64>(p) : p.head_dim == 128 ? step_bytes<128>(p)
             : p.head_dim == 256 ? step_bytes<256>(p) : step_bytes<512>(p);
  return G4_OK;
}

int g4_pagedAttn8(g4_ctx* ctx, const float* q, const int8_t* k_pool, const int8_t* v_pool, const float* k_scale,
                  const float* v_scale, const int32_t* page_table, const uint32_t* seq_lens,
                  const uint32_t* row_starts, float* output, g4_kv8_params p, void* workspace,
                  size_t workspace_bytes) {
  G4_ENTER(ctx);
  G4_REQUIRE(q && k_pool && v_pool && k_scale && v_scale && page_table && seq_lens && output && workspace,
             "g4_pagedAttn8: null buffer");
  int rc = g4_internal_kv8_check(__func__, p, row_starts);
  if (rc) return rc;
  size_t need = 0;
  rc = g4_pagedAttn8_workspace_size(p, &need);
  if (rc) return rc;
  G4_REQUIRE(workspace_bytes >= need, "g4_pagedAttn8: workspace %zu bytes < %zu required", workspace_bytes, need);
  G4_REQUIRE((((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)output | (uintptr_t)workspace) & 15) == 0,
             "g4_pagedAttn8: rows, pools and workspace must be 16-byte aligned");
  const uint32_t tiles = p.page_size / 16;
  const Args a{q, k_pool, v_pool, k_scale, v_scale, page_table,
               {seq_lens, row_starts, p.num_seqs, p.num_rows, p.max_rows, p.max_seq_len},
               p.num_q_heads, p.num_kv_heads, p.num_q_heads / p.num_kv_heads, tiles,
               tiles == 1 ? 0u : (uint32_t)(((1ull << 32) + tiles - 1) / tiles), tiles == 1 ? ~0u : 0u, p.max_pages, p.num_pages, p.sliding_window, p.scale,
               output, 0, nullptr, nullptr};
  switch (p.head_dim) {
    case 64: return attend<64>(ctx, p, a, workspace);
    case 128: return attend<128>(ctx, p, a, workspace);
    case 256: return attend<256>(ctx, p, a, workspace);
    default: return attend<512>(ctx, p, a, workspace);
  }
}

}  // extern "C"
