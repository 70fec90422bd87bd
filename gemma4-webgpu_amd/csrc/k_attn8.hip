// k_attn8.hip — attention over the 8-bit paged K/V pool (k_kv8.hip writes it)
// on the gfx950 matrix cores.
//
//   S[pos][col] = scale * scale_k[page] * (code_k[pos] . q[col]),
//   out[col] = sum P[pos][col] * scale_v[page] * code_v[pos] / sum P,  P = softmax of S,
//
// a column being one query row and head of a KV head. Both products read the
// codes as they are stored or as exact f16:
//  * scores: v_mfma_i32_16x16x64_i8 of 16 K rows by 64 dims straight from the
//    pool's bytes. q is an integer per element (times a power of two of its
//    column, the largest 2^21 .. 2^22) in three signed 8-bit digits, so a score
//    is exact integer arithmetic, rounded to f32 when its three sums are joined:
//    no conversion of K, and q is rounded to 2^-23 of its largest element.
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

#include "attn_paged.hpp"

namespace {

using namespace g4kv8;

using g4mm::h2;
using g4mm::h8;
using g4mm::static_for;
typedef int i4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));

constexpr int COLS = 16;                 // columns of a matrix product
constexpr float kLog2e = 1.44269504f;    // the softmax works in powers of two
constexpr float kPScale = 32768.f, kLoScale = 2048.f;
constexpr float kLeastScale = 0x1p-100f;  // V scales are taken relative to one of at least this (theirs: 2^-64 or 0)

struct Args : PagedArgs {
  const int8_t *kp, *vp;
  const float *ks, *vs;
};

// A V scale, NaN where it is infinite (relative to that one the others would be lost).
__device__ __forceinline__ float finite(float x) { return x < INFINITY ? x : __builtin_nanf(""); }


// The power of two that brings the largest |q| of a column to 2^21 .. 2^22, and
// its inverse; NaN where it is not finite.
__device__ __forceinline__ float digit_scale(float am, float& inverse) {
  int ex = 0;
  (void)frexpf(am, &ex);
  const int k = am > 0.f ? min(max(22 - ex, -120), 120) : 0;
  const bool fin = am < INFINITY;
  inverse = fin ? ldexpf(1.0f, -k) : __builtin_nanf("");
  return fin ? ldexpf(1.0f, k) : 0.f;
}
// x * up, at most 2^22, as three signed digits, one a byte (the top byte is
// not used): 1.5 * 2^23 + x up has the rounded integer in its low bits, and that
// plus 0x808080 the digits plus 128 as its bytes.
__device__ __forceinline__ uint32_t digits(float x, float up) {
  return (__float_as_uint(fmaf(x, up, 12582912.f)) + (0x808080u - 0x4b400000u)) ^ 0x808080u;
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
//
// Measured: 32 long contexts at head dim 512 (362 MB) 78 us, 4.6 TB/s where a copy
// moves 4.7 and reads alone go at 5.3; 64 mixed ones at 256 (93 MB) 24.5 us; one
// window of 512 7.9 us, the latency of a unit (lengths, page ids, rows, products,
// the waves' sums); the partials 3 to 4.8 us more. Units of 1024, so that a window has no partials,
// took 15.6 us instead of 11.4: a wave's step of 32 positions is 1.8 us.
constexpr int NT = 256, UNIT = 128;
template <int HD>
struct StepShape {
  static constexpr uint32_t WGS = HD == 512 ? 256 : 512;  // one or two per CU (registers)
  static constexpr uint32_t SLOT = COLS * (HD + 2);       // floats of a partial: max, sum [16], o [16][HD]
};

template <int HD>
__global__ __launch_bounds__(NT, HD == 512 ? 1 : 2) void attn8_step_kernel(Args a) {
  constexpr int VB = HD / 16, KJ = HD / 64, BL = HD < 256 ? 1 : HD / 256;
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
    // page ids of the next step and, on their way, of the one after it (vector loads, issued before the rows that
    // go before them in use: a scalar load's wait is that of the LDS reads too)
    int32_t pg[2], pg_far[2];
    const uint32_t st1 = 4 * (off + take), tiles = (end - lo + 15) / 16, t0 = lo / 16;
    const uint32_t steps = min(st1, (tiles + 1) / 2);  // (the last unit may be short)
    const uint32_t k_at = c * (uint32_t)rs + 16 * qd, v_at = 4 * qd * (uint32_t)rs + VB * c;
    const int32_t* list = a.page_table + (size_t)s * a.max_pages;
    auto pages = [&](uint32_t st, int32_t* to) {
#pragma unroll
      for (int p = 0; p < 2; ++p) to[p] = list[page_of(a, t0 + min(2 * st + p, tiles - 1))];
    };
    // a tile's rows as a buffer; of no bytes past the last step, so that nothing is read there (a branch around the
    // loads of the next step would spill)
    auto tile_at = [&](const int8_t* pool, uint32_t st, int p) -> __amdgpu_buffer_rsrc_t {
      const uint32_t t = t0 + min(2 * st + p, tiles - 1), slot = (t - page_of(a, t) * a.page_tiles) * 16;
      const size_t row = (size_t)clamp_page(a, uni_i(pg[p])) * (a.page_tiles * 16) + slot;
      const uint64_t at = uni((uint64_t)(pool + row * rs + kvh * HD));
      return __builtin_amdgcn_make_buffer_rsrc((void*)at, (short)0, st < steps ? (int)(15 * (uint32_t)rs + HD) : 0,
                                               0x00020000);
    };
    auto load_scales = [&](float* k, float* v) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const size_t at = (size_t)clamp_page(a, uni_i(pg[p])) * a.nkh + kvh;
        k[p] = a.ks[at];
        v[p] = a.vs[at];
      }
    };
    auto load_k = [&](uint32_t st) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const __amdgpu_buffer_rsrc_t r = tile_at(a.kp, st, p);
#pragma unroll
        for (int j = 0; j < KJ; ++j)
          K[p][j] = __builtin_bit_cast(i4, __builtin_amdgcn_raw_buffer_load_b128(r, k_at + 64 * j, 0, 0));
      }
    };
    auto load_v = [&](uint32_t st) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const __amdgpu_buffer_rsrc_t r = tile_at(a.vp, st, p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (VB >= 16) {
#pragma unroll
            for (int k = 0; k < VB / 16; ++k) {
              const i4 x = __builtin_bit_cast(
                  i4, __builtin_amdgcn_raw_buffer_load_b128(r, v_at + 16 * k, i * (uint32_t)rs, 0));
#pragma unroll
              for (int e = 0; e < 4; ++e) V[4 * p + i][4 * k + e] = (uint32_t)x[e];
            }
          } else {
#pragma unroll
            for (int e = 0; e < VB / 4; ++e)
              V[4 * p + i][e] = __builtin_amdgcn_raw_buffer_load_b32(r, v_at + 4 * e, i * (uint32_t)rs, 0);
          }
        }
      }
    };

    // q, 16 threads a column (asked for before the rows, whose arrival its digits then do not wait for)
    constexpr int E = HD / 16;
    const uint32_t col = tid >> 4, part_of = tid & 15, cc = min(col, ncols - 1);
    const float* qg = a.q + row_of(a, sq.first, kvh, cc) * HD + part_of * E;
    f4 x[E / 4];
#pragma unroll
    for (int e = 0; e < E / 4; ++e) x[e] = *(const f4*)(qg + 4 * e);
    uint32_t st = 4 * off + w;
    // (a wave without a step too, of no bytes: behind a branch q would be waited for together with the rows)
    pages(st, pg);
    pages(min(st + 4, steps - 1), pg_far);  // (before the rows: what comes after them is waited for with them)
    load_scales(ks, vs);
    load_k(st);
    load_v(st);
    pg[0] = pg_far[0];
    pg[1] = pg_far[1];
    // ---- q's digits ----
    __syncthreads();  // the previous sequence's are done with
    {
      float am = 0.f;
      bool nan = false;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        am = fmaxf(am, fabsf(x[e / 4][e % 4]));
        nan |= x[e / 4][e % 4] != x[e / 4][e % 4];
      }
      am = g4d::max16(nan ? INFINITY : am);
      float un;
      const float up = digit_scale(am, un);
      if (part_of == 0) s_un[col] = un;
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        uint32_t d[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = digits(x[e / 4][i], up);
        const uint32_t dim = part_of * E + e;
        uint32_t* dst = s_q + (((dim / 64) * 64 + dim % 64 / 16 * 16 + col) * 4 + dim % 16 / 4);
        dst[0] = plane<0>(d[0], d[1], d[2], d[3]);
        dst[KJ * 256] = plane<1>(d[0], d[1], d[2], d[3]);
        dst[2 * KJ * 256] = plane<2>(d[0], d[1], d[2], d[3]);
      }
    }
    __syncthreads();
    // this lane's column: positions clo .. clo + width - 1
    const float s_scale = s_un[c] * (a.scale * kLog2e);
    const uint32_t cpos = sq.base + div_g(a, c);
    const uint32_t clo = a.window && cpos + 1 > a.window ? cpos + 1 - a.window : 0u;
    const uint32_t width = (uint32_t)c < ncols ? cpos + 1 - clo : 0u;
    f4 O[VB];
#pragma unroll
    for (int e = 0; e < VB; ++e) O[e] = f4{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.f;  // of column c
    for (; st < steps; st += 4) {
      const uint32_t next = st + 4;
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
      float ksn[2], vsn[2];
      load_scales(ksn, vsn);
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
      // (vmax finite where both are NaN: not every column sees them)
      const float v0 = finite(vs[0]), v1 = finite(vs[1]), vmax = fmaxf(fmaxf(v0, v1), kLeastScale);
      const float vr[2] = {v0 / vmax * kPScale, v1 / vmax * kPScale};
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
      for (int p = 0; p < 2; ++p) {
        pg[p] = pg_far[p];
        ks[p] = ksn[p];
        vs[p] = vsn[p];
      }
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
      float* o = whole ? a.out + row_of(a, sq.first, kvh, col) * HD : part + 2 * COLS + col * HD;
      if (whole) y *= 1.0f / L;
      *(f4*)(o + d) = y;
      if constexpr (HD >= 256) {
        if (whole && a.ops)  // (uniform; a wave holds 256 values of one row and head)
          write_ops(a, sq.first + div_g(a, col), (kvh * a.G + col - div_g(a, col) * a.G) * BL + d / 256, l, y);
      }
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
    if (HD >= 256 && a.ops)
      for (uint32_t b = w; b < q.n * a.G * BL; b += NT / 64)
        write_ops(a, q.first + b / (a.G * BL), i % a.nkh * a.G * BL + b % (a.G * BL), l, f4{0.f, 0.f, 0.f, 0.f});
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
  y *= 1.0f / L;
  const uint32_t row = q.first + col / a.G, head = kvh * a.G + col % a.G;
  *(f4*)(a.out + ((size_t)row * a.nqh + head) * HD + d) = y;
  if (HD >= 256 && a.ops) write_ops(a, row, head * (HD / 256) + d / 256, threadIdx.x & 63, y);
}

// ---------------------------------------------------------------------------
// many rows a sequence (prompts, mixed batches)
// ---------------------------------------------------------------------------
//
// Workgroup (64 columns of a sequence and KV head, part of their positions),
// steps of 64 positions through LDS: K as stored, V as f16 in the order of the
// P V product's operand. A wave holds 16 columns: their q digits and output sums
// in registers; two waves per SIMD, so that one's softmax runs beside the
// other's products. The next step's rows are on their way in registers.
//
// Head dim 512 (eight waves): the two waves of a column tile have 256 dims each,
// and 32 of the step's positions each for the softmax: they hand each other
// their integer sums of the other's positions, then their maxima and P, through
// LDS (q's digits of all 512 dims in one wave would spill).
//
// P is f16 hi + lo at 2^15 here, in one sum: its products go into the output
// sums without further arithmetic (sums of their own per step, hi apart from lo,
// cost as many VALU operations as the softmax). That holds P to 22 bits down to
// 2^-17 of the row's largest and to 2^-40 of it below. P also carries the V
// scale of its page relative to the largest of the pages so far.
//
// Page ids and scales come through LDS, 32 steps at a time: scalar loads share
// their counter with LDS reads, so that the products of a step would wait for
// those of the next one.
//
// The steps of all column tiles, and kTileCost more for each tile (its q, its
// output: about as long as so many steps), are dealt to the workgroups in equal
// shares, one or two workgroups a CU: a causal prompt's last tiles are twice the
// average, and a tile each, or tiles cut into parts, leaves CUs idle at the end. A
// tile held by one workgroup is written by it, else its workgroups leave partials
// that attn8_tile_merge_kernel adds in order.
//
// Measured: a prompt of 1900 rows of 8 heads at head dim 512 (29.6 GFLOP of scores
// and P V, 1.75 times that as digits and halves) 94 us, then 12.3 for the 95 MB of
// partials and output, by the trace's kernel times; both together 94 us in passes
// one after the other without it.
constexpr float kNothing = -3e38f;  // the maximum of no positions: finite, so that differences are
template <int HD>
struct TileShape {
  static constexpr bool PAIR = HD == 512;
  static constexpr int NTH = PAIR ? 512 : 256;
  static constexpr int KS = HD + 16;             // K row stride in LDS (bytes): 16 rows on different banks
  static constexpr int KB = TP * KS;
  static constexpr int VB = HD / 16;             // dims of a lane and its row's share
  static constexpr int VBYTES = TP * HD * 2;
  static constexpr int KP = TP * HD / 16 / NTH;  // 16-byte pieces of K a thread and step
  static constexpr int VD = PAIR ? 16 : VB;      // dims a thread moves of 4 positions of V
  static constexpr uint32_t WGS = HD == 512 ? 256 : HD >= 128 ? 512 : 768;  // that run at once (registers, LDS)
  static constexpr uint32_t SLOT = TC * (HD + 2);                           // floats of a partial: max, sum [64], o
};

template <int HD>
__global__ __launch_bounds__(TileShape<HD>::NTH, HD == 64 ? 3 : 2) void attn8_tile_kernel(Args a) {
  using S_ = TileShape<HD>;
  constexpr bool PAIR = S_::PAIR;
  constexpr int KJ = PAIR ? 4 : HD / 64, KP = S_::KP, VD = S_::VD, VB = S_::VB;
  constexpr int NE = PAIR ? 16 : VB;  // products over a wave's dims
  constexpr int PT = PAIR ? 2 : 4;    // tiles of a wave's softmax
  constexpr int CH = 32;              // steps whose tiles and scales are in LDS
  __shared__ __align__(16) int8_t s_k[S_::KB];
  __shared__ __align__(16) uint8_t s_v[S_::VBYTES];
  __shared__ __align__(16) h8 s_p[PAIR ? 4 * 2 * 2 * 64 : 1];  // P: [column tile][32 positions][hi, lo][lane]
  __shared__ __align__(16) i4 s_d[PAIR ? 4 * 2 * 2 * 2 * 64 : 1];  // sums: [column tile][half][tile][part][lane]
  __shared__ float s_mx[PAIR ? 2 * TC : 1];
  __shared__ uint32_t s_tile[4 * CH];
  __shared__ __align__(16) float s_ks[4 * CH], s_vs[4 * CH];
  __shared__ float s_big[2];
  __shared__ uint32_t s_upto[S_::NTH + 1], s_sum[S_::NTH / 64], s_at[2];  // s_upto: units before each thread's run
  __shared__ float s_all[S_::NTH / 64];
  const int tid = threadIdx.x, l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), qd = l >> 4, c = l & 15;
  const int wc = w & 3, wd = PAIR ? w >> 2 : 0;  // column tile; half

  // ---- this workgroup's share of the whole cost: a run of column tiles a thread, summed up ----
  const uint32_t wg = blockIdx.x, pairs = a.rows.num_seqs * a.tiles, run = (pairs + S_::NTH - 1) / S_::NTH;
  const uint32_t j0 = min(tid * run, pairs), j1 = min(j0 + run, pairs);
  uint64_t mine = 0;
  for (uint32_t j = j0; j < j1; ++j) mine += (uint64_t)cost_of(a, j) * a.nkh;
  uint32_t upto = wave_scan((uint32_t)mine);
  const float wave_all = g4d::wave_sum_dpp((float)mine);
  if (l == 63) {
    s_sum[w] = upto;
    s_all[w] = wave_all;
  }
  __syncthreads();
  uint32_t total = 0;
  float all = 0.f;
#pragma unroll
  for (int i = 0; i < S_::NTH / 64; ++i) {
    if (i < w) upto += s_sum[i];
    total += s_sum[i];
    all += s_all[i];
  }
  // Rows that are one sequence's each cost less than 2^31 (checked by the host). Starts that descend in between may
  // give rows to many sequences, past what 32 bits number: nothing is written then, and nothing added up.
  if (all > 3e9f) {  // (uniform)
    for (uint64_t i = (uint64_t)wg * S_::NTH + tid; i < (uint64_t)pairs * a.nkh; i += (uint64_t)gridDim.x * S_::NTH)
      a.meta[i] = make_uint2(0, 0);
    return;
  }
  total = uni(total);
  s_upto[tid + 1] = upto;
  if (tid == 0) s_upto[0] = 0;
  __syncthreads();
  const Share sh{total, min(a.wgs, (total + kLeast - 1) / kLeast)};
  const uint32_t ub = wg < sh.W ? sh.first(wg) : 0u, ue = wg < sh.W ? sh.first(wg + 1) : 0u;
  uint32_t pair = 0, before = 0, used = 0;  // column tile at hand, the units before it; partials written
  auto locate = [&](uint32_t unit) {  // the column tile of a unit, by the thread whose run holds it
    if (s_upto[tid] <= unit && s_upto[tid + 1] > unit) {
      uint32_t j = tid * run, at = s_upto[tid];
      if (run > 1)  // (a run of one is that tile)
        for (uint32_t n; at + (n = cost_of(a, j) * a.nkh) <= unit; ++j) at += n;
      s_at[0] = j;
      s_at[1] = at;
    }
    __syncthreads();
    pair = uni(s_at[0]);
    before = uni(s_at[1]);
    __syncthreads();
  };
  if (ub < ue) locate(ub);

  for (uint32_t u = ub; u < ue;) {
  const uint32_t s = pair / a.tiles, ct = pair % a.tiles;
  const Seq sq = seq_rows(a.rows, s);
  const uint32_t n = uni(sq.n), ncols = n * a.G, base = uni(sq.base), first = uni(sq.first);
  if (!uni(sq.len) || ct * TC >= ncols) {  // behind the sequence's last tile
    locate(u);
    continue;
  }
  const Tile T = tile_of(a, Seq{first, n, base, uni(sq.len)}, ct);
  const uint32_t lo = uni(T.lo), end = uni(T.end), steps = uni(T.steps), cost = kTileCost + steps;
  if (u >= before + cost * a.nkh) {
    before += cost * a.nkh;
    ++pair;
    if (pair >= pairs) locate(u);
    continue;
  }
  const uint32_t kvh = a.nkh == 1 ? 0u : uni((u - before) / cost);
  const uint32_t seg = before + kvh * cost, stop = min(seg + cost, ue);  // the tile's first unit, the last here
  const uint32_t seg0 = seg + kTileCost, st0 = max(u, seg0) - seg0, st1 = max(stop, seg0) - seg0;
  u = stop;
  if (st0 == st1) continue;  // (the share ends before the tile's first step)
  __syncthreads();  // the previous tile's rows are done with
  const size_t rs = (size_t)a.nkh * HD;
  const uint32_t t0 = lo / 16, tlast = (end - 1) / 16;
  const int32_t* list = a.page_table + (size_t)s * a.max_pages;

  // this lane's column
  const uint32_t g = ct * TC + 16 * wc + c, gr = min(g, ncols - 1);
  const uint32_t cpos = base + div_g(a, gr);
  const uint32_t clo = a.window && cpos + 1 > a.window ? cpos + 1 - a.window : 0u;
  const uint32_t width = g < ncols ? cpos + 1 - clo : 0u;
  // positions every column sees: those from the last row's window on, up to the first row's own
  const uint32_t all0 = a.window && end > a.window ? end - a.window : 0u, all1 = base + div_g(a, ct * TC);

  // ---- rows on their way ----
  i4 kr[KP];
  uint32_t vr_[4][VD / 4];
  // This thread's V: positions 4 vq .. + 3 of tile vt, dims from vdim on. Its K pieces: round i in tile kt(i) (the
  // same for all lanes of a wave).
  const int vt = 2 * (PAIR ? (w >> 1) & 1 : w >> 1) + (l >> 5), vq = 2 * (w & 1) + ((l >> 4) & 1);
  const uint32_t vdim = PAIR ? 256 * wd + 16 * c : VB * c;
  constexpr int PR = HD / 16, RPI = S_::NTH / PR;  // pieces of a row, rows of a round
  auto kt = [&](int i) { return RPI == 16 ? i : RPI == 32 ? 2 * i + (w >> 1) : w; };
  uint32_t k_at[KP];
#pragma unroll
  for (int i = 0; i < KP; ++i) k_at[i] = ((i * RPI + tid / PR) % 16) * (uint32_t)rs + tid % PR * 16;
  const uint32_t v_at = 4 * vq * (uint32_t)rs + vdim;
  const int8_t *kp = a.kp + kvh * HD, *vp_ = a.vp + kvh * HD;
  // Tiles (of the pool) and scales of the steps from `st` on; V's relative to the
  // largest so far. Returns what that one grew by (1 / growth).
  float v_ref = kLeastScale;
  auto refill = [&](uint32_t st) __attribute__((always_inline)) -> float {
    float vs = 0.f;
    if (tid < 4 * CH) {
      const uint32_t t = min(t0 + 4 * st + tid, tlast), at = page_of(a, t), pg = clamp_page(a, list[at]);
      const float ks = a.ks[(size_t)pg * a.nkh + kvh], v = a.vs[(size_t)pg * a.nkh + kvh];
      s_tile[tid] = pg * a.page_tiles + (t - at * a.page_tiles);
      vs = finite(v);
      s_ks[tid] = ks;
      const float big = g4d::wave_max_dpp(vs);  // (a NaN is not the larger one)
      if (l == 0) s_big[w] = big;
    }
    __syncthreads();
    const float ref = fmaxf(v_ref, fmaxf(s_big[0], s_big[1])), by = v_ref / ref;
    if (tid < 4 * CH) s_vs[tid] = vs / ref * kTileP;
    __syncthreads();
    v_ref = ref;
    return by;
  };
  // (K as buffers: an address made scalar would be a generic one, whose loads the LDS reads of the step wait for)
  auto load_k = [&](uint32_t k) __attribute__((always_inline)) {  // (of the refilled steps)
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      const uint64_t at = uni((uint64_t)(kp + (size_t)uni(s_tile[4 * k + kt(i)]) * (16 * rs)));
      kr[i] = __builtin_bit_cast(
          i4, __builtin_amdgcn_raw_buffer_load_b128(
                  __builtin_amdgcn_make_buffer_rsrc((void*)at, (short)0, (int)(15 * (uint32_t)rs + HD), 0x00020000),
                  k_at[i], 0, 0));
    }
  };
  auto load_v = [&](uint32_t k) __attribute__((always_inline)) {
    const int8_t* vp = vp_ + (size_t)s_tile[4 * k + vt] * (16 * rs) + v_at;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t* r = (const uint32_t*)(vp + i * rs);
      if constexpr (VD == 16) {
        const i4 x = *(const i4*)r;
#pragma unroll
        for (int e = 0; e < 4; ++e) vr_[i][e] = (uint32_t)x[e];
      } else {
#pragma unroll
        for (int e = 0; e < VD / 4; ++e) vr_[i][e] = r[e];
      }
    }
  };
  // K rows as they are; V [32 positions][product e][lane (q, c)] 16 B: slots 4 (tile & 1) + i of position 4 q + i
  auto store_step = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < KP; ++i) *(i4*)(s_k + (i * RPI + tid / PR) * S_::KS + tid % PR * 16) = kr[i];
    uint8_t* dst = s_v + (((vt >> 1) * (PAIR ? 2 : 1) + wd) * NE * 64 + vq * 16 + c) * 16 + (vt & 1) * 8;
    static_for<VD>([&](auto e) __attribute__((always_inline)) {
      constexpr int k = decltype(e)::value;
      const h2 x = two_codes<k % 4>(vr_[0][k / 4], vr_[1][k / 4]), y = two_codes<k % 4>(vr_[2][k / 4], vr_[3][k / 4]);
      *(g4mm::u32x2*)(dst + k * 1024) = g4mm::u32x2{__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y)};
    });
  };
  const float* qg = a.q + row_of(a, first, kvh, gr) * HD + 16 * qd;
  f4 qx[KJ][4];  // q of this lane's column: dims 64 j + 16 qd .. + 15 (PAIR: from 256 wd on), asked for first
#pragma unroll
  for (int j = 0; j < KJ; ++j)
#pragma unroll
    for (int k = 0; k < 4; ++k) qx[j][k] = *(const f4*)(qg + 256 * wd + 64 * j + 4 * k);
  (void)refill(st0);
  load_k(0);
  load_v(0);

  // ---- q's digits ----
  i4 qb[3][KJ];
  float s_scale;
  {
    float am = 0.f;
    bool nan = false;
    auto largest = [&](const f4& y) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        am = fmaxf(am, fabsf(y[i]));
        nan |= y[i] != y[i];
      }
    };
#pragma unroll
    for (int j = 0; j < KJ; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) largest(qx[j][k]);
    am = g4d::xmax32(g4d::xmax16(nan ? INFINITY : am));
    if constexpr (PAIR) {  // one scale for all 512 dims
      if (qd == 0) s_mx[wd * TC + 16 * wc + c] = am;
      __syncthreads();
      am = fmaxf(am, s_mx[(wd ^ 1) * TC + 16 * wc + c]);
    }
    float un;
    float up = digit_scale(am, un);
    // the joined sums are in units of the second digit; the scale's sign goes to q, a scale of 0 leaves equal scores
    if (a.scale < 0.f) up = -up;
    if (a.scale == 0.f) up = 0.f;
    s_scale = a.scale == 0.f ? un : un * (fabsf(a.scale) * (kLog2e * 256.f));
#pragma unroll
    for (int j = 0; j < KJ; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t d[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = digits(qx[j][k][i], up);
        qb[0][j][k] = (int)plane<0>(d[0], d[1], d[2], d[3]);
        qb[1][j][k] = (int)plane<1>(d[0], d[1], d[2], d[3]);
        qb[2][j][k] = (int)plane<2>(d[0], d[1], d[2], d[3]);
      }
  }

  f4 O[NE];
#pragma unroll
  for (int e = 0; e < NE; ++e) O[e] = f4{0.f, 0.f, 0.f, 0.f};
  float m_run = kNothing, l_run = 0.f;  // of column c (PAIR: l of this wave's positions)

  float ksc[PT], vsc[PT];  // scales of the step at hand: of this wave's tiles
  bool odd;                // whether one of the step's is not finite
  auto turn = [&](uint32_t st, uint32_t next, bool inside) __attribute__((always_inline)) {
    // ---- scores of this wave's PT tiles ----
    float x[PT][4];
    auto score = [&](int p, const i4& hi, const i4& low) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[p][i] = fmaf((float)low[i], 1.f / 256, (float)hi[i]);
    };
    i4 own[PAIR ? 2 : 1][2];
    // (PAIR: the other wave's two tiles first. A tile's rows are read while the one before is multiplied.)
    i4 A[2][KJ];
    const int8_t* ka = s_k + c * S_::KS + 256 * wd + 16 * qd;
    auto read_a = [&](int pp, i4* to) __attribute__((always_inline)) {
      const int p = PAIR ? (2 * (wd ^ 1) + pp) & 3 : pp;
#pragma unroll
      for (int j = 0; j < KJ; ++j) to[j] = *(const i4*)(ka + 16 * p * S_::KS + 64 * j);
    };
    read_a(0, A[0]);
#pragma unroll
    for (int pp = 0; pp < 4; ++pp) {
      if (pp < 3) read_a(pp + 1, A[(pp + 1) & 1]);
      __builtin_amdgcn_sched_barrier(0);
      i4 D[3];
#pragma unroll
      for (int d = 0; d < 3; ++d) D[d] = i4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < KJ; ++j)
#pragma unroll
        for (int d = 0; d < 3; ++d) D[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(A[pp & 1][j], qb[d][j], D[d], 0, 0, 0);
      i4 hi;
#pragma unroll
      for (int i = 0; i < 4; ++i) hi[i] = (D[2][i] << 8) + D[1][i];
      if constexpr (!PAIR) {
        score(pp, hi, D[0]);
      } else if (pp < 2) {
        i4* to = s_d + (((wc * 2 + wd) * 2 + pp) * 2) * 64 + l;
        to[0] = hi;
        to[64] = D[0];
      } else {
        own[pp - 2][0] = hi;
        own[pp - 2][1] = D[0];
      }
    }
    if constexpr (PAIR) {
      __syncthreads();
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const i4* from = s_d + (((wc * 2 + (wd ^ 1)) * 2 + p) * 2) * 64 + l;
        score(p, own[p][0] + from[0], own[p][1] + from[64]);
      }
    }
    if (!inside) {  // (uniform; the whole step twice, with and without, spills)
      const uint32_t pb = lo + TP * st + 32 * wd + 4 * qd - clo;
#pragma unroll
      for (int p = 0; p < PT; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[p][i] = pb + 16 * p + i < width ? x[p][i] : -INFINITY;
    }
    float mx = -INFINITY, sc[PT];  // (sc >= 0)
#pragma unroll
    for (int p = 0; p < PT; ++p) {
      sc[p] = s_scale * ksc[p];
      sc[p] = sc[p] < 1.2e-38f ? 1.2e-38f : sc[p];  // (0 times a masked -Inf would be NaN; a NaN stays)
      mx = fmaxf(mx, fmaxf(fmaxf(x[p][0], x[p][1]), fmaxf(x[p][2], x[p][3])) * sc[p]);
    }
    mx = g4d::xmax32(g4d::xmax16(mx));
    // P relative to a power of two (PAIR: of this wave's positions), so that a later one rescales it exactly
    const float m_own = fmaxf(m_run, ceilf(mx));
    float ps = 0.f;
    h8 ph[2], pl[2];  // of 32 positions each
    auto weights = [&](int k) __attribute__((always_inline)) {
      float e[2][4], es[2][4];
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[p][i] = exp2_h(fmaf(x[2 * k + p][i], sc[2 * k + p], -m_own));
          es[p][i] = e[p][i] * vsc[2 * k + p];
        }
      if (odd) {  // (uniform) a page whose scale is not finite: 0 where it is masked
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            e[p][i] = x[2 * k + p][i] == -INFINITY ? 0.f : e[p][i];
            es[p][i] = x[2 * k + p][i] == -INFINITY ? 0.f : es[p][i];
          }
      }
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        ps += (e[p][0] + e[p][1]) + (e[p][2] + e[p][3]);
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const h2 hi = __builtin_convertvector((f2{es[p][i], es[p][i + 1]}), h2);
          const h2 lo = __builtin_convertvector(
              (f2{fmaf((float)hi[0], -1.f, es[p][i]), fmaf((float)hi[1], -1.f, es[p][i + 1])}), h2);
          ph[k][4 * p + i] = hi[0];
          ph[k][4 * p + i + 1] = hi[1];
          pl[k][4 * p + i] = lo[0];
          pl[k][4 * p + i + 1] = lo[1];
        }
      }
    };
#pragma unroll
    for (int k = 0; k < PT / 2; ++k) weights(k);
    ps = g4d::xsum32(g4d::xsum16(ps));
    float m_new = m_own;
    if constexpr (PAIR) {
      h8* pp = s_p + (wc * 2 * 2) * 64 + l;
      pp[(wd * 2) * 64] = ph[0];
      pp[(wd * 2 + 1) * 64] = pl[0];
      if (qd == 0) s_mx[wd * TC + 16 * wc + c] = m_own;
      __syncthreads();
      const float m_other = s_mx[(wd ^ 1) * TC + 16 * wc + c];
      m_new = fmaxf(m_own, m_other);
      const float f_own = exp2_h(m_own - m_new), f_other = exp2_h(m_other - m_new);
      ps *= f_own;
      ph[0] = pp[0];
      pl[0] = pp[64];
      ph[1] = pp[128];
      pl[1] = pp[192];
      if (__ballot(f_own != f_other)) {  // (one of them is 1; f16 ends at 2^-24, so the powers of two in two halves)
        const float d0 = (wd ? m_other : m_own) - m_new, d1 = (wd ? m_own : m_other) - m_new;
        const float a0 = ceilf(d0 * 0.5f), a1 = ceilf(d1 * 0.5f);
        const _Float16 f0 = (_Float16)exp2_h(a0), g0 = (_Float16)exp2_h(d0 - a0);
        const _Float16 f1 = (_Float16)exp2_h(a1), g1 = (_Float16)exp2_h(d1 - a1);
        ph[0] = ph[0] * f0 * g0;
        pl[0] = pl[0] * f0 * g0;
        ph[1] = ph[1] * f1 * g1;
        pl[1] = pl[1] * f1 * g1;
      }
    }
    const float alpha = exp2_h(m_run - m_new);
    l_run = l_run * alpha + ps;
    m_run = m_new;
    if (__ballot(alpha != 1.f)) {  // O's rows are columns 4 qd + i
      float ar[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) ar[i] = __shfl(alpha, 4 * qd + i, 64);
#pragma unroll
      for (int e = 0; e < NE; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) O[e][i] *= ar[i];
    }
    load_v(next);
    // ---- P V ----
    // groups of four dims and 32 positions, the next group's operands read while one is multiplied
    const uint8_t* vb = s_v + wd * NE * 1024 + l * 16;
    h8 B[2][4];
    auto read_b = [&](int u, h8* to) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) to[e] = *(const h8*)(vb + ((u & 1) * (PAIR ? 2 : 1) * NE + u / 2 * 4 + e) * 1024);
    };
    read_b(0, B[0]);
#pragma unroll
    for (int u = 0; u < NE / 2; ++u) {
      if (u + 1 < NE / 2) read_b(u + 1, B[(u + 1) & 1]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f4& o = O[u / 2 * 4 + e];
        o = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl[u & 1], B[u & 1][e], o, 0, 0, 0);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f4& o = O[u / 2 * 4 + e];
        o = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[u & 1], B[u & 1][e], o, 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  for (uint32_t st = st0; st < st1; ++st) {
    __syncthreads();  // every wave is done with the previous step's rows
    store_step();
    {
      const uint32_t k = 4 * ((st - st0) % CH);
      const f4 kk = *(const f4*)(s_ks + k), vv = *(const f4*)(s_vs + k);
      odd = __ballot(!((vv[0] + vv[1] + vv[2] + vv[3]) + (kk[0] + kk[1] + kk[2] + kk[3]) < INFINITY));
#pragma unroll
      for (int p = 0; p < PT; ++p) {
        ksc[p] = kk[p];
        vsc[p] = vv[p];
        if (PAIR && wd) {
          ksc[p] = kk[(p + 2) & 3];
          vsc[p] = vv[(p + 2) & 3];
        }
      }
    }
    __syncthreads();
    // the next step's rows are in flight during this one, K's from before its scores, V's from before its P V (past
    // the last step: its own rows again, not used)
    const uint32_t next = (min(st + 1, st1 - 1) - st0) % CH;
    float by = 1.f;
    if (next == 0 && st + 1 < st1) by = refill(st + 1);  // (uniform)
    load_k(next);
    const uint32_t p0 = lo + TP * st;
    turn(st, next, p0 >= all0 && p0 + TP - 1 <= all1);
    if (by != 1.f) {  // (uniform) V's scales are relative to a larger one from here on
#pragma unroll
      for (int e = 0; e < NE; ++e) O[e] *= by;
    }
  }

  // ---- columns 4 qd + i of the wave's tile, dims NE c + e (PAIR: 256 wd + 16 c + e) ----
  if constexpr (PAIR) {
    __syncthreads();
    if (qd == 0) s_mx[wd * TC + 16 * wc + c] = l_run;
    __syncthreads();
    l_run = s_mx[16 * wc + c] + s_mx[TC + 16 * wc + c];
  }
  const bool whole = st1 - st0 == steps;
  const uint32_t slot = 2 * wg + used;  // (0 for a tile begun by another workgroup: it comes first)
  used = 1;
  float* part = a.part + (size_t)slot * TileShape<HD>::SLOT;
  // Row by row through LDS (where V was), so that a wave stores whole KB: lanes storing their own 16 bytes of every 64
  // take four times the requests. Four dims of a lane turned by c: its 16 lanes meet different banks.
  constexpr int RD = NE * 16, QG = NE / 4, RPS = 16 / NE;  // a wave's dims of a row; a lane's groups; rows a store
  if constexpr (!PAIR) __syncthreads();  // (every wave is done with V)
  float* turn_s = (float*)s_v + w * 4 * RD;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float L = __shfl(l_run, 4 * qd + i, 64), f = (whole ? 1.0f / L : 1.f) * (v_ref * (1.f / kTileP));
#pragma unroll
    for (int e = 0; e < QG; ++e)
      *(f4*)(turn_s + qd * RD + c * NE + 4 * ((e + c) % QG)) =
          f4{O[4 * e][i] * f, O[4 * e + 1][i] * f, O[4 * e + 2][i] * f, O[4 * e + 3][i] * f};
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");  // (the wave's own region: its LDS operations are in order)
#pragma unroll
    for (int r0 = 0; r0 < 4; r0 += RPS) {
      const int r = r0 + l / (RD / 4), d4 = l % (RD / 4), lc = d4 / QG;
      const f4 y = *(const f4*)(turn_s + r * RD + lc * NE + 4 * ((d4 % QG + lc) % QG));
      const uint32_t col = 16 * wc + 4 * r + i, og = ct * TC + col;
      if (og < ncols)
        *(f4*)((whole ? a.out + row_of(a, first, kvh, og) * HD : part + 2 * TC + col * HD) + 256 * wd + 4 * d4) = y;
    }
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
  }
  if (!whole && wd == 0 && qd == 0) {
    part[16 * wc + c] = m_run;
    part[TC + 16 * wc + c] = l_run;
  }
  if (st0 == 0 && tid == 0) a.meta[(size_t)pair * a.nkh + kvh] = make_uint2(slot, sh.owner(seg + cost - 1));
  }

  // rows that see nothing
  for (uint32_t j = wg; j < pairs; j += gridDim.x) {
    const Seq q = seq_rows(a.rows, j / a.tiles);
    const uint32_t g0 = j % a.tiles * TC, ncols = q.n * a.G;
    if (q.len || g0 >= ncols) continue;
    for (uint32_t i = tid; i < min((uint32_t)TC, ncols - g0) * a.nkh * HD; i += S_::NTH) {
      const uint32_t g = g0 + i / HD / a.nkh, kvh = i / HD % a.nkh;
      a.out[row_of(a, q.first, kvh, g) * HD + i % HD] = 0.f;
    }
  }
}

// out of a row and head from its tile's partials, in order: that of workgroup
// meta.x / 2 (slot meta.x), then slot 0 of each up to meta.y.
template <int HD>
__global__ __launch_bounds__(HD / 4) void attn8_tile_merge_kernel(Args a) {
  const uint32_t row = blockIdx.x / a.nqh, head = blockIdx.x % a.nqh, d = threadIdx.x * 4;
  const uint32_t s = seq_of_row(a.rows, row);
  if (s >= a.rows.num_seqs) return;
  const Seq q = seq_rows(a.rows, s);
  if (!q.len) return;
  const uint32_t g = (row - q.first) * a.G + head % a.G, col = g % TC;
  const uint2 mt = a.meta[((size_t)s * a.tiles + g / TC) * a.nkh + head / a.G];
  const uint32_t w0 = mt.x / 2, n = mt.y - w0 + 1;
  if (n == 1) return;  // written by its workgroup
  auto part = [&](uint32_t k) { return a.part + (size_t)(k ? 2 * (w0 + k) : mt.x) * TileShape<HD>::SLOT; };
  constexpr int MS = 4;  // partials on their way
  float M = kNothing, L = 0.f;
  f4 o = f4{0.f, 0.f, 0.f, 0.f};
  for (uint32_t k0 = 0; k0 < n; k0 += MS) {
    float pm[MS], pl[MS];
    f4 po[MS];
#pragma unroll
    for (int k = 0; k < MS; ++k) {
      const float* p = part(min(k0 + k, n - 1));
      pm[k] = p[col];
      pl[k] = p[TC + col];
      po[k] = *(const f4*)(p + 2 * TC + col * HD + d);
    }
    float mn = M;
#pragma unroll
    for (int k = 0; k < MS; ++k) mn = fmaxf(mn, pm[k]);
    const float al = exp2_h(M - mn);
    L *= al;
    o *= al;
#pragma unroll
    for (int k = 0; k < MS; ++k) {
      if (k0 + k >= n) continue;
      const float f = exp2_h(pm[k] - mn);
      L += f * pl[k];
      o += f * po[k];
    }
    M = mn;
  }
  *(f4*)(a.out + (size_t)blockIdx.x * HD + d) = o * (1.0f / L);
}

bool step_fits(const g4_kv8_params& p) {
  return (uint64_t)p.max_rows * (p.num_q_heads / p.num_kv_heads) <= COLS;
}
// Units a sequence may have (a window of several rows spans max_rows - 1 more positions, and up to 15 of its first
// tile).
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
uint32_t tile_wgs(const g4_kv8_params& p) {
  return (uint32_t)std::min<uint64_t>(TileShape<HD>::WGS, (all_cost(p) + kLeast - 1) / kLeast);
}
size_t tile_meta_bytes(const g4_kv8_params& p) {
  return ((size_t)p.num_seqs * tiles_of(p) * p.num_kv_heads * sizeof(uint2) + 255) / 256 * 256;
}
template <int HD>
size_t tile_bytes(const g4_kv8_params& p) {
  return tile_meta_bytes(p) + 2ull * tile_wgs<HD>(p) * TileShape<HD>::SLOT * sizeof(float);
}
template <int HD>
size_t attn_bytes(const g4_kv8_params& p) {
  return step_fits(p) ? step_bytes<HD>(p) : tile_bytes<HD>(p);
}

template <int HD>
int attend(g4_ctx* ctx, const g4_kv8_params& p, Args a, void* workspace) {
  if (step_fits(p)) {
    G4_REQUIRE(most_units(p) * p.num_seqs * p.num_kv_heads < (1ull << 31),
               "g4_pagedAttn8: %u sequences of up to %u positions and %u KV heads in one call", p.num_seqs,
               p.max_seq_len, p.num_kv_heads);
    G4_REQUIRE((uint64_t)p.num_seqs * p.num_kv_heads * p.max_rows * a.G < 1u << 24,
               "g4_pagedAttn8: %u sequences of up to %u rows of %u heads in one call", p.num_seqs, p.max_rows,
               p.num_q_heads);
    a.wgs = step_wgs<HD>(p);
    a.meta = (uint2*)workspace;
    a.part = (float*)((uint8_t*)workspace + meta_bytes(p));
    hipLaunchKernelGGL(attn8_step_kernel<HD>, dim3(a.wgs), dim3(NT), 0, ctx->stream, a);
    G4_LAUNCHED(ctx, "attn8_step");
    const uint64_t units = most_units(p);
    if (units == 1) return G4_OK;  // no sequence has partials
    const dim3 grid(p.num_seqs * p.num_kv_heads * p.max_rows * a.G);
    if (std::min<uint64_t>(units, a.wgs) <= 32 || grid.x >= 1u << 22)
      hipLaunchKernelGGL((attn8_merge_kernel<HD, 256>), grid, dim3(256), 0, ctx->stream, a);
    else
      hipLaunchKernelGGL((attn8_merge_kernel<HD, 1024>), grid, dim3(1024), 0, ctx->stream, a);
    G4_LAUNCHED(ctx, "attn8_merge");
    return G4_OK;
  }
  a.tiles = tiles_of(p);
  G4_REQUIRE(all_cost(p) < (1ull << 31) && (uint64_t)a.tiles * p.num_seqs * p.num_kv_heads < (1ull << 31),
             "g4_pagedAttn8: %u sequences of up to %u rows and %u positions in one call", p.num_seqs, p.max_rows,
             p.max_seq_len);
  G4_REQUIRE((uint64_t)p.num_rows * p.num_q_heads < 1u << 25, "g4_pagedAttn8: %u rows of %u heads in one call",
             p.num_rows, p.num_q_heads);
  a.wgs = tile_wgs<HD>(p);
  a.meta = (uint2*)workspace;
  a.part = (float*)((uint8_t*)workspace + tile_meta_bytes(p));
  hipLaunchKernelGGL(attn8_tile_kernel<HD>, dim3(a.wgs), dim3(TileShape<HD>::NTH), 0, ctx->stream, a);
  G4_LAUNCHED(ctx, "attn8_tile");
  if (a.wgs == 1) return G4_OK;  // no tile has partials
  hipLaunchKernelGGL(attn8_tile_merge_kernel<HD>, dim3(p.num_rows * p.num_q_heads), dim3(HD / 4), 0, ctx->stream, a);
  G4_LAUNCHED(ctx, "attn8_tile_merge");
  return G4_OK;
}

}  // namespace

extern "C" {

int g4_pagedAttn8_workspace_size(g4_kv8_params p, size_t* bytes) {
  G4_REQUIRE(bytes, "g4_pagedAttn8_workspace_size: null out");
  int rc = g4_internal_kv8_check(__func__, p, p.max_rows == 1 && p.num_rows == p.num_seqs ? nullptr : &p.num_rows);
  if (rc) return rc;
  *bytes = p.head_dim == 64 ? attn_bytes<64>(p) : p.head_dim == 128 ? attn_bytes<128>(p)
           : p.head_dim == 256 ? attn_bytes<256>(p) : attn_bytes<512>(p);
  return G4_OK;
}

int g4_pagedAttn8(g4_ctx* ctx, const float* q, const int8_t* k_pool, const int8_t* v_pool, const float* k_scale,
                  const float* v_scale, const int32_t* page_table, const uint32_t* seq_lens,
                  const uint32_t* row_starts, float* output, g4_kv8_params p, void* workspace,
                  size_t workspace_bytes) {
  return g4_pagedAttn8Ops(ctx, q, k_pool, v_pool, k_scale, v_scale, page_table, seq_lens, row_starts, output, p,
                          workspace, workspace_bytes, nullptr);
}

int g4_pagedAttn8Ops(g4_ctx* ctx, const float* q, const int8_t* k_pool, const int8_t* v_pool, const float* k_scale,
                     const float* v_scale, const int32_t* page_table, const uint32_t* seq_lens,
                     const uint32_t* row_starts, float* output, g4_kv8_params p, void* workspace,
                     size_t workspace_bytes, void* ops) {
  G4_ENTER(ctx);
  G4_REQUIRE(q && k_pool && v_pool && k_scale && v_scale && page_table && seq_lens && output && workspace,
             "g4_pagedAttn8: null buffer");
  int rc = g4_internal_kv8_check(__func__, p, row_starts);
  if (rc) return rc;
  size_t need = 0;
  rc = g4_pagedAttn8_workspace_size(p, &need);
  if (rc) return rc;
  G4_REQUIRE(workspace_bytes >= need, "g4_pagedAttn8: workspace %zu bytes < %zu required", workspace_bytes, need);
  const uintptr_t all = (uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)output | (uintptr_t)workspace;
  G4_REQUIRE((all & 15) == 0,
             "g4_pagedAttn8: rows, pools and workspace must be 16-byte aligned");
  G4_REQUIRE(!ops || (p.head_dim % 256 == 0 && p.num_rows <= 64 && step_fits(p) && ((uintptr_t)ops & 15) == 0),
             "g4_pagedAttn8Ops: operand blocks need head_dim a multiple of 256, <= 64 rows, <= 16 rows x heads of a "
             "KV head and a 16-byte aligned buffer");
  const Args a{paged_args(p, q, page_table, seq_lens, row_starts, output, ops), k_pool, v_pool, k_scale, v_scale};
  switch (p.head_dim) {
    case 64: return attend<64>(ctx, p, a, workspace);
    case 128: return attend<128>(ctx, p, a, workspace);
    case 256: return attend<256>(ctx, p, a, workspace);
    default: return attend<512>(ctx, p, a, workspace);
  }
}

}  // extern "C"
