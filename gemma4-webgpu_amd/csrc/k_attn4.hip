// k_attn4.hip — attention over the 4-bit paged K/V pool (k_kv4.hip writes it),
// and the attention weight of its rows, on the gfx950 matrix cores.
//
//   S[pos][col] = k[pos] . q[col],  out[col] = sum P[pos][col] * v[pos],  P = softmax of scale * S,
//   mass[pos] += sum over cols of P[pos][col]
//
// a column being one query row and head of a KV head.
//  * scores: v_mfma_scale_f32_16x16x128_f8f6f4 takes 16 K rows' codes and scales as
//    they lie in the pool (e2m1, e8m0 per 32 dims). q is five e2m3 digits of 5 bits
//    a block of 32 dims, each with a scale of its own, so that all sum up in one
//    f32 accumulator: digits in [-16, 16] / 8, q rounded to 2^-24 of its block's
//    largest. Products and sums of one instruction are exact but for one rounding
//    (2^-23.2 of the magnitudes' sum at most, over random blocks and scales). No
//    conversion of K, and 16 cycles for 128 dims and a digit.
//  * P V: v_mfma_f32_16x16x32_bf16, P * 2^15 as three bf16 of 8 bits each in one sum:
//    all 24 bits of every P, whatever its size (two f16 hold them down to 2^-17 of
//    the row's largest: a far key's share is then lost where the near ones' values
//    are 0). V is exact in bf16 (codes of 2 bits): one conversion for two codes with
//    their scale, and one byte permutation for the order of the operand.
// Sums over steps are f32. Maxima are taken to the next power of two, so that a
// later one rescales exactly.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attn_paged.hpp"
#include "kv4.hpp"

namespace {

using namespace g4kv8;
using g4kv4::BAD;
using g4kv4::BLOCK;
using g4mm::static_for;
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef int i6 __attribute__((ext_vector_type(6)));
typedef int i8 __attribute__((ext_vector_type(8)));
typedef float f16x __attribute__((ext_vector_type(16)));

constexpr int COLS = 16;               // columns of a matrix product
constexpr double kLog2e = 1.4426950408889634;  // the softmax works in powers of two
constexpr float kPScale = 32768.f;
constexpr float kNothing = -3e38f;     // the maximum of no positions: finite, so that differences are
constexpr int DIGITS = 5;

struct Args : PagedArgs {
  float scale_part;  // scale * log2(e) = scale_part * 2^scale_up, its magnitude in 0.5 .. 1 (or 0)
  int scale_up;
  const uint8_t *kp, *vp, *ks, *vs;
  float* mass;              // or null
  float2* sums;             // with mass: maximum and 1 / sum of each row and query head
  float* scores;            // few rows, with mass: [sequence][KV head][unit][column][128 positions]
  uint32_t units, columns;  // of a sequence and KV head there; many rows: 16 columns at a time, of a KV head
  uint8_t* qdigits;         // many rows, with mass: [KV head][16 columns][digit][128 dims][lane] 24 B, and the scales
  uint2* qscales;
  float* weights;           // [sequence][KV head][256 positions at a time][split][position]
  uint32_t splits, blocks;  // (few rows: the workgroups that weigh a sequence and KV head)
  uint32_t* done;           // many rows, with mass: whether the tiles were written
};

// ---- q as digits ----

// The exponent of a block of q with the largest magnitude am (its bits, so that a NaN is the largest), and the scale
// bytes of its five digits, with the exponent `up` of the scores' scale in them: so the sums are the scores within a
// factor of two, whatever q's size and the scale's. A block that is not finite counts as 0 under a scale of NaN; one
// below 2^-106 of a score as 0 (the last digit's scale ends there).
struct QScale {
  int down;     // times 2^down the largest is in 1 .. 2
  uint2 bytes;  // of the first four; of the last
};
__device__ __forceinline__ QScale q_scale(uint32_t am, int up) {
  QScale z;
  const bool bad = am >= 0x7f800000u;
  const int e = max((int)(am >> 23), 1) - 127, to = min(e + up, 127);  // am < 2^(e + 1)
  const bool none = to < -106;
  z.down = none ? -300 : -e;
  const uint32_t s = none ? 127u : (uint32_t)(to + 127);
  z.bytes.x = bad ? 0x7f7f7f00u | BAD : s | (s - 5) << 8 | (s - 10) << 16 | (s - 15) << 24;
  z.bytes.y = bad ? 127u : s - 20;
  return z;
}
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// The digits of N neighbouring elements x of a block (the rest of it taken as 0), as their codes: to(digit, code). Below 2
// units a code's steps are 1 / 8 of one, so that each conversion rounds to a digit and leaves at most half of a step, two
// units of the next. (An element that is not finite has any digits; the block's scale is NaN then.)
template <int N, typename F>
__device__ __forceinline__ void digits_of(const float* x, const QScale& z, F&& to) {
  f16x a, b;  // even, odd elements (the conversion takes them in turn)
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    a[i] = 2 * i < N ? __builtin_amdgcn_ldexpf(x[2 * i < N ? 2 * i : 0], z.down) : 0.f;
    b[i] = 2 * i < N ? __builtin_amdgcn_ldexpf(x[2 * i < N ? 2 * i + 1 : 0], z.down) : 0.f;
  }
  static_for<DIGITS>([&](auto d) __attribute__((always_inline)) {
    constexpr int D = decltype(d)::value;
    constexpr float unit = 1.f / (float)(1u << (5 * D));
    const auto code = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(a, b, unit);
    to(d, __builtin_bit_cast(i6, code));
    if constexpr (D < DIGITS - 1) {
      const auto u = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(code, unit);
#pragma unroll
      for (int i = 0; 2 * i < N; ++i) {
        a[i] -= u[2 * i];
        b[i] -= u[2 * i + 1];
      }
    }
  });
}

// One digit of q times 128 dims of 16 K rows, added to c. KS and QS: the bytes of ks and qs with their scales.
template <int KS, int QS>
__device__ __forceinline__ f4 product(const i4& k, const i6& q, f4 c, uint32_t ks, uint32_t qs) {
  const i8 a{k[0], k[1], k[2], k[3], 0, 0, 0, 0}, b{q[0], q[1], q[2], q[3], q[4], q[5], 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 2, KS, (int)ks, QS, (int)qs);
}

__device__ __forceinline__ void read_digit(const uint8_t* from, i6& to) {
#pragma unroll
  for (int e = 0; e < 3; ++e) {
    const uint2 y = ((const uint2*)from)[e];
    to[2 * e] = (int)y.x;
    to[2 * e + 1] = (int)y.y;
  }
}

// ---- P and V as bf16 ----

// Eight values in three parts: 8 bits of each from the top, by cutting (the differences are exact).
__device__ __forceinline__ void in_parts(const float* x, b8& hi, b8& mid, b8& lo) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = x[i];
  auto part = [&](b8& to, bool more) __attribute__((always_inline)) {
    i4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i)  // (the upper halves of two)
      y[i] = (int)__builtin_amdgcn_perm(__float_as_uint(r[2 * i + 1]), __float_as_uint(r[2 * i]), 0x07060302u);
    to = __builtin_bit_cast(b8, y);
    if (more)
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] -= __uint_as_float(__float_as_uint(r[i]) & 0xffff0000u);
  };
  part(hi, true);
  part(mid, true);
  part(lo, false);
}

// Byte I of four as the power of two that it is the exponent of (255: infinity, 0: 0).
template <int I>
__device__ __forceinline__ float exponent(uint32_t w) {
  return __uint_as_float(I < 3 ? (w << (24 - 8 * I) >> 24) << 23 : w >> 24 << 23);
}
__device__ __forceinline__ bool any_bad(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & w & 0x80808080u; }
// The two codes of byte B of x and of y, each times its row's scale: (first of x, first of y), (second, second).
template <int B>
__device__ __forceinline__ void two_by_two(uint32_t x, float sx, uint32_t y, float sy, uint32_t& first, uint32_t& second) {
  const uint32_t u = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, sx, B));
  const uint32_t v = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(y, sy, B));
  first = __builtin_amdgcn_perm(v, u, 0x05040100u);
  second = __builtin_amdgcn_perm(v, u, 0x07060302u);
}

// ---------------------------------------------------------------------------
// few rows a sequence (a decode step): rows * query heads per KV head <= 16
// ---------------------------------------------------------------------------
//
// HBM bounds it: every byte of K and V goes from the pool to LDS once, without
// registers in between, two steps of 32 positions ahead of each wave, and from
// there to registers in the matrix operands' order. Rows in flight in registers
// (72 of them at head dim 256) spilled, and a spilled value's reload waits for
// every row asked for before it.
//
// The positions of all sequences, in units of 128, are dealt to the workgroups
// in equal shares whatever the lengths (a share may end in one sequence and go
// on in the next), 32 positions at a time to each of the four waves. A sequence
// held by one workgroup is written by it; else its workgroups leave partials
// (max, sum, o), which attn4_merge_kernel adds in order. With masses, the scores
// go to the workspace, and the merge's launch turns them into weights: 4 bytes a
// position and column written and read, where K again would be HD / 2 * 17 / 16
// bytes a position and the products once more. It adds 3 to 6 us to a step (head
// dim 512: 64 sequences of up to 4352 positions 31.6 and 34.5, 32 of up to 32000 57
// and 63; in a launch of its own behind the merge 1.2 more).
//
// In the loop the pool comes at 5.4 TB/s (head dim 512, 64 sequences: 3.3 us a step of
// the four waves, before P had a third part, which costs 3 % there), around it stand
// 7.4 us until the first rows are there (lengths 0.8, page ids and the first rows'
// requests 3, q's digits 2, the wait 1.6) and 2.7 for the waves' sums. One sequence of 777 positions and a window of 512 at head dim 256
// takes 8.1 us, 64 of up to 8192 18.5 (50 MB), 32 of up to 32000 at 512 54 (193 MB);
// the merge 3.4 to 4.8.
constexpr int NT = 256, UNIT = 128;
constexpr uint32_t kSeqCost = 1;  // cost of a sequence and KV head besides its units: its q, its sums
template <int HD>
struct StepShape {
  static constexpr uint32_t WGS = HD == 512 ? 256 : HD == 256 ? 512 : 768;  // one to three per CU (LDS)
  static constexpr uint32_t SLOT = COLS * (HD + 2);       // floats of a partial: max, sum [16], o [16][HD]
  // A step's rows in LDS: K of two tiles, V of two tiles, scales of K, K, V, V (256 B each). 16-byte pieces of a row
  // are exchanged by its number, so that eight rows' same pieces are on different banks.
  static constexpr int PRW = HD / 32, KI = HD < 128 ? 1 : HD / 128;  // pieces of a row; KB of a tile (a load each)
  static constexpr int BYTES = 4 * KI * 1024 + 1024, LOADS = 4 * KI + 4;
  static __device__ __forceinline__ uint32_t turn(uint32_t row) {
    return PRW >= 8 ? row & 7u : row / (8 / PRW) & (PRW - 1u);
  }
};

// SIZE bytes a lane from base + off to LDS at `at` (uniform), lane by lane (16 apart for
// 16 bytes, else 4). Written as the instruction itself because the compiler, which knows
// the builtin's LDS write, waits for every such load before LDS is read; the waits are the
// caller's. (m0 takes the LDS address, with one wait state after its write; it is a
// reserved register, which the compiler sets at each use of its own.)
template <int SIZE>
__device__ __forceinline__ void to_lds(uint32_t off, const uint8_t* base, uint32_t at) {
  if constexpr (SIZE == 16)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(at) : "memory");
  else if constexpr (SIZE == 4)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(at) : "memory");
  else
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_ushort %0, %1" ::"v"(off), "s"(base), "s"(at) : "memory");
}
// A barrier that waits for LDS operations alone, not for the loads to LDS on their way.
__device__ __forceinline__ void ring_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// At most N vector memory operations in flight, and no LDS one.
template <int N>
__device__ __forceinline__ void wait_for_lds() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(N) : "memory");
}

template <int HD, bool MASS>
__global__ __launch_bounds__(NT, HD == 512 ? 1 : HD == 256 ? 2 : 3) void attn4_step_kernel(Args a) {
  using S_ = StepShape<HD>;
  constexpr int VB = HD / 16, NB = HD / BLOCK, J = HD < 128 ? 1 : HD / 128, BL = HD < 256 ? 1 : HD / 256;
  constexpr int VW = VB < 8 ? 1 : VB / 8;  // words of a lane's share of a V row
  constexpr int KI = S_::KI, PRW = S_::PRW;
  __shared__ __align__(1024) uint8_t s_ring[2 * 4 * S_::BYTES];  // [step in turn][wave]
  // (the same bytes) digits as B operands, [digit][128 dims][lane] 24 B, where the second steps go; at the end the
  // waves' sums
  uint8_t* s_q = s_ring + 4 * S_::BYTES;
  float* s_o = (float*)s_ring;
  static_assert(DIGITS * J * 64 * 24 <= 4 * S_::BYTES && 4 * COLS * HD * 4 <= sizeof(s_ring));
  __shared__ __align__(8) uint2 s_qs[J * 64];
  __shared__ float s_m[4 * COLS], s_l[4 * COLS];
  const int tid = threadIdx.x, l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), qd = l >> 4, c = l & 15;
  const uint32_t S = a.rows.num_seqs, wg = blockIdx.x;

  // The sequences 64 at a time, one a lane (in every wave alike): their units
  // summed up, T in all; then those that hold this workgroup's share.
  Seq mine{};
  uint32_t c0 = 0, mine_units = 0, incl = 0, total = 0;
  auto load_chunk = [&](uint32_t first) {
    c0 = first;
    mine = first + l < S ? seq_rows(a.rows, first + l) : Seq{0, 0, 0, 0};
    mine_units = mine.len ? (mine.len - first_seen(a, mine) + UNIT - 1) / UNIT + kSeqCost : 0u;
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

  uint32_t u = ub, used = 0;  // partials written
  while (u < ue) {
    while (before + total <= u) {  // (u < T: a later chunk holds it)
      before += total;
      load_chunk(c0 + 64);
    }
    const int at = __ffsll((unsigned long long)__ballot(before + incl > u)) - 1;
    const uint32_t s = c0 + at;
    const Seq sq{pick(mine.first, at), pick(mine.n, at), pick(mine.base, at), pick(mine.len, at)};
    const uint32_t cost = pick(mine_units, at), units = cost - kSeqCost, seq0 = before + pick(incl, at) - cost * a.nkh;
    const uint32_t lo = first_seen(a, sq), end = sq.len;
    const uint32_t kvh = a.nkh == 1 ? 0u : uni((u - seq0) / cost);
    const uint32_t seg = seq0 + kvh * cost, stop = min(seg + cost, ue);  // its first unit, the last here
    const uint32_t off = max(u, seg + kSeqCost) - (seg + kSeqCost), to = max(stop, seg + kSeqCost) - (seg + kSeqCost);
    u = stop;
    if (off == to) continue;  // (the share ends before its first positions)
    const uint32_t take = to - off;
    const uint32_t ncols = sq.n * a.G;
    const uint32_t rs = a.nkh * (HD / 2), ss = a.nkh * NB;  // bytes from a row to the next: codes, K scales

    // This wave's steps k are those of 32 positions st0 + 4 k; their tiles (of the pool) 32 steps at a time, a lane each:
    // a page id is asked for once, and reaches the addresses without memory in between.
    const uint32_t st0 = 4 * off + w, tiles = (end - lo + 15) / 16, t0 = lo / 16;
    const uint32_t last = min(4 * (off + take), (tiles + 1) / 2);  // (the last unit may be short)
    const uint32_t n = st0 < last ? (last - st0 + 3) / 4 : 0u;
    const int32_t* list = a.page_table + (size_t)s * a.max_pages;
    uint32_t ahead;
    auto refill = [&](uint32_t k) {
      const uint32_t t = t0 + min(2 * (st0 + 4 * (k + l / 2)) + (l & 1), tiles - 1), at = page_of(a, t);
      ahead = clamp_page(a, list[at]) * a.page_tiles + (t - at * a.page_tiles);
    };
    // where a lane's pieces are in a tile: those of row i * 64 / PRW + l / PRW in load i (head dim 64: half a load; 512:
    // every other load's rows are four on)
    const uint32_t pl = HD == 64 ? l & 31 : l, prow = pl / PRW, pp = pl % PRW;
    const uint32_t piece0 = prow * rs + 16 * (pp ^ S_::turn(prow)), piece1 = prow * rs + 16 * (pp ^ S_::turn(prow + 4));
    const uint32_t zl = HD == 64 ? l & 15 : l % (4 * NB);
    const uint32_t kz = HD == 64 ? zl * ss : zl / (NB / 4 > 0 ? NB / 4 : 1) * ss + 4 * (zl % (NB / 4 > 0 ? NB / 4 : 1));
    const uint32_t vz = 4 * (l % (4 * NB));
    const uint32_t ring = uni((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)s_ring) + w * S_::BYTES;
    auto load = [&](uint32_t k) __attribute__((always_inline)) {
      const uint32_t to = ring + (k & 1) * (4 * S_::BYTES);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const size_t t = pick(ahead, (2 * k + p) & 63);
        const uint8_t *kb = a.kp + t * (16 * (size_t)rs) + kvh * (HD / 2), *vb = a.vp + t * (16 * (size_t)rs) + kvh * (HD / 2);
#pragma unroll
        for (int i = 0; i < KI; ++i) {
          const uint32_t piece = HD == 512 && (i & 1) ? piece1 : piece0;
          to_lds<16>(piece, kb + i * (64 / PRW) * (size_t)rs, to + (p * KI + i) * 1024);
          to_lds<16>(piece, vb + i * (64 / PRW) * (size_t)rs, to + ((2 + p) * KI + i) * 1024);
        }
        to_lds<HD == 64 ? 2 : 4>(kz, a.ks + t * (16 * (size_t)ss) + kvh * NB, to + 4 * KI * 1024 + p * 256);
        to_lds<4>(vz, a.vs + (t * a.nkh + kvh) * (NB * 16), to + 4 * KI * 1024 + 512 + p * 256);
      }
    };

    // q, QE dims of a column a thread (asked for before the page ids, so that it has come when the rows are asked for)
    constexpr int QE = 16, QC = 128 * J / QE;                // threads of a column
    constexpr int QCOLS = COLS * QC <= NT ? COLS : NT / QC;  // columns at once (head dim 512: 8 of the 16)
    static_assert(QCOLS == COLS || 2 * QCOLS == COLS);
    int qt = tid;
    asm volatile("" : "+v"(qt));  // (what follows from it is not kept over the sequences: registers would spill)
    const uint32_t qdim = qt % QC * QE, block = qdim / BLOCK;
    float qx[QE];
    auto load_q = [&](uint32_t col) __attribute__((always_inline)) {
      const float* qg = a.q + row_of(a, sq.first, kvh, min(col, ncols - 1)) * HD + (HD == 64 ? qdim % 64 : qdim);
#pragma unroll
      for (int e = 0; e < QE; e += 4) {
        const f4 y = *(const f4*)(qg + e);
#pragma unroll
        for (int i = 0; i < 4; ++i) qx[e + i] = HD == 64 && block >= 2 ? 0.f : y[i];
      }
    };
    if (qt < QCOLS * QC) load_q(qt / QC);
    refill(0);
    ring_barrier();  // the previous sequence's sums are done with
    if (n > 0) load(0);  // (uniform)
    // ---- q's digits ----
    auto store_digits = [&](uint32_t col) __attribute__((always_inline)) {
      uint32_t am = 0;
#pragma unroll
      for (int e = 0; e < QE; ++e) am = max(am, magnitude(qx[e]));
      am = max(am, (uint32_t)g4d::dppi<g4d::kDppXor1>((int)am));
      const QScale z = q_scale(am, a.scale_up);
      const uint32_t j = block % J, lane = block / J * 16 + col;
      s_qs[j * 64 + lane] = z.bytes;
      digits_of<QE>(qx, z, [&](auto d, const i6& code) __attribute__((always_inline)) {
        uint32_t* to = (uint32_t*)(s_q + ((decltype(d)::value * J + j) * 64 + lane) * 24 + qdim % BLOCK / 4 * 3);
#pragma unroll
        for (int i = 0; i < QE * 3 / 16; ++i) to[i] = (uint32_t)code[i];
      });
    };
    if (qt < QCOLS * QC) store_digits(qt / QC);
    if (QCOLS < COLS && ncols > QCOLS) {  // (uniform; columns past the last one keep any digits: their weights are 0)
      load_q(qt / QC + QCOLS);
      store_digits(qt / QC + QCOLS);
    }
    ring_barrier();
    i6 qb[DIGITS][J];
    uint2 qs[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      qs[j] = s_qs[j * 64 + l];
#pragma unroll
      for (int d = 0; d < DIGITS; ++d) read_digit(s_q + ((d * J + j) * 64 + l) * 24, qb[d][j]);
    }
    ring_barrier();  // every wave has them
    if (n > 1) load(1);
    // this lane's column: positions clo .. clo + width - 1
    const float s_scale = a.scale_part;
    const uint32_t cpos = sq.base + div_g(a, c);
    const uint32_t clo = a.window && cpos + 1 > a.window ? cpos + 1 - a.window : 0u;
    const uint32_t width = (uint32_t)c < ncols ? cpos + 1 - clo : 0u;
    const uint32_t first = a.window && sq.base + 1 > a.window ? sq.base + 1 - a.window : 0u;  // of any column
    float* score_at = nullptr;
    if (MASS)
      score_at = a.scores + (((size_t)(s * a.nkh + kvh) * a.units) * a.columns + min((uint32_t)c, a.columns - 1)) * UNIT;
    f4 O[VB];
#pragma unroll
    for (int e = 0; e < VB; ++e) O[e] = f4{0.f, 0.f, 0.f, 0.f};
    float m_run = kNothing, l_run = 0.f;  // of column c, the sum times 2^15
    // a lane's pieces of K (row c) and V (rows 4 qd + i) of a tile
    uint32_t k_at[J], v_at[4];
#pragma unroll
    for (int j = 0; j < J; ++j) k_at[j] = c * (HD / 2) + 16 * ((HD == 64 ? qd & 1 : qd * J + j) ^ S_::turn(c));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t row = 4 * qd + i, byte = VB / 2 * c;
      v_at[i] = row * (HD / 2) + 16 * (byte / 16 ^ S_::turn(row)) + byte % 16;
    }
    const uint32_t kz_at = HD == 64 ? 4 * c + (qd & 1) : c * NB + J * qd, vz_at = VB * c / BLOCK * 16 + 4 * qd;
    for (uint32_t k = 0; k < n; ++k) {
      const uint32_t st = st0 + 4 * k;
      const uint8_t* in = s_ring + (k & 1) * (4 * S_::BYTES) + w * S_::BYTES;
      const uint8_t* z = in + 4 * KI * 1024;
      // this step's rows are there once at most the next one's are on their way (a store among them: all)
      if (k + 1 < n) wait_for_lds<S_::LOADS>();
      else wait_for_lds<0>();
      // ---- scores ----
      f4 D[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        uint32_t kw = J == 4 ? *(const uint32_t*)(z + 256 * p + kz_at) : J == 2 ? *(const uint16_t*)(z + 256 * p + kz_at)
                                                                              : z[256 * p + kz_at];
        if (HD == 64 && qd >= 2) kw = 127;  // (no dims there)
        i4 K[J];
#pragma unroll
        for (int j = 0; j < J; ++j) K[j] = *(const i4*)(in + p * (KI * 1024) + k_at[j]);
        D[p] = f4{0.f, 0.f, 0.f, 0.f};
        static_for<DIGITS * J>([&](auto i) __attribute__((always_inline)) {
          constexpr int d = DIGITS - 1 - decltype(i)::value / J, j = decltype(i)::value % J;  // (the smallest first)
          D[p] = product<j, d % 4>(K[j], qb[d][j], D[p], kw, d == 4 ? qs[j].y : qs[j].x);
        });
      }
      // ---- softmax over the step's 32 positions ----
      const uint32_t p0 = lo + 32 * st, pb = p0 + 4 * qd;
      const uint32_t vw[2] = {*(const uint32_t*)(z + 512 + vz_at), *(const uint32_t*)(z + 768 + vz_at)};
      float x[8], vsc[8], mx = -INFINITY;
      auto live = [&](int i) { return pb + 16 * (i / 4) + i % 4 - clo < width; };
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = D[i / 4][i % 4] * s_scale;
      static_for<8>([&](auto i) __attribute__((always_inline)) {
        constexpr int n = decltype(i)::value;
        vsc[n] = exponent<n % 4>(vw[n / 4]);
      });
      // (uniform) rows that no column sees may hold anything; of the others, one that is not finite makes the weight of
      // every column that sees it NaN
      if (p0 < first || p0 + 32 > end || __ballot(any_bad(vw[0]) || any_bad(vw[1]))) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t pos = pb + 16 * (i / 4) + i % 4;
          const bool bad = vsc[i] == INFINITY;
          if (bad) x[i] = __builtin_nanf("");
          if (bad || pos < first || pos >= end) vsc[i] = 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = live(i) ? x[i] : -INFINITY;
        mx = fmaxf(mx, x[i]);
      }
      if (MASS && (uint32_t)c < ncols) {
        float* to = score_at + (size_t)(st / 4) * a.columns * UNIT + st % 4 * 32 + 4 * qd;
        *(f4*)to = f4{x[0], x[1], x[2], x[3]};
        *(f4*)(to + 16) = f4{x[4], x[5], x[6], x[7]};
      }
      mx = g4d::xmax32(g4d::xmax16(mx));
      const float m_new = fmaxf(m_run, ceilf(mx)), up = 15.f - m_new;
      const float alpha = exp2_h(m_run - m_new);
      float ps = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = exp2_h(x[i] + up);
        ps += x[i];
      }
      b8 P[3];
      in_parts(x, P[2], P[1], P[0]);
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
      // ---- P V, two dims (a byte of V) at a time ----
      uint32_t V[8][VW];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint8_t* y = in + (2 + i / 4) * (KI * 1024) + v_at[i % 4];
        if constexpr (VW == 4) {
          const i4 x4 = *(const i4*)y;
#pragma unroll
          for (int e = 0; e < 4; ++e) V[i][e] = (uint32_t)x4[e];
        } else if constexpr (VW == 2) {
          const uint2 x2 = *(const uint2*)y;
          V[i][0] = x2.x;
          V[i][1] = x2.y;
        } else {
          V[i][0] = VB == 8 ? *(const uint32_t*)y : *(const uint16_t*)y;
        }
      }
      static_for<VB / 2>([&](auto e) __attribute__((always_inline)) {
        constexpr int b = decltype(e)::value % 4, v = decltype(e)::value / 4, n = 2 * decltype(e)::value;
        i4 B[2];
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          uint32_t y, z;
          two_by_two<b>(V[j][v], vsc[j], V[j + 1][v], vsc[j + 1], y, z);
          B[0][j / 2] = (int)y;
          B[1][j / 2] = (int)z;
        }
#pragma unroll
        for (int k = 0; k < 3; ++k)  // (the smallest first)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            O[n + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(P[k], __builtin_bit_cast(b8, B[i]), O[n + i], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      });
      if (k + 2 < n) {  // (uniform) into the bytes that this step has read
        if (((k + 2) & 31) == 0) refill(k + 2);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        load(k + 2);
      }
    }

    // ---- the four waves' sums, in their order ----
    __syncthreads();  // every wave is done with the rows
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
    const uint32_t slot = 2 * wg + used;  // (0 for a sequence begun by another workgroup: it comes first)
    used = 1;
    float* part = a.part + (size_t)slot * StepShape<HD>::SLOT;
    for (uint32_t i = tid; i < ncols * (HD / 4); i += NT) {
      const uint32_t col = i / (HD / 4), d = i % (HD / 4) * 4;
      float M = kNothing, L = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) M = fmaxf(M, s_m[k * COLS + col]);
      f4 y = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float f = exp2_h(s_m[k * COLS + col] - M);
        L += s_l[k * COLS + col] * f;
        y += *(const f4*)(s_o + (k * COLS + col) * HD + d / VB * VB + 4 * ((d % VB / 4 + d / VB) % QG)) * f;
      }
      const size_t row = row_of(a, sq.first, kvh, col);
      float* o = whole ? a.out + row * HD : part + 2 * COLS + col * HD;
      if (whole) y *= 1.0f / L;
      *(f4*)(o + d) = y;
      if constexpr (HD >= 256) {
        if (whole && a.ops)  // (uniform; a wave holds 256 values of one row and head)
          write_ops(a, sq.first + div_g(a, col), (kvh * a.G + col - div_g(a, col) * a.G) * BL + d / 256, l, y);
      }
      if (d == 0) {
        if (!whole) {
          part[col] = M;
          part[COLS + col] = L;
        } else if (MASS) {
          a.sums[row] = make_float2(M, kPScale / L);
        }
      }
    }
    if (off == 0 && tid == 0) a.meta[(size_t)s * a.nkh + kvh] = make_uint2(slot, sh.owner(seg + cost - 1));
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
//
// With masses, the workgroups behind those of the columns weigh the positions of a
// sequence and KV head, a thread each, from their scores: they find the columns'
// maxima and sums from the partials themselves rather than wait for the merge.
template <int HD, int MT>
__device__ __forceinline__ void weigh_positions(const Args& a, uint32_t b) {
  __shared__ float2 s_sum[COLS];
  const uint32_t sh = b / a.blocks, s = sh / a.nkh, kvh = sh % a.nkh, tid = threadIdx.x;
  const Seq q = seq_rows(a.rows, s);
  const uint32_t lo = first_seen(a, q), ncols = q.n * a.G;
  uint32_t t = lo + b % a.blocks * MT + tid;
  if (t - tid >= q.len) return;  // (uniform; a length of 0 too)
  static_assert(MT >= COLS * 16);
  const uint2 mt = a.meta[sh];
  const uint32_t col = tid / 16, w0 = mt.x / 2, n = mt.y - w0 + 1;
  if (col < ncols) {
    if (n == 1) {  // (uniform) written by its workgroup
      s_sum[col] = a.sums[row_of(a, q.first, kvh, col)];
    } else {
      auto part = [&](uint32_t k) { return a.part + (size_t)(k ? 2 * (w0 + k) : mt.x) * StepShape<HD>::SLOT + col; };
      float m = kNothing, sum = 0.f;
      for (uint32_t k = tid % 16; k < n; k += 16) m = fmaxf(m, *part(k));
      m = g4d::max16(m);
      for (uint32_t k = tid % 16; k < n; k += 16) sum += exp2_h(*part(k) - m) * part(k)[COLS];
      sum = g4d::sum16(sum);
      if (tid % 16 == 0) s_sum[col] = make_float2(m, kPScale / sum);
    }
  }
  __syncthreads();
  for (; t < q.len; t += a.blocks * MT) {
    const uint32_t at = t - lo, tile = t / 16, page = page_of(a, tile);
    const int32_t id = a.page_table[(size_t)s * a.max_pages + page];
    const float* x = a.scores + ((size_t)sh * a.units + at / UNIT) * a.columns * UNIT + at % UNIT;
    float got = 0.f;
    for (uint32_t c = 0; c < ncols; ++c) {
      const float y = x[c * UNIT];  // (-Inf: the column does not see the position, and its sum may be NaN)
      const float2 sum = s_sum[c];
      const float e = exp2_h(y - sum.x) * sum.y;
      got += y == -INFINITY ? 0.f : e;
    }
    if (id >= 0 && id < (int32_t)a.num_pages)
      a.mass[((size_t)id * (a.page_tiles * 16) + (t - page * a.page_tiles * 16)) * a.nkh + kvh] += got;
  }
}
template <int HD, int MT, bool MASS>
__global__ __launch_bounds__(MT) void attn4_merge_kernel(Args a) {
  constexpr int TG = HD / 4, NG = MT / TG, MS = 4;  // threads a partial row, groups, loads in flight of each
  __shared__ float s_m[NG], s_l[NG];
  __shared__ __align__(16) float s_o[NG * HD];
  const uint32_t cols = a.rows.max_rows * a.G, col = blockIdx.x % cols;
  if (const uint32_t merges = a.rows.num_seqs * a.nkh * cols; MASS && blockIdx.x >= merges) {
    weigh_positions<HD, MT>(a, blockIdx.x - merges);
    return;
  }
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
  float m = kNothing, l = 0.f;
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
    for (int k = 0; k < MS; ++k) mn = fmaxf(mn, i0 + NG * k < n ? pm[k] : kNothing);
    const float al = exp2_h(m - mn);
    l *= al;
    o *= al;
#pragma unroll
    for (int k = 0; k < MS; ++k) {
      if (i0 + NG * k >= n) continue;
      const float f = exp2_h(pm[k] - mn);
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
  float M = kNothing, L = 0.f;
  for (int i = 0; i < NG; ++i) M = fmaxf(M, s_m[i]);
  f4 y = f4{0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < NG; ++i) {
    const float f = exp2_h(s_m[i] - M);
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
// steps of 64 positions through LDS: K and its scales as stored, V as bf16 in the
// order of the P V product's operand. A wave holds 16 columns: their q digits and
// output sums in registers; two waves per SIMD, so that one's softmax runs beside
// the other's products. The next step's rows are on their way in registers.
//
// Head dim 512 (eight waves): the two waves of a column tile have 256 dims each,
// and 32 of the step's positions each for the softmax: they hand each other
// their sums of the other's positions, then their maxima and P, through LDS (q's
// digits of all 512 dims in one wave would spill).
//
// Page ids come through LDS, 32 steps at a time: scalar loads share their counter
// with LDS reads, so that the products of a step would wait for those of the next
// one.
//
// The work is dealt to the workgroups in equal shares (Walk), one or two
// workgroups a CU. A tile held by one workgroup is written by it, else its
// workgroups leave partials that attn4_tile_merge_kernel adds in order.
//
// A prompt of 4500 rows of 8 heads: 114 us at head dim 128, 180 at 256 and 364 at 512
// (364, 460 and 456 TFLOP/s), of 1500 rows 34, 46 and 73 to 78, the merge included. The
// matrix cores work 18 % of the time and the VALUs 30 (at a step of 64 positions and
// head dim 256 a wave has 136 products and 470 VALU instructions: V's codes to bf16,
// the softmax, the masks), the rest waits: for LDS, and at the steps' barriers, since
// registers allow two waves a SIMD. At head dim 512 a step of two barriers, with the
// next step's rows in flight for all of it, spilled and took 82 us where this one's
// four took 76.
template <int HD>
struct TileShape {
  static constexpr bool PAIR = HD == 512;
  static constexpr int NTH = PAIR ? 512 : 256;
  static constexpr int RB = HD / 2;              // bytes of a K row
  static constexpr int KS = RB + 16;             // its stride in LDS: 16 rows on different banks
  static constexpr int VBYTES = TP * HD * 2;
  static constexpr int PR = RB / 16;             // 16-byte pieces of a K row
  static constexpr int RPI = NTH / PR < TP ? NTH / PR : TP;  // rows of a round of pieces
  static constexpr int KP = TP / RPI;            // rounds
  static constexpr int VD = PAIR ? 16 : HD / 16; // dims a thread moves of 4 positions of V
  static constexpr int J = HD == 64 ? 1 : PAIR ? 2 : HD / 128;  // products of a wave's dims
  static constexpr uint32_t WGS = HD == 512 ? 256 : HD >= 128 ? 512 : 768;  // that run at once (registers, LDS)
  static constexpr uint32_t SLOT = TC * (HD + 2);                           // floats of a partial: max, sum [64], o
};
// Where a sequence's columns, 16 at a time, stand among those of all.
__device__ __forceinline__ uint32_t first_columns(const Args& a, uint32_t s, const Seq& q) { return q.first * a.G / 16 + s; }

template <int HD, bool MASS>
__global__ __launch_bounds__(TileShape<HD>::NTH, HD == 64 ? 3 : 2) void attn4_tile_kernel(Args a) {
  using S_ = TileShape<HD>;
  constexpr bool PAIR = S_::PAIR;
  constexpr int J = S_::J, KP = S_::KP, VD = S_::VD, RB = S_::RB, NB = HD / BLOCK;
  constexpr int NE = PAIR ? 16 : HD / 16;  // products over a wave's dims
  constexpr int PT = PAIR ? 2 : 4;         // tiles of a wave's softmax
  constexpr int CH = 32;                   // steps whose tiles are in LDS
  constexpr int VW = VD < 8 ? 1 : VD / 8;  // words of a thread's share of a V row
  constexpr int SB = NB < 4 ? NB : 4, SR = NB / SB;  // bytes of K scales a thread loads, threads of a row
  __shared__ __align__(16) uint8_t s_k[TP * S_::KS];
  __shared__ __align__(16) uint8_t s_z[TP * NB];  // K's scales
  __shared__ __align__(16) uint8_t s_v[S_::VBYTES];
  __shared__ __align__(16) f4 s_p[PAIR ? 4 * 2 * 2 * 64 : 1];  // P: [column tile][half][tile][lane]
  __shared__ __align__(16) f4 s_d[PAIR ? 4 * 2 * 2 * 64 : 1];  // sums: [column tile][half][tile][lane]
  __shared__ float s_mx[PAIR ? 2 * TC : 1];
  __shared__ uint32_t s_tile[4 * CH], s_bad[TP / 4];  // s_bad: rows of V that are not finite, four a word
  __shared__ WalkLds<S_::NTH> s_walk;
  Walk<S_::NTH> walk{a, s_walk};
  const bool ok = walk.begin();
  if (MASS && blockIdx.x == 0 && threadIdx.x == 0) *a.done = ok;
  if (!ok) return;

  Part pt;
  while (walk.next(pt)) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // (what follows from it is formed anew for each part: kept over all of them it spills)
    const int l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), qd = l >> 4, c = l & 15;
    const int wc = w & 3, wd = PAIR ? w >> 2 : 0;  // column tile; half
    __syncthreads();  // the previous tile's rows are done with
    const uint32_t ncols = pt.q.n * a.G, base = pt.q.base, first = pt.q.first, kvh = pt.kvh, ct = pt.ct;
    const uint32_t lo = pt.t.lo, end = pt.t.end, st0 = pt.st0, st1 = pt.st1;
    const uint32_t rs = a.nkh * RB, ss = a.nkh * NB;
    const uint32_t t0 = lo / 16, tlast = (end - 1) / 16;
    const int32_t* list = a.page_table + (size_t)pt.s * a.max_pages;

    // this lane's column
    const uint32_t g = ct * TC + 16 * wc + c, gr = min(g, ncols - 1);
    const uint32_t cpos = base + div_g(a, gr);
    const uint32_t clo = a.window && cpos + 1 > a.window ? cpos + 1 - a.window : 0u;
    const uint32_t width = g < ncols ? cpos + 1 - clo : 0u;
    // positions every column sees: those from the last row's window on, up to the first row's own; and that any sees
    const uint32_t r0 = base + div_g(a, ct * TC), all0 = a.window && end > a.window ? end - a.window : 0u, all1 = r0;
    const uint32_t any0 = a.window && r0 + 1 > a.window ? r0 + 1 - a.window : 0u;

    // ---- rows on their way ----
    i4 kr[KP];
    uint32_t zr = 0, vr_[4][VW], vw = 0;
    // This thread's V: positions 4 vq .. + 3 of tile vt, dims from vdim on.
    const int vt = 2 * (PAIR ? (w >> 1) & 1 : w >> 1) + (l >> 5), vq = 2 * (w & 1) + ((l >> 4) & 1);
    const uint32_t vdim = PAIR ? 256 * wd + 16 * c : VD * c;
    const bool has_k = S_::PR * S_::RPI >= S_::NTH || tid < S_::PR * S_::RPI;
    const uint32_t kpiece = tid % S_::PR * 16, krow = tid / S_::PR;
    const uint32_t v_at = 4 * vq * rs + vdim / 2, vs_at = vdim / BLOCK * 16 + 4 * vq;
    const uint32_t zrow = tid / SR, zbyte = tid % SR * SB;
    const uint8_t *kp = a.kp + kvh * RB, *vp = a.vp + kvh * RB, *kz = a.ks + kvh * NB;
    auto refill = [&](uint32_t st) __attribute__((always_inline)) {  // tiles (of the pool) of the steps from `st` on
      if (tid < 4 * CH) {
        const uint32_t t = min(t0 + 4 * st + tid, tlast), at = page_of(a, t);
        s_tile[tid] = clamp_page(a, list[at]) * a.page_tiles + (t - at * a.page_tiles);
      }
      __syncthreads();
    };
    auto load_k = [&](uint32_t k) __attribute__((always_inline)) {  // (of the refilled steps)
      if (has_k) {
#pragma unroll
        for (int i = 0; i < KP; ++i) {
          const uint32_t row = i * S_::RPI + krow;
          kr[i] = *(const i4*)(kp + (size_t)s_tile[4 * k + row / 16] * (16 * rs) + (row % 16 * rs + kpiece));
        }
      }
      if (SR * TP >= S_::NTH || tid < SR * TP) {
        const uint8_t* z = kz + (size_t)s_tile[4 * k + zrow / 16] * (16 * ss) + (zrow % 16 * ss + zbyte);
        zr = SB == 4 ? *(const uint32_t*)z : *(const uint16_t*)z;
      }
    };
    auto load_v = [&](uint32_t k) __attribute__((always_inline)) {
      const size_t t = s_tile[4 * k + vt];
      const uint8_t* x = vp + t * (16 * rs) + v_at;
      vw = *(const uint32_t*)(a.vs + (t * a.nkh + kvh) * (NB * 16) + vs_at);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (VW == 2) {
          const uint2 y = *(const uint2*)(x + i * rs);
          vr_[i][0] = y.x;
          vr_[i][1] = y.y;
        } else if constexpr (VD == 8) {
          vr_[i][0] = *(const uint32_t*)(x + i * rs);
        } else {
          vr_[i][0] = *(const uint16_t*)(x + i * rs);
        }
      }
    };
    // K rows as they are; V [32 positions][product e][lane (q, c)] 16 B: slots 4 (tile & 1) + i of position 4 q + i
    auto store_step = [&](uint32_t st) __attribute__((always_inline)) {
      if (has_k) {
#pragma unroll
        for (int i = 0; i < KP; ++i) *(i4*)(s_k + (i * S_::RPI + krow) * S_::KS + kpiece) = kr[i];
      }
      if (SR * TP >= S_::NTH || tid < SR * TP) {
        if constexpr (SB == 4) *(uint32_t*)(s_z + zrow * NB + zbyte) = zr;
        else *(uint16_t*)(s_z + zrow * NB + zbyte) = (uint16_t)zr;
      }
      float sc[4] = {exponent<0>(vw), exponent<1>(vw), exponent<2>(vw), exponent<3>(vw)};
      const uint32_t p0 = lo + TP * st;
      uint32_t bad = 0;
      if (p0 < any0 || p0 + TP > end || __ballot(any_bad(vw))) {  // (uniform) rows that no column sees hold anything
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t pos = p0 + 16 * vt + 4 * vq + i;
          const bool seen = pos >= any0 && pos < end;
          if (seen && sc[i] == INFINITY) bad |= 1u << i;
          if (!seen || sc[i] == INFINITY) sc[i] = 0.f;
        }
      }
      if (wd == 0 && c == 0) s_bad[4 * vt + vq] = bad;
      uint8_t* dst = s_v + (((vt >> 1) * (PAIR ? 2 : 1) + wd) * NE * 64 + vq * 16 + c) * 16 + (vt & 1) * 8;
      static_for<VD / 2>([&](auto e) __attribute__((always_inline)) {
        constexpr int k = decltype(e)::value;
        uint32_t x, y, x2, y2;
        two_by_two<k % 4>(vr_[0][k / 4], sc[0], vr_[1][k / 4], sc[1], x, y);
        two_by_two<k % 4>(vr_[2][k / 4], sc[2], vr_[3][k / 4], sc[3], x2, y2);
        *(g4mm::u32x2*)(dst + 2 * k * 1024) = g4mm::u32x2{x, x2};
        *(g4mm::u32x2*)(dst + (2 * k + 1) * 1024) = g4mm::u32x2{y, y2};
      });
    };
    refill(st0);
    load_k(0);
    load_v(0);

    // ---- q's digits: the scale's sign goes to q; a scale of 0 leaves equal scores ----
    i6 qb[DIGITS][J];
    uint2 qs[J];
    const float sign = a.scale_part < 0.f ? -1.f : a.scale_part == 0.f ? 0.f : 1.f;
    const float sc = a.scale_part == 0.f ? 1.f : fabsf(a.scale_part);  // (0 times a masked -Inf: NaN)
    static_for<J>([&](auto jj) __attribute__((always_inline)) {
      constexpr int j = decltype(jj)::value;
      const bool pad = HD == 64 && qd >= 2;
      const float* qg = a.q + row_of(a, first, kvh, gr) * HD + BLOCK * (pad ? 0 : qd * J + j) + 256 * wd;
      float x[BLOCK];
#pragma unroll
      for (int e = 0; e < BLOCK; e += 4) {
        const f4 y = *(const f4*)(qg + e);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[e + i] = pad ? 0.f : y[i] * sign;
      }
      uint32_t am = 0;
#pragma unroll
      for (int e = 0; e < BLOCK; ++e) am = max(am, magnitude(x[e]));
      const QScale q = q_scale(am, a.scale_up);
      qs[j] = q.bytes;
      digits_of<BLOCK>(x, q, [&](auto d, const i6& code) __attribute__((always_inline)) {
        qb[decltype(d)::value][j] = code;
      });
      __builtin_amdgcn_sched_barrier(0);  // (the next one's elements not before these are digits)
    });
    if (MASS && st0 == 0 && ct * TC + 16 * wc < ncols) {  // (for the weights, by the one that begins the tile)
      constexpr int JT = PAIR ? 4 : J;
      const size_t tile = (size_t)kvh * a.columns + first_columns(a, pt.s, pt.q) + 4 * ct + wc;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int jt = PAIR ? 2 * wd + j : j;
        a.qscales[(tile * JT + jt) * 64 + l] = qs[j];
#pragma unroll
        for (int d = 0; d < DIGITS; ++d) {
          uint2* to = (uint2*)(a.qdigits + ((tile * DIGITS + d) * JT + jt) * (64 * 24) + l * 24);
#pragma unroll
          for (int i = 0; i < 3; ++i) to[i] = make_uint2(qb[d][j][2 * i], qb[d][j][2 * i + 1]);
        }
      }
    }

    f4 O[NE];
#pragma unroll
    for (int e = 0; e < NE; ++e) O[e] = f4{0.f, 0.f, 0.f, 0.f};
    float m_run = kNothing, l_run = 0.f;  // of column c, times 2^15 (PAIR: l of this wave's positions)
    const uint8_t* ka = s_k + c * S_::KS + (HD == 64 ? 16 * (qd & 1) : 16 * J * qd) + 128 * wd;
    const uint8_t* za = s_z + c * NB + (HD == 64 ? qd & 1 : J * qd) + 8 * wd;
    auto turn = [&](uint32_t st, uint32_t next, bool inside) __attribute__((always_inline)) {
      // ---- scores of this wave's PT tiles ----
      f4 x[PT];
      f4 own[PAIR ? 2 : 1];
      // (PAIR: the other wave's two tiles first. A tile's rows are read while the one before is multiplied.)
      i4 A[2][J];
      uint32_t z[2];
      auto read_a = [&](int pp, int to) __attribute__((always_inline)) {
        const int p = PAIR ? (2 * (wd ^ 1) + pp) & 3 : pp;
#pragma unroll
        for (int j = 0; j < J; ++j) A[to][j] = *(const i4*)(ka + 16 * p * S_::KS + 16 * j);
        z[to] = J == 2 ? *(const uint16_t*)(za + 16 * p * NB) : za[16 * p * NB];
        if (HD == 64 && qd >= 2) z[to] = 127;  // (no dims there)
      };
      read_a(0, 0);
#pragma unroll
      for (int pp = 0; pp < 4; ++pp) {
        if (pp < 3) read_a(pp + 1, (pp + 1) & 1);
        __builtin_amdgcn_sched_barrier(0);
        f4 D = f4{0.f, 0.f, 0.f, 0.f};
        static_for<DIGITS * J>([&](auto k) __attribute__((always_inline)) {
          constexpr int d = DIGITS - 1 - decltype(k)::value / J, j = decltype(k)::value % J;  // (the smallest first)
          D = product<j, d % 4>(A[pp & 1][j], qb[d][j], D, z[pp & 1], d == 4 ? qs[j].y : qs[j].x);
        });
        if constexpr (!PAIR) x[pp] = D;
        else if (pp < 2) s_d[((wc * 2 + wd) * 2 + pp) * 64 + l] = D;
        else own[pp - 2] = D;
      }
      if constexpr (PAIR) {
        __syncthreads();
#pragma unroll
        for (int p = 0; p < 2; ++p) x[p] = own[p] + s_d[((wc * 2 + (wd ^ 1)) * 2 + p) * 64 + l];
      }
      if (__ballot(s_bad[l & 15])) {  // (uniform) a row of V that is not finite: NaN where it is seen
#pragma unroll
        for (int p = 0; p < PT; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (s_bad[4 * (p + (PAIR ? 2 * wd : 0)) + qd] >> i & 1u) x[p][i] = __builtin_nanf("");
      }
      if (!inside) {  // (uniform; the whole step twice, with and without, spills)
        const uint32_t pb = lo + TP * st + 32 * wd + 4 * qd - clo;
#pragma unroll
        for (int p = 0; p < PT; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[p][i] = pb + 16 * p + i < width ? x[p][i] : -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int p = 0; p < PT; ++p) mx = fmaxf(mx, fmaxf(fmaxf(x[p][0], x[p][1]), fmaxf(x[p][2], x[p][3])));
      mx = g4d::xmax32(g4d::xmax16(mx)) * sc;
      // P relative to a power of two (PAIR: of this wave's positions), so that a later one rescales it exactly
      const float m_own = fmaxf(m_run, ceilf(mx)), m_up = 15.f - m_own;
      float ps = 0.f;
      f4 P[4];  // (PAIR: this wave's two tiles, then all four)
#pragma unroll
      for (int p = 0; p < PT; ++p) {
#pragma unroll
        for (int i = 0; i < 4; ++i) P[p][i] = exp2_h(fmaf(x[p][i], sc, m_up));
        ps += (P[p][0] + P[p][1]) + (P[p][2] + P[p][3]);
      }
      ps = g4d::xsum32(g4d::xsum16(ps));
      float m_new = m_own;
      if constexpr (PAIR) {
        f4* pp = s_p + (wc * 2 * 2) * 64 + l;
        pp[(wd * 2) * 64] = P[0];
        pp[(wd * 2 + 1) * 64] = P[1];
        if (qd == 0) s_mx[wd * TC + 16 * wc + c] = m_own;
        __syncthreads();
        const float m_other = s_mx[(wd ^ 1) * TC + 16 * wc + c];
        m_new = fmaxf(m_own, m_other);
        const float f_own = exp2_h(m_own - m_new), f_other = exp2_h(m_other - m_new);
        ps *= f_own;
#pragma unroll
        for (int p = 0; p < 4; ++p) P[p] = pp[p * 64];
        if (__ballot(f_own != f_other)) {  // (powers of two, one of them 1)
          const float f0 = wd ? f_other : f_own, f1 = wd ? f_own : f_other;
#pragma unroll
          for (int p = 0; p < 4; ++p) P[p] *= p < 2 ? f0 : f1;
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
      // 32 positions and groups of four dims, the next group's operands read while one is multiplied
      const uint8_t* vb = s_v + wd * NE * 1024 + l * 16;
      b8 B[2][4];
      constexpr int GROUPS = NE / 4;
      auto read_b = [&](int u, b8* to) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          to[e] = *(const b8*)(vb + (u / GROUPS * (PAIR ? 2 : 1) * NE + u % GROUPS * 4 + e) * 1024);
      };
      read_b(0, B[0]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x[8];
        b8 part[3];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = P[2 * h + i / 4][i % 4];
        in_parts(x, part[2], part[1], part[0]);
#pragma unroll
        for (int u = h * GROUPS; u < (h + 1) * GROUPS; ++u) {
          if (u + 1 < 2 * GROUPS) read_b(u + 1, B[(u + 1) & 1]);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int k = 0; k < 3; ++k)  // (the smallest first)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              f4& o = O[u % GROUPS * 4 + e];
              o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(part[k], B[u & 1][e], o, 0, 0, 0);
            }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    for (uint32_t st = st0; st < st1; ++st) {
      __syncthreads();  // every wave is done with the previous step's rows
      store_step(st);
      __syncthreads();
      // the next step's rows are in flight during this one, K's from before its scores, V's from before its P V (past
      // the last step: its own rows again, not used)
      const uint32_t next = (min(st + 1, st1 - 1) - st0) % CH;
      if (next == 0 && st + 1 < st1) refill(st + 1);  // (uniform)
      load_k(next);
      const uint32_t p0 = lo + TP * st;
      turn(st, next, p0 >= all0 && p0 + TP - 1 <= all1);
    }

    // ---- columns 4 qd + i of the wave's tile, dims NE c + e (PAIR: 256 wd + 16 c + e) ----
    if constexpr (PAIR) {
      __syncthreads();
      if (qd == 0) s_mx[wd * TC + 16 * wc + c] = l_run;
      __syncthreads();
      l_run = s_mx[16 * wc + c] + s_mx[TC + 16 * wc + c];
    }
    const bool whole = st1 - st0 == pt.t.steps;
    float* part = a.part + (size_t)pt.slot * S_::SLOT;
    // Row by row through LDS (where V was), so that a wave stores whole KB: lanes storing their own 16 bytes of every 64
    // take four times the requests. Four dims of a lane turned by c: its 16 lanes meet different banks.
    constexpr int RD = NE * 16, QG = NE / 4, RPS = 16 / NE;  // a wave's dims of a row; a lane's groups; rows a store
    if constexpr (!PAIR) __syncthreads();  // (every wave is done with V)
    float* turn_s = (float*)s_v + w * 4 * RD;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float L = __shfl(l_run, 4 * qd + i, 64), f = whole ? 1.0f / L : 1.f;
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
    if (wd == 0 && qd == 0) {
      if (!whole) {
        part[16 * wc + c] = m_run;
        part[TC + 16 * wc + c] = l_run;
      } else if (MASS && g < ncols) {
        a.sums[row_of(a, first, kvh, g)] = make_float2(m_run, kTileP / l_run);
      }
    }
    if (st0 == 0 && tid == 0) a.meta[walk.tile_index(pt)] = pt.meta;
  }
  clear_rows<HD, S_::NTH>(a);
}

// out of a row and head from its tile's partials, in order: that of workgroup
// meta.x / 2 (slot meta.x), then slot 0 of each up to meta.y.
template <int HD>
__global__ __launch_bounds__(HD / 4) void attn4_tile_merge_kernel(Args a) {
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
  if (a.sums && d == 0) a.sums[blockIdx.x] = make_float2(M, kTileP / L);
}

// The weights of 256 positions of a sequence and KV head, a wave 64 of them: the
// scores again, of K rows that stay in registers, with q's digits as the tiles left
// them, 16 columns at a time through LDS; a lane adds up those of its column and
// positions, over 16 column tiles and then over all (a sum of thousands in one chain
// would be 2e-6 off), the lanes of a position at the end. The columns of a block of
// positions come in `splits` parts, which attn4_mass_kernel adds in order: a prompt's
// first block is seen by all of its columns and its last by few, so twice the
// workgroups that fit at once are dealt out (4500 rows of 8 heads, dim 128: 161 us with
// the attention, as many as fit 183; 168 with three parts of P), in parts of 4 column tiles or more (375 rows, dim
// 512: 53 us with the attention, of 8 tiles 63, of 2 51, but 68 at 750 rows for 66).
// The products take 5.5 us of 32 at 1500 rows and dim 512: what bounds it is the way
// to them, a row's page and digits, and one wave's exponentials beside another's products.
constexpr int WT = 256, WP = 256;  // threads, positions of a workgroup
template <int HD>
__global__ __launch_bounds__(WT, 2) void attn4_tile_weigh_kernel(Args a) {
  constexpr int J = HD < 128 ? 1 : HD / 128, NB = HD / BLOCK, PT = 4;
  constexpr int BYTES = DIGITS * J * 64 * 24, PIECES = BYTES / 16, PER = (PIECES + WT - 1) / WT;
  __shared__ __align__(16) uint8_t s_q[2][BYTES];
  const int tid = threadIdx.x, l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), qd = l >> 4, c = l & 15;
  const uint32_t s = blockIdx.y / a.nkh, kvh = blockIdx.y % a.nkh;
  const uint32_t block = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  const Seq q = seq_rows(a.rows, s);
  const uint32_t lo = first_seen(a, q), b0 = lo + block * WP;
  if (b0 >= q.len || !*a.done) return;  // (a length of 0 too)
  // rows that see any of the block's positions, and their columns, 16 at a time
  const uint32_t r0 = max(b0, q.base) - q.base, last = b0 + WP - 1;
  const bool leaves = a.window && a.window < q.len && last + a.window < q.len;  // the last rows do not see it
  const uint32_t r1 = leaves ? last + a.window - q.base : q.n;                   // past the last that does
  const uint32_t c0 = r0 * a.G / 16, c1 = (r1 * a.G + 15) / 16, per = (c1 - c0 + a.splits - 1) / a.splits;
  const uint32_t ct0 = min(c0 + split * per, c1), ct1 = min(ct0 + per, c1);
  const uint32_t ncols = q.n * a.G;

  i4 A[PT][J];
  uint32_t z[PT];
  const uint32_t rs = a.nkh * (HD / 2), ss = a.nkh * NB, tlast = (q.len - 1) / 16;
  const int32_t* list = a.page_table + (size_t)s * a.max_pages;
#pragma unroll
  for (int p = 0; p < PT; ++p) {
    const uint32_t t = min(b0 / 16 + 4 * w + p, tlast), at = page_of(a, t);
    const size_t tile = (size_t)clamp_page(a, list[at]) * a.page_tiles + (t - at * a.page_tiles);
    // (dims as the tiles have them: two neighbouring blocks a lane; at head dim 512 of each half)
    const uint32_t b = HD == 64 ? qd & 1 : HD == 128 ? qd : 2 * qd;
    const uint8_t* k = a.kp + tile * (16 * (size_t)rs) + c * rs + kvh * (HD / 2) + 16 * b;
    const uint8_t* y = a.ks + tile * (16 * (size_t)ss) + c * ss + kvh * NB + b;
#pragma unroll
    for (int j = 0; j < J; ++j) A[p][j] = *(const i4*)(k + 128 * (j / 2) + 16 * (j % 2));
    z[p] = J == 1 ? *y : *(const uint16_t*)y;
    if constexpr (J == 4) z[p] |= (uint32_t)*(const uint16_t*)(y + 8) << 16;
    if (HD == 64 && qd >= 2) z[p] = 127;  // (no dims there)
  }
  const float sc = a.scale_part == 0.f ? 1.f : fabsf(a.scale_part);
  const size_t first = (size_t)kvh * a.columns + first_columns(a, s, q);
  f4 sum[PT], part[PT];
#pragma unroll
  for (int p = 0; p < PT; ++p) sum[p] = part[p] = f4{0.f, 0.f, 0.f, 0.f};
  i4 next[PER];
  uint2 qnext[J];
  float2 mlnext{0.f, 0.f};
  auto load = [&](uint32_t ct) __attribute__((always_inline)) {
    const i4* from = (const i4*)(a.qdigits + (first + ct) * BYTES);
#pragma unroll
    for (int i = 0; i < PER; ++i) next[i] = from[min(i * WT + tid, PIECES - 1)];
#pragma unroll
    for (int j = 0; j < J; ++j) qnext[j] = a.qscales[((first + ct) * J + j) * 64 + l];
    mlnext = a.sums[row_of(a, q.first, kvh, min(16 * ct + c, ncols - 1))];
  };
  auto store = [&](int to) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i * WT + tid < PIECES) *(i4*)(s_q[to] + (i * WT + tid) * 16) = next[i];
  };
  if (ct0 < ct1) {
    load(ct0);
    store(0);
  }
  for (uint32_t ct = ct0; ct < ct1; ++ct) {
    const int at = (ct - ct0) & 1;
    const float2 ml = mlnext;
    uint2 qs[J];
#pragma unroll
    for (int j = 0; j < J; ++j) qs[j] = qnext[j];
    __syncthreads();
    if (ct + 1 < ct1) load(ct + 1);
    const uint32_t g = 16 * ct + c, gr = min(g, ncols - 1), cpos = q.base + div_g(a, gr);
    const uint32_t clo = a.window && cpos + 1 > a.window ? cpos + 1 - a.window : 0u;
    const uint32_t width = g < ncols ? cpos + 1 - clo : 0u;
    f4 D[PT];
#pragma unroll
    for (int p = 0; p < PT; ++p) D[p] = f4{0.f, 0.f, 0.f, 0.f};
    static_for<DIGITS * J>([&](auto k) __attribute__((always_inline)) {
      constexpr int d = DIGITS - 1 - decltype(k)::value / J, j = decltype(k)::value % J;  // (the smallest first)
      i6 B;
      read_digit(s_q[at] + ((d * J + j) * 64 + l) * 24, B);
#pragma unroll
      for (int p = 0; p < PT; ++p) D[p] = product<j, d % 4>(A[p][j], B, D[p], z[p], d == 4 ? qs[j].y : qs[j].x);
    });
    const uint32_t pb = b0 + 64 * w + 4 * qd - clo;
#pragma unroll
    for (int p = 0; p < PT; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        part[p][i] += pb + 16 * p + i < width ? exp2_h(fmaf(D[p][i], sc, -ml.x)) * ml.y : 0.f;
    if ((ct - ct0) % 16 == 15 || ct + 1 == ct1) {
#pragma unroll
      for (int p = 0; p < PT; ++p) {
        sum[p] += part[p];
        part[p] = f4{0.f, 0.f, 0.f, 0.f};
      }
    }
    if (ct + 1 < ct1) store(at ^ 1);
  }
  const size_t out = ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * WP;
#pragma unroll
  for (int p = 0; p < PT; ++p)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y = g4d::sum16(sum[p][i]);
      if (c == 4 * p + i) a.weights[out + 64 * w + 16 * p + 4 * qd + i] = y;
    }
}
// Adds the parts of each position's weight: 64 positions a workgroup, a wave every fourth part of them.
constexpr int SP = 64, SW = 4;
__global__ __launch_bounds__(SP * SW) void attn4_mass_kernel(Args a) {
  __shared__ float s_got[SW][SP];
  const int w = threadIdx.x / SP, i = threadIdx.x % SP;
  const uint32_t s = blockIdx.y / a.nkh, kvh = blockIdx.y % a.nkh, i0 = blockIdx.x * SP + i;  // (from the first seen)
  const Seq q = seq_rows(a.rows, s);
  const uint32_t t = first_seen(a, q) + i0;
  if (first_seen(a, q) + blockIdx.x * SP >= q.len || !*a.done) return;  // (uniform; a length of 0 too)
  const float* from = a.weights + ((size_t)blockIdx.y * a.blocks + i0 / WP) * a.splits * WP + i0 % WP;
  float got = 0.f;
  for (uint32_t k0 = w; k0 < a.splits; k0 += 16 * SW) {  // (16 on their way)
    float x[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) x[k] = from[(size_t)min(k0 + k * SW, a.splits - 1) * WP];
#pragma unroll
    for (int k = 0; k < 16; ++k) got += k0 + k * SW < a.splits ? x[k] : 0.f;
  }
  s_got[w][i] = got;
  __syncthreads();
  if (w || t >= q.len) return;
#pragma unroll
  for (int k = 1; k < SW; ++k) got += s_got[k][i];
  const uint32_t tile = t / 16, page = page_of(a, tile);
  const int32_t id = a.page_table[(size_t)s * a.max_pages + page];
  if (id >= 0 && id < (int32_t)a.num_pages)
    a.mass[((size_t)id * (a.page_tiles * 16) + (t - page * a.page_tiles * 16)) * a.nkh + kvh] += got;
}

bool step_fits(const g4_kv4_params& p) {
  return (uint64_t)p.max_rows * (p.num_q_heads / p.num_kv_heads) <= COLS;
}
// Units a sequence may have (a window of several rows spans max_rows - 1 more positions, and up to 15 of its first
// tile).
uint64_t most_units(const g4_kv4_params& p) {
  uint64_t span = p.max_seq_len;
  if (p.sliding_window) span = std::min<uint64_t>(span, (uint64_t)p.sliding_window + p.max_rows - 1 + 15);
  return (span + UNIT - 1) / UNIT;
}
size_t up256(size_t n) { return (n + 255) / 256 * 256; }
template <int HD>
uint32_t step_wgs(const g4_kv4_params& p) {
  return (uint32_t)std::min<uint64_t>(StepShape<HD>::WGS, most_units(p) * p.num_seqs * p.num_kv_heads);
}
// The parts of a workspace, one after the other.
struct Sizes {
  size_t meta, part, sums, scores, digits, scales, weights, done;
  size_t all() const { return meta + part + sums + scores + digits + scales + weights + done; }
};
// Many rows: 256 positions at a time of a sequence, parts of their columns (so many that the workgroups fill the device
// twice over, of four column tiles or more), and how often 16 columns may begin (those of each sequence by themselves).
uint64_t weigh_blocks(const g4_kv4_params& p) {
  uint64_t span = p.max_seq_len;
  if (p.sliding_window) span = std::min<uint64_t>(span, (uint64_t)p.sliding_window + p.max_rows - 1 + 15);
  return (span + WP - 1) / WP;
}
uint32_t weigh_splits(const g4_kv4_params& p) {
  const uint64_t blocks = weigh_blocks(p) * p.num_seqs * p.num_kv_heads, tiles = tiles_of(p) * (TC / 16);
  return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(1024 / blocks, tiles / 4));
}
uint64_t weigh_columns(const g4_kv4_params& p) {
  return (uint64_t)p.num_rows * (p.num_q_heads / p.num_kv_heads) / 16 + p.num_seqs + 1;
}
template <int HD>
uint32_t tile_wgs(const g4_kv4_params& p) {
  return (uint32_t)std::min<uint64_t>(TileShape<HD>::WGS, (all_cost(p) + kLeast - 1) / kLeast);
}
template <int HD>
Sizes sizes_of(const g4_kv4_params& p, bool mass) {
  Sizes z{};
  const size_t pairs = (size_t)p.num_seqs * p.num_kv_heads;
  if (step_fits(p)) {
    z.meta = up256(pairs * sizeof(uint2));
    z.part = up256(2ull * step_wgs<HD>(p) * StepShape<HD>::SLOT * sizeof(float));
    if (mass)
      z.scores = pairs * most_units(p) * (p.max_rows * (p.num_q_heads / p.num_kv_heads)) * UNIT * sizeof(float);
  } else {
    z.meta = up256(pairs * tiles_of(p) * sizeof(uint2));
    z.part = up256(2ull * tile_wgs<HD>(p) * TileShape<HD>::SLOT * sizeof(float));
    if (mass) {
      const size_t lanes = p.num_kv_heads * weigh_columns(p) * (HD < 128 ? 1 : HD / 128) * 64;
      z.digits = up256(lanes * DIGITS * 24);
      z.scales = up256(lanes * sizeof(uint2));
      z.weights = up256(pairs * weigh_blocks(p) * weigh_splits(p) * WP * sizeof(float));
      z.done = 256;
    }
  }
  if (mass) z.sums = up256((size_t)p.num_rows * p.num_q_heads * sizeof(float2));
  return z;
}

template <int HD>
int attend(g4_ctx* ctx, const g4_kv4_params& p, Args a, void* workspace) {
  const Sizes z = sizes_of<HD>(p, a.mass);
  uint8_t* w = (uint8_t*)workspace;
  a.meta = (uint2*)w;
  a.part = (float*)(w + z.meta);
  a.sums = a.mass ? (float2*)(w + z.meta + z.part) : nullptr;
  a.scores = (float*)(w + z.meta + z.part + z.sums);
  if (step_fits(p)) {
    const uint64_t units = most_units(p), pairs = (uint64_t)p.num_seqs * p.num_kv_heads;
    G4_REQUIRE((units + kSeqCost) * pairs < (1ull << 31), "g4_pagedAttn4: %u sequences of up to %u positions and %u KV heads in one "
               "call", p.num_seqs, p.max_seq_len, p.num_kv_heads);
    G4_REQUIRE(pairs * (p.max_rows * a.G + (a.mass ? 1 : 0)) < 1u << 23, "g4_pagedAttn4: %u sequences of up to %u rows of %u heads in one "
               "call", p.num_seqs, p.max_rows, p.num_q_heads);
    a.wgs = step_wgs<HD>(p);
    a.units = (uint32_t)units;
    a.columns = p.max_rows * a.G;
    const dim3 grid(a.wgs);
    if (a.mass) hipLaunchKernelGGL((attn4_step_kernel<HD, true>), grid, dim3(NT), 0, ctx->stream, a);
    else hipLaunchKernelGGL((attn4_step_kernel<HD, false>), grid, dim3(NT), 0, ctx->stream, a);
    G4_LAUNCHED(ctx, "attn4_step");
    const uint64_t merges = pairs * p.max_rows * a.G;
    const bool wide = std::min<uint64_t>(units, a.wgs) > 32 && merges < 1u << 20;
    const unsigned threads = wide ? 1024 : 256;
    if (a.mass) {
      // a position a thread, in at most 2^20 workgroups
      a.blocks = (uint32_t)std::min<uint64_t>(ceil_div(units * UNIT, threads), std::max<uint64_t>(1, (1u << 20) / pairs));
      const dim3 grid((unsigned)(merges + pairs * a.blocks));
      if (wide) hipLaunchKernelGGL((attn4_merge_kernel<HD, 1024, true>), grid, dim3(threads), 0, ctx->stream, a);
      else hipLaunchKernelGGL((attn4_merge_kernel<HD, 256, true>), grid, dim3(threads), 0, ctx->stream, a);
      G4_LAUNCHED(ctx, "attn4_merge");
    } else if (units > 1) {  // (else no sequence has partials)
      const dim3 grid((unsigned)merges);
      if (wide) hipLaunchKernelGGL((attn4_merge_kernel<HD, 1024, false>), grid, dim3(threads), 0, ctx->stream, a);
      else hipLaunchKernelGGL((attn4_merge_kernel<HD, 256, false>), grid, dim3(threads), 0, ctx->stream, a);
      G4_LAUNCHED(ctx, "attn4_merge");
    }
    return G4_OK;
  }
  a.tiles = tiles_of(p);
  G4_REQUIRE(all_cost(p) < (1ull << 31) && (uint64_t)a.tiles * p.num_seqs * p.num_kv_heads < (1ull << 31),
             "g4_pagedAttn4: %u sequences of up to %u rows and %u positions in one call", p.num_seqs, p.max_rows,
             p.max_seq_len);
  G4_REQUIRE((uint64_t)p.num_rows * p.num_q_heads < 1u << 25, "g4_pagedAttn4: %u rows of %u heads in one call",
             p.num_rows, p.num_q_heads);
  a.wgs = tile_wgs<HD>(p);
  if (a.mass) {
    a.columns = (uint32_t)weigh_columns(p);
    a.splits = weigh_splits(p);
    a.blocks = (uint32_t)weigh_blocks(p);
    a.qdigits = w + z.meta + z.part + z.sums + z.scores;
    a.qscales = (uint2*)(a.qdigits + z.digits);
    a.weights = (float*)((uint8_t*)a.qscales + z.scales);
    a.done = (uint32_t*)((uint8_t*)a.weights + z.weights);
  }
  const dim3 grid(a.wgs), threads(TileShape<HD>::NTH);
  if (a.mass) hipLaunchKernelGGL((attn4_tile_kernel<HD, true>), grid, threads, 0, ctx->stream, a);
  else hipLaunchKernelGGL((attn4_tile_kernel<HD, false>), grid, threads, 0, ctx->stream, a);
  G4_LAUNCHED(ctx, "attn4_tile");
  if (a.wgs > 1) {  // (else no tile has partials)
    hipLaunchKernelGGL(attn4_tile_merge_kernel<HD>, dim3(p.num_rows * p.num_q_heads), dim3(HD / 4), 0, ctx->stream, a);
    G4_LAUNCHED(ctx, "attn4_tile_merge");
  }
  if (!a.mass) return G4_OK;
  const unsigned pairs = p.num_seqs * p.num_kv_heads;
  hipLaunchKernelGGL(attn4_tile_weigh_kernel<HD>, dim3(a.blocks * a.splits, pairs), dim3(WT), 0, ctx->stream, a);
  G4_LAUNCHED(ctx, "attn4_tile_weigh");
  hipLaunchKernelGGL(attn4_mass_kernel, dim3(a.blocks * (WP / SP), pairs), dim3(SP * SW), 0, ctx->stream, a);
  G4_LAUNCHED(ctx, "attn4_mass");
  return G4_OK;
}

}  // namespace

extern "C" {

int g4_pagedAttn4_workspace_size(g4_kv4_params p, int with_mass, size_t* bytes) {
  G4_REQUIRE(bytes, "g4_pagedAttn4_workspace_size: null out");
  int rc = g4_internal_kv8_check(__func__, p, p.max_rows == 1 && p.num_rows == p.num_seqs ? nullptr : &p.num_rows);
  if (rc) return rc;
  const bool mass = with_mass != 0;
  G4_REQUIRE(!mass || step_fits(p) || weigh_blocks(p) * WP * SW < 1ull << 32,
             "%s: weights of many rows over up to %u positions", __func__, p.max_seq_len);  // (threads of the mass kernel)
  const Sizes z = p.head_dim == 64 ? sizes_of<64>(p, mass) : p.head_dim == 128 ? sizes_of<128>(p, mass)
                  : p.head_dim == 256 ? sizes_of<256>(p, mass) : sizes_of<512>(p, mass);
  *bytes = std::max<size_t>(z.all(), 16);
  return G4_OK;
}

int g4_pagedAttn4(g4_ctx* ctx, const float* q, const uint8_t* k_pool, const uint8_t* v_pool, const uint8_t* k_scale,
                  const uint8_t* v_scale, const int32_t* page_table, const uint32_t* seq_lens,
                  const uint32_t* row_starts, float* output, float* mass, g4_kv4_params p, void* workspace,
                  size_t workspace_bytes, void* ops) {
  G4_ENTER(ctx);
  G4_REQUIRE(q && k_pool && v_pool && k_scale && v_scale && page_table && seq_lens && output && workspace,
             "g4_pagedAttn4: null buffer");
  int rc = g4_internal_kv8_check(__func__, p, row_starts);
  if (rc) return rc;
  size_t need = 0;
  rc = g4_pagedAttn4_workspace_size(p, mass != nullptr, &need);
  if (rc) return rc;
  G4_REQUIRE(workspace_bytes >= need, "g4_pagedAttn4: workspace %zu bytes < %zu required", workspace_bytes, need);
  const uintptr_t all = (uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)output |
                        (uintptr_t)workspace | (uintptr_t)k_scale | (uintptr_t)v_scale;
  G4_REQUIRE((all & 15) == 0, "g4_pagedAttn4: rows, pools, scales and workspace must be 16-byte aligned");
  G4_REQUIRE(!ops || (p.head_dim % 256 == 0 && p.num_rows <= 64 && step_fits(p) && ((uintptr_t)ops & 15) == 0),
             "g4_pagedAttn4: operand blocks need head_dim a multiple of 256, <= 64 rows, <= 16 rows x heads of a KV "
             "head and a 16-byte aligned buffer");
  G4_REQUIRE(!mass || (uint64_t)p.num_seqs * p.num_kv_heads <= 65535, "g4_pagedAttn4: %u sequences of %u KV heads",
             p.num_seqs, p.num_kv_heads);
  int up = 0;
  double part = p.scale * kLog2e;
  if (std::isfinite(part)) part = std::frexp(part, &up);
  const Args a{paged_args(p, q, page_table, seq_lens, row_starts, output, ops), (float)part, up,
               k_pool, v_pool, k_scale, v_scale, mass, nullptr, nullptr, 0, 0, nullptr, nullptr, nullptr, 1, 0, nullptr};
  switch (p.head_dim) {
    case 64: return attend<64>(ctx, p, a, workspace);
    case 128: return attend<128>(ctx, p, a, workspace);
    case 256: return attend<256>(ctx, p, a, workspace);
    default: return attend<512>(ctx, p, a, workspace);
  }
}

}  // extern "C"
