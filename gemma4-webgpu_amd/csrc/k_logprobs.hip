// k_logprobs.hip — log probabilities of given tokens, entropy and the likeliest
// alternatives of rows of logits (g4_logprobsBatch in g4hip.h).
//
//   m = max x, z = sum e^(x - m), h = sum (x - m) e^(x - m):
//   logprob = x[token] - m - log z, entropy = log z - h / z.
//
// Reading the logits bounds it. Workgroup (chunk, row) holds its part of the
// row in registers, 8 or 32 values a thread, from one round of 16-byte loads, and leaves
// (m, z, h) of the chunk and its ntop largest; a second launch, a workgroup a
// row, joins them: z_row = sum z_c e^(m_c - m), h_row = sum (h_c + (m_c - m) z_c) e^(m_c - m).
//
// The largest of a chunk: the ntop-th largest of the 256 threads' maxima
// (bisected on their ordered bits by counting lanes, no sort) has ntop values at
// or above it, so only what reaches it - some 21 of 8192 values at ntop 20 - goes
// to LDS, where each counts those before it. (A bound from each wave's 64 lanes
// alone lets 64 through.) The row's are found in the same way from the chunks'
// r-th largest. Where too many reach a bound (rows of equal or masked values)
// they are taken one after the other: ntop rounds over the chunk, whose values
// the caches then hold (64 rows of 262144, ntop 20, masked but for 20 tokens: 221 us a
// call, 23 unmasked and with 2000 left; ntop 5: 60 and 20; one row 59 and 13).
//
// Sums: eight values in f32, the rest in f64: behind a likely token's 1 the
// 30000 others of 1e-7 each would otherwise fall below half a step.
//
// Measured: 500 rows of 100003 (200 MB) 38 us, 5.3 TB/s, and 5 for the join; 64 of
// 262144 17.3 and 5.0 (a workgroup has one round of loads, whose arrival nothing
// hides); one row 5.3 and 4.2, two launches of 2.3 when empty.
#include <algorithm>

#include "g4_internal.hpp"

namespace {

typedef float f4a __attribute__((ext_vector_type(4), aligned(4)));  // rows are aligned as a float is

constexpr int NT = 256, NW = NT / 64;
constexpr uint32_t CAP = 1024;  // candidates held in LDS
constexpr float kLog2e = 1.44269504f;

// Bits that order as the values do; -0 as 0, a NaN (0) behind every number.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return v == v ? b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u) : 0u;
}
__device__ __forceinline__ float unordered(uint32_t k) {
  return k ? __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)) : __builtin_nanf("");
}
// An alternative: its value's bits over its index's complement, so that the
// larger number comes first, equal values by index. 0 is none.
typedef uint64_t Top;
__device__ __forceinline__ Top make_top(float v, uint32_t i) { return (Top)ordered(v) << 32 | ~i; }

struct Stat {
  double z, h;  // NaN where the chunk holds a NaN or +Inf
  float m;
  uint32_t pad;
};

struct Args {
  const float* x;
  const uint32_t* tokens;
  uint32_t size, ntop, chunks;
  float *logprobs, *entropy, *top_logprobs;
  uint32_t* top_ids;
  Stat* stat;  // [row][chunk]
  Top* top;    // [row][chunk][ntop], in order
};

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(v, 63);
}
__device__ __forceinline__ Top wave_first(Top t) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) t = max(t, (Top)__shfl_xor((unsigned long long)t, o, 64));
  return t;
}

// The largest value that `need` of the wave's 64 N keys reach, or a smaller one
// that exactly `need` reach (0: fewer keys are not 0).
template <int N>
__device__ __forceinline__ uint32_t reached_by(const uint32_t (&key)[N], uint32_t need) {
  uint32_t most = 0, least = 0, some = 0;  // (of those that are not 0; the least as its complement)
#pragma unroll
  for (int i = 0; i < N; ++i) {
    most = max(most, key[i]);
    least = max(least, key[i] ? ~key[i] : 0u);
    some += __popcll(__ballot(key[i] != 0));
  }
  if (some < need) return 0;
  uint32_t hi = wave_max_u32(most), lo = ~wave_max_u32(least);  // lo: reached by enough; above hi: by too few
  while (lo < hi) {
    const uint32_t mid = hi - (hi - lo) / 2;
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) n += __popcll(__ballot(key[i] >= mid));
    if (n >= need) {
      lo = mid;
      if (n == need) break;
    } else {
      hi = mid - 1;
    }
  }
  return lo;
}

// The n candidates in LDS, each to its rank where that is below ntop (every
// thread calls it; the candidates' order in LDS does not matter). Up to 64 of
// them are counted by the four waves together.
template <typename Out>
__device__ __forceinline__ void by_rank(const Top* list, uint32_t n, uint32_t ntop, uint32_t (*cnt)[64], Out&& out) {
  const uint32_t tid = threadIdx.x;
  if (n <= 64) {  // (uniform)
    const uint32_t i = tid & 63, w = tid >> 6;
    const Top t = list[min(i, n - 1)];
    uint32_t r = 0;
#pragma unroll 4
    for (uint32_t j = w; j < n; j += NW) r += list[j] > t;
    cnt[w][i] = r;
    __syncthreads();
    r = cnt[0][i] + cnt[1][i] + cnt[2][i] + cnt[3][i];
    if (tid < n && r < ntop) out(r, t);
    return;
  }
  for (uint32_t i = tid; i < n; i += NT) {
    const Top t = list[i];
    uint32_t r = 0;
#pragma unroll 8
    for (uint32_t j = 0; j < n; ++j) r += list[j] > t;
    if (r < ntop) out(r, t);
  }
}

// E values a thread: vectors of 4, NT threads apart.
template <int E>
__global__ __launch_bounds__(NT) void logprobs_chunk_kernel(Args a) {
  __shared__ float s_lm[NT];
  __shared__ uint32_t s_n, s_cnt[NW][64];
  __shared__ double s_z[NW], s_h[NW];
  __shared__ Top s_list[CAP], s_best[NW];
  constexpr int V = E / 4;
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6;
  const uint32_t chunk = blockIdx.x, row = blockIdx.y;
  const float* x = a.x + (size_t)row * a.size;
  const uint32_t first = chunk * (NT * E);
  auto index = [&](int e) { return first + (e / 4 * NT + tid) * 4 + e % 4; };  // of this thread's value e
  float v[E];
  const bool inside = first + NT * E <= a.size;  // (uniform)
  if (inside) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const f4a y = *(const f4a*)(x + index(4 * k));
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * k + i] = y[i];
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = index(e) < a.size ? x[index(e)] : -INFINITY;
  }
  float lm = -INFINITY;  // (a NaN is not the larger one)
#pragma unroll
  for (int e = 0; e < E; ++e) lm = fmaxf(lm, v[e]);
  s_lm[tid] = lm;
  if (tid == 0) s_n = 0;
  __syncthreads();
  float all[NW], m = -INFINITY;  // lane l's maxima in the four waves
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    all[i] = s_lm[64 * i + l];
    m = fmaxf(m, all[i]);
  }
  m = g4d::wave_max_dpp(m);
  const float mf = m == -INFINITY ? 0.f : m;
  double z = 0.0, h = 0.0;
#pragma unroll
  for (int g = 0; g < E; g += 8) {
    float zs[8], hs[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float d = v[g + i] - mf;
      d = d < -200.f ? -200.f : d;  // (e^-200 is 0, and so is 0 times it; -Inf ends here, a NaN and an Inf - Inf go on)
      zs[i] = __builtin_amdgcn_exp2f(d * kLog2e);
      hs[i] = d * zs[i];
    }
#pragma unroll
    for (int s = 4; s > 0; s /= 2)
#pragma unroll
      for (int i = 0; i < s; ++i) {
        zs[i] += zs[i + s];
        hs[i] += hs[i + s];
      }
    z += (double)zs[0];
    h += (double)hs[0];
  }
  z = g4d::wave_sum_dpp(z);
  h = g4d::wave_sum_dpp(h);
  if (l == 0) {
    s_z[w] = z;
    s_h[w] = h;
  }
  Top* top = a.top + ((size_t)row * a.chunks + chunk) * a.ntop;
  float t = -INFINITY;
  if (a.ntop) {
    const uint32_t key[NW] = {ordered(all[0]), ordered(all[1]), ordered(all[2]), ordered(all[3])};
    t = unordered(reached_by(key, a.ntop));
  }
  // (a bound of -Inf in a row's last chunk: what fills it up would reach it, too)
  if (a.ntop && (inside || t > -INFINITY) && __ballot(lm >= t)) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool in = v[e] >= t;
      const unsigned long long who = __ballot(in);
      if (who) {
        uint32_t at = 0;
        if (l == 0) at = atomicAdd(&s_n, (uint32_t)__popcll(who));
        const uint32_t below = __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0);
        at = __builtin_amdgcn_readfirstlane(at) + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), below);
        if (in && at < CAP) s_list[at] = make_top(v[e], index(e));
      }
    }
  }
  __syncthreads();
  if (tid == 0) {
    a.stat[(size_t)row * a.chunks + chunk] =
        Stat{(s_z[0] + s_z[1]) + (s_z[2] + s_z[3]), (s_h[0] + s_h[1]) + (s_h[2] + s_h[3]), m, 0};
  }
  if (!a.ntop) return;
  const uint32_t n = s_n;
  if (n >= a.ntop && n <= CAP) {
    by_rank(s_list, n, a.ntop, s_cnt, [&](uint32_t r, Top c) { top[r] = c; });
    return;
  }
  // one after the other: the first behind the last one taken (read again: values kept for this cost registers)
  const uint32_t end = min(first + NT * E, a.size);
  Top last = ~(Top)0;
  for (uint32_t k = 0; k < a.ntop; ++k) {
    Top c = 0;
#pragma unroll 4
    for (uint32_t i = first + tid; i < end; i += NT) {
      const Top y = make_top(x[i], i);
      c = y < last && y > c ? y : c;
    }
    c = wave_first(c);
    __syncthreads();
    if (l == 0) s_best[w] = c;
    __syncthreads();
    last = max(max(s_best[0], s_best[1]), max(s_best[2], s_best[3]));
    if (tid == 0) top[k] = last;
    if (!last) {  // (uniform) no more
      for (uint32_t r = k + 1 + tid; r < a.ntop; r += NT) top[r] = 0;
      return;
    }
  }
}

__global__ __launch_bounds__(NT) void logprobs_row_kernel(Args a) {
  __shared__ float s_m[NW];
  __shared__ double s_z[NW], s_h[NW];
  __shared__ Top s_list[CAP], s_best[NW];
  __shared__ uint32_t s_n, s_cnt[NW][64];
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6;
  const uint32_t row = blockIdx.x;
  const Stat* st = a.stat + (size_t)row * a.chunks;
  const Top* top = a.top + (size_t)row * a.chunks * a.ntop;
  // Of the chunks' r-th largest, lane l holding the largest of every 64th chunk's,
  // the ceil(ntop / r)-th: r ceil(ntop / r) values are at or above it. Half of
  // the lanes or fewer are to reach it.
  const uint32_t lanes = min(a.chunks, 64u), r = a.ntop ? min(max(1u, (2 * a.ntop + lanes - 1) / lanes), a.ntop) : 1u;
  float m = -INFINITY;
  for (uint32_t c = tid; c < a.chunks; c += NT) m = fmaxf(m, st[c].m);
  uint32_t bound = 0;
  if (a.ntop) {
    uint32_t key[1] = {0};
    for (uint32_t c = l; c < a.chunks; c += 64) key[0] = max(key[0], (uint32_t)(top[(size_t)c * a.ntop + r - 1] >> 32));
    bound = reached_by(key, (a.ntop + r - 1) / r);
  }
  m = g4d::wave_max_dpp(m);
  if (tid == 0) s_n = 0;
  if (l == 0) s_m[w] = m;
  __syncthreads();
  m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  double z = 0.0, h = 0.0;
  for (uint32_t c = tid; c < a.chunks; c += NT) {
    const Stat s = st[c];
    if (s.m == -INFINITY && s.z == s.z) continue;  // no probability
    const double d = (double)s.m - (double)m, f = exp(d);
    z += f * s.z;
    h += f * (s.h + d * s.z);
  }
  z = g4d::wave_sum_dpp(z);
  h = g4d::wave_sum_dpp(h);
  if (l == 0) {
    s_z[w] = z;
    s_h[w] = h;
  }
  const uint32_t all = a.chunks * a.ntop;
  for (uint32_t i = tid; i < all; i += NT) {
    const Top t = top[i];
    if (t && (uint32_t)(t >> 32) >= bound) {
      const uint32_t at = atomicAdd(&s_n, 1u);
      if (at < CAP) s_list[at] = t;
    }
  }
  __syncthreads();
  z = (s_z[0] + s_z[1]) + (s_z[2] + s_z[3]);
  h = (s_h[0] + s_h[1]) + (s_h[2] + s_h[3]);
  const double lz = z > 0.0 ? log(z) : __builtin_nan("");  // (0: nothing but -Inf; NaN stays)
  const float* x = a.x + (size_t)row * a.size;
  if (tid == 0) {
    if (a.logprobs) {
      const uint32_t t = a.tokens[row];
      a.logprobs[row] = t < a.size ? (float)((double)x[t] - (double)m - lz) : __builtin_nanf("");
    }
    if (a.entropy) a.entropy[row] = (float)(lz - h / z);
  }
  if (!a.ntop) return;
  auto put = [&](uint32_t r, Top t) {
    a.top_ids[(size_t)row * a.ntop + r] = ~(uint32_t)t;
    a.top_logprobs[(size_t)row * a.ntop + r] = (float)((double)unordered((uint32_t)(t >> 32)) - (double)m - lz);
  };
  const uint32_t n = s_n;
  if (n >= a.ntop && n <= CAP) {
    by_rank(s_list, n, a.ntop, s_cnt, put);
    return;
  }
  Top last = ~(Top)0;
  for (uint32_t k = 0; k < a.ntop; ++k) {
    Top c = 0;
    for (uint32_t i = tid; i < all; i += NT) {
      const Top y = top[i];
      c = y < last && y > c ? y : c;
    }
    c = wave_first(c);
    __syncthreads();
    if (l == 0) s_best[w] = c;
    __syncthreads();
    last = max(max(s_best[0], s_best[1]), max(s_best[2], s_best[3]));
    if (tid == 0) put(k, last);
  }
}

// Values a thread: 32 (64 rows of 262144 22.2 us; 16 values 25.8, 24 23.5, 48 22.5,
// 64 22.1), or 8 where 32 would leave the launch with less than two workgroups per
// CU (one row 9.5 us, with 32 9.8).
uint32_t chunks_of(uint32_t size, uint32_t e) { return ceil_div(size, NT * e); }
constexpr uint32_t kManyChunks = 512;
uint32_t pick_e(uint32_t size, uint32_t batch) { return (uint64_t)chunks_of(size, 32) * batch >= kManyChunks ? 32 : 8; }
// Chunks of the batch or of any smaller one, whichever has most: the most rows that take 8 values a thread may have
// more of them than the batch, whose workspace serves those calls too.
size_t most_chunks(uint32_t size, uint32_t batch) {
  const uint32_t few = std::min(batch, (kManyChunks - 1) / chunks_of(size, 32));
  return std::max((size_t)batch * chunks_of(size, pick_e(size, batch)), (size_t)few * chunks_of(size, 8));
}

int check_shape(uint32_t size, uint32_t batch, uint32_t ntop) {
  G4_REQUIRE(size > 0 && size <= (1u << 28) && batch > 0 && batch <= 65535 && ntop <= 64 && ntop <= size,
             "g4_logprobsBatch: 1..65535 rows of at most 2^28 logits, ntop (%u) at most 64 and the row's size (%u)",
             ntop, size);
  return G4_OK;
}

}  // namespace

extern "C" {

int g4_logprobsBatch_workspace_size(uint32_t size, uint32_t batch, uint32_t ntop, size_t* bytes) {
  G4_REQUIRE(bytes, "g4_logprobsBatch_workspace_size: null out");
  int rc = check_shape(size, batch, ntop);
  if (rc) return rc;
  *bytes = most_chunks(size, batch) * (sizeof(Stat) + ntop * sizeof(Top));
  return G4_OK;
}

int g4_logprobsBatch(g4_ctx* ctx, const float* logits, const uint32_t* tokens, uint32_t size, uint32_t batch,
                     float* logprobs, float* entropy, uint32_t ntop, uint32_t* top_ids, float* top_logprobs,
                     void* workspace, size_t workspace_bytes) {
  G4_ENTER(ctx);
  size_t need = 0;
  int rc = g4_logprobsBatch_workspace_size(size, batch, ntop, &need);
  if (rc) return rc;
  G4_REQUIRE(logits && workspace, "g4_logprobsBatch: null buffer");
  G4_REQUIRE(!tokens == !logprobs, "g4_logprobsBatch: tokens and logprobs go together");
  G4_REQUIRE(ntop == 0 || (top_ids && top_logprobs), "g4_logprobsBatch: null top buffer");
  G4_REQUIRE(workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0,
             "g4_logprobsBatch: workspace %zu bytes < %zu required, or not 16-byte aligned", workspace_bytes, need);
  const uint32_t e = pick_e(size, batch), chunks = chunks_of(size, e);
  Stat* stat = (Stat*)workspace;
  const Args a{logits, tokens, size, ntop, chunks, logprobs, entropy, top_logprobs, top_ids, stat,
               (Top*)(stat + (size_t)batch * chunks)};
  const dim3 grid(chunks, batch);
  if (e == 32) hipLaunchKernelGGL(logprobs_chunk_kernel<32>, grid, dim3(NT), 0, ctx->stream, a);
  else hipLaunchKernelGGL(logprobs_chunk_kernel<8>, grid, dim3(NT), 0, ctx->stream, a);
  G4_LAUNCHED(ctx, "logprobs_chunk");
  hipLaunchKernelGGL(logprobs_row_kernel, dim3(batch), dim3(NT), 0, ctx->stream, a);
  G4_LAUNCHED(ctx, "logprobs_row");
  return G4_OK;
}

}  // extern "C"
