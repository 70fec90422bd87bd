// k_logprobs.hip — log probabilities of given tokens, entropy and the likeliest
// alternatives of rows of logits (g4_logprobsBatch in g4hip.h).
#include "g4_internal.hpp"

namespace {

constexpr int NT = 256;

// Order of the alternatives: larger value first, equal ones by index, NaN last.
struct Top {
  float v;
  uint32_t i;
};
__device__ __forceinline__ bool before(const Top& a, const Top& b) {
  if (a.v != a.v) return b.v != b.v && a.i < b.i;
  return b.v != b.v || a.v > b.v || (a.v == b.v && a.i < b.i);
}

struct Args {
  const float* x;
  const uint32_t* tokens;
  uint32_t size, ntop;
  float *logprobs, *entropy, *top_logprobs;
  uint32_t* top_ids;
};

__device__ float block_reduce(float v, float* red, bool mx) {
  v = mx ? g4d::wave_max(v) : g4d::wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return mx ? fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])) : (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ __launch_bounds__(NT) void logprobs_kernel(Args a) {
  __shared__ float red[4];
  __shared__ Top best[NT];
  const uint32_t r = blockIdx.x, t = threadIdx.x;
  const float* x = a.x + (size_t)r * a.size;
  float m = -INFINITY, bad = 0.f;
  for (uint32_t i = t; i < a.size; i += NT) {
    m = fmaxf(m, x[i]);
    if (x[i] != x[i] || x[i] == INFINITY) bad = 1.f;
  }
  m = block_reduce(m, red, true);
  bad = block_reduce(bad, red, true);
  if (m == -INFINITY) bad = 1.f;
  double zd = 0.0, hd = 0.0;  // (in f32 a likely token's 1 swallows the ends of the others behind it)
  for (uint32_t i = t; i < a.size; i += NT) {
    const float d = x[i] - m, e = expf(d);
    zd += e;
    hd += e > 0.f ? e * d : 0.f;
  }
  __shared__ double red64[2 * NT];
  red64[t] = zd;
  red64[NT + t] = hd;
  __syncthreads();
  zd = hd = 0.0;
  for (int i = 0; i < NT; ++i) {
    zd += red64[i];
    hd += red64[NT + i];
  }
  const float lz = bad > 0.f ? __builtin_nanf("") : (float)log(zd);
  if (t == 0) {
    if (a.logprobs) a.logprobs[r] = a.tokens[r] < a.size ? (x[a.tokens[r]] - m) - lz : __builtin_nanf("");
    if (a.entropy) a.entropy[r] = (float)(log(zd) - hd / zd) + (lz - lz);
  }
  Top last{INFINITY, 0};
  for (uint32_t k = 0; k < a.ntop; ++k) {
    Top c{__builtin_nanf(""), 0xffffffffu};
    for (uint32_t i = t; i < a.size; i += NT) {
      const Top n{x[i], i};
      if ((k == 0 || before(last, n)) && before(n, c)) c = n;
    }
    __syncthreads();
    best[t] = c;
    __syncthreads();
    for (int s = NT / 2; s > 0; s >>= 1) {
      if (t < (uint32_t)s && before(best[t + s], best[t])) best[t] = best[t + s];
      __syncthreads();
    }
    last = best[0];
    if (t == 0) {
      a.top_ids[(size_t)r * a.ntop + k] = last.i;
      a.top_logprobs[(size_t)r * a.ntop + k] = (last.v - m) - lz;
    }
  }
}

int check_shape(uint32_t size, uint32_t batch, uint32_t ntop) {
  G4_REQUIRE(size > 0 && size <= 0x7fffffffu && batch > 0 && batch <= 65535 && ntop <= 64 && ntop <= size,
             "g4_logprobsBatch: 1..65535 rows of logits, ntop (%u) at most 64 and the row's size (%u)", ntop, size);
  return G4_OK;
}

}  // namespace

extern "C" {

int g4_logprobsBatch_workspace_size(uint32_t size, uint32_t batch, uint32_t ntop, size_t* bytes) {
  G4_REQUIRE(bytes, "g4_logprobsBatch_workspace_size: null out");
  int rc = check_shape(size, batch, ntop);
  if (rc) return rc;
  *bytes = 16;
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
  const Args a{logits, tokens, size, ntop, logprobs, entropy, top_logprobs, top_ids};
  hipLaunchKernelGGL(logprobs_kernel, dim3(batch), dim3(NT), 0, ctx->stream, a);
  G4_LAUNCHED(ctx, "logprobs");
  return G4_OK;
}

}  // extern "C"
