// k_attn4.hip — attention over the 4-bit paged K/V pool (k_kv4.hip writes it),
// and the attention weight of its rows.
//
//   p[t] = softmax over t of scale * (q . k[t]),  out = sum p[t] * v[t],
//   mass[t] += sum of p[t] over a KV head's query heads and the sequence's rows
//
// attn4_row_kernel: a workgroup one row and query head, a wave every fourth
// position, one pass with the running maximum and sum. attn4_mass_kernel: a wave
// one position and KV head, the scores again with the rows' maxima and sums.
#include <algorithm>

#include "kv4.hpp"

namespace {

using namespace g4kv8;
using g4kv4::BLOCK;

constexpr int NT = 256, NW = NT / 64;

struct Args {
  const float* q;
  g4kv4::Pool pool;
  g4kv4::Shape sh;
  const int32_t* page_table;
  Rows rows;
  uint32_t nqh, G, max_pages, num_pages, window;
  float scale;
  float* out;
  float2* sums;  // maximum and 1 / sum of each row and query head
};

__device__ __forceinline__ uint32_t page_at(const Args& a, uint32_t s, uint32_t t) {
  const int32_t pg = a.page_table[(size_t)s * a.max_pages + t / a.sh.page_size];
  return pg < 0 ? 0u : min((uint32_t)pg, a.num_pages - 1);
}
// Dims l * HD / 64 .. of a row.
template <int HD>
__device__ __forceinline__ void read_row(const uint8_t* codes, const uint8_t* scales, uint32_t stride, int l, float* x) {
  constexpr int D = HD / 64;
#pragma unroll
  for (int e = 0; e < D; ++e) {
    const int d = l * D + e;
    x[e] = g4kv4::value_of(codes[d / 2] >> (4 * (d & 1))) * g4kv4::scale_of(scales[d / BLOCK * stride]);
  }
}
template <int HD>
__device__ __forceinline__ float score(const Args& a, const float* q, uint32_t pg, uint32_t slot, uint32_t h, int l) {
  constexpr int D = HD / 64;
  float k[D], x = 0.f;
  read_row<HD>(a.pool.k + a.sh.code(pg, slot, h), a.pool.ks + a.sh.k_scale(pg, slot, h, 0), 1, l, k);
#pragma unroll
  for (int e = 0; e < D; ++e) x = fmaf(q[e], k[e], x);
  return g4d::wave_sum_dpp(x) * a.scale;
}

template <int HD>
__global__ __launch_bounds__(NT) void attn4_row_kernel(Args a) {
  constexpr int D = HD / 64;
  __shared__ float s_m[NW], s_l[NW], s_o[NW * HD];
  const uint32_t row = blockIdx.x / a.nqh, hq = blockIdx.x % a.nqh, h = hq / a.G;
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint32_t s = seq_of_row(a.rows, row);
  if (s >= a.rows.num_seqs) return;
  const Seq sq = seq_rows(a.rows, s);
  if (row - sq.first >= sq.n) return;
  float* out = a.out + (size_t)blockIdx.x * HD;
  if (!sq.len) {
    for (int d = threadIdx.x; d < HD; d += NT) out[d] = 0.f;
    return;
  }
  const uint32_t pos = sq.base + (row - sq.first), lo = a.window && pos + 1 > a.window ? pos + 1 - a.window : 0u;
  float q[D], o[D], m = -INFINITY, sum = 0.f;
#pragma unroll
  for (int e = 0; e < D; ++e) {
    q[e] = a.q[(size_t)blockIdx.x * HD + l * D + e];
    o[e] = 0.f;
  }
  for (uint32_t t = lo + w; t <= pos; t += NW) {
    const uint32_t pg = page_at(a, s, t), slot = t % a.sh.page_size;
    const float x = score<HD>(a, q, pg, slot, h, l);
    const float mn = fmaxf(m, x), al = expf(m - mn), p = expf(x - mn);
    float v[D];
    read_row<HD>(a.pool.v + a.sh.code(pg, slot, h), a.pool.vs + a.sh.v_scale(pg, slot, h, 0), 16, l, v);
    m = mn;
    sum = sum * al + p;
#pragma unroll
    for (int e = 0; e < D; ++e) o[e] = o[e] * al + p * v[e];
  }
  if (l == 0) {
    s_m[w] = m;
    s_l[w] = sum;
  }
#pragma unroll
  for (int e = 0; e < D; ++e) s_o[w * HD + l * D + e] = o[e];
  __syncthreads();
  float M = s_m[0], L = 0.f;
  for (int i = 1; i < NW; ++i) M = fmaxf(M, s_m[i]);
  float f[NW];
  for (int i = 0; i < NW; ++i) {
    f[i] = s_m[i] == -INFINITY ? 1.f : expf(s_m[i] - M);  // (-Inf: sums of 0, or NaN)
    L += f[i] * s_l[i];
  }
  for (int d = threadIdx.x; d < HD; d += NT) {
    float y = 0.f;
    for (int i = 0; i < NW; ++i) y += f[i] * s_o[i * HD + d];
    out[d] = y / L;
  }
  if (a.sums && threadIdx.x == 0) a.sums[blockIdx.x] = make_float2(M, 1.0f / L);
}

template <int HD>
__global__ __launch_bounds__(NT) void attn4_mass_kernel(Args a) {
  constexpr int D = HD / 64;
  const uint32_t s = blockIdx.y / a.sh.nkh, h = blockIdx.y % a.sh.nkh;
  const int l = threadIdx.x & 63;
  const Seq sq = seq_rows(a.rows, s);
  for (uint32_t t = blockIdx.x * NW + (threadIdx.x >> 6); t < sq.len; t += gridDim.x * NW) {
    const int32_t id = a.page_table[(size_t)s * a.max_pages + t / a.sh.page_size];
    if (id < 0 || id >= (int32_t)a.num_pages) continue;
    const uint32_t slot = t % a.sh.page_size;
    float got = 0.f;
    for (uint32_t r = 0; r < sq.n; ++r) {
      const uint32_t pos = sq.base + r;
      if (t > pos || (a.window && t + a.window <= pos)) continue;
      for (uint32_t g = 0; g < a.G; ++g) {
        const size_t at = (size_t)(sq.first + r) * a.nqh + h * a.G + g;
        float q[D];
#pragma unroll
        for (int e = 0; e < D; ++e) q[e] = a.q[at * HD + l * D + e];
        const float2 ml = a.sums[at];
        got += expf(score<HD>(a, q, (uint32_t)id, slot, h, l) - ml.x) * ml.y;
      }
    }
    if (l == 0) a.pool.mass[a.sh.row((uint32_t)id, slot, h)] += got;
  }
}

template <int HD>
int attend(g4_ctx* ctx, const g4_kv4_params& p, const Args& a) {
  hipLaunchKernelGGL(attn4_row_kernel<HD>, dim3(p.num_rows * p.num_q_heads), dim3(NT), 0, ctx->stream, a);
  G4_LAUNCHED(ctx, "attn4_row");
  if (!a.sums) return G4_OK;
  const dim3 grid(std::min(ceil_div(p.max_seq_len, NW), 4096u), p.num_seqs * p.num_kv_heads);
  hipLaunchKernelGGL(attn4_mass_kernel<HD>, grid, dim3(NT), 0, ctx->stream, a);
  G4_LAUNCHED(ctx, "attn4_mass");
  return G4_OK;
}

}  // namespace

extern "C" {

int g4_pagedAttn4_workspace_size(g4_kv4_params p, int with_mass, size_t* bytes) {
  G4_REQUIRE(bytes, "g4_pagedAttn4_workspace_size: null out");
  int rc = g4_internal_kv8_check(__func__, p, p.max_rows == 1 && p.num_rows == p.num_seqs ? nullptr : &p.num_rows);
  if (rc) return rc;
  *bytes = with_mass ? (size_t)p.num_rows * p.num_q_heads * sizeof(float2) : 16;
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
  const uintptr_t all = (uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)output | (uintptr_t)workspace;
  G4_REQUIRE((all & 15) == 0, "g4_pagedAttn4: rows, pools and workspace must be 16-byte aligned");
  G4_REQUIRE(!ops, "g4_pagedAttn4: operand blocks are not written");
  G4_REQUIRE((uint64_t)p.num_rows * p.num_q_heads < 1u << 24, "g4_pagedAttn4: %u rows of %u heads in one call",
             p.num_rows, p.num_q_heads);
  G4_REQUIRE(!mass || (uint64_t)p.num_seqs * p.num_kv_heads <= 65535, "g4_pagedAttn4: %u sequences of %u KV heads",
             p.num_seqs, p.num_kv_heads);
  const Args a{q,
               {(uint8_t*)k_pool, (uint8_t*)v_pool, (uint8_t*)k_scale, (uint8_t*)v_scale, mass},
               {p.page_size, p.num_kv_heads, p.head_dim},
               page_table,
               {seq_lens, row_starts, p.num_seqs, p.num_rows, p.max_rows, p.max_seq_len},
               p.num_q_heads,
               p.num_q_heads / p.num_kv_heads,
               p.max_pages,
               p.num_pages,
               p.sliding_window,
               p.scale,
               output,
               mass ? (float2*)workspace : nullptr};
  switch (p.head_dim) {
    case 64: return attend<64>(ctx, p, a);
    case 128: return attend<128>(ctx, p, a);
    case 256: return attend<256>(ctx, p, a);
    default: return attend<512>(ctx, p, a);
  }
}

}  // extern "C"
