// k_attn8.hip — attention over the 8-bit paged K/V pool (k_kv8.hip writes it).
#include "kv8.hpp"

namespace {

using namespace g4kv8;

constexpr int NT = 256;

struct Args {
  const float* q;
  const int8_t *kp, *vp;
  const float *ks, *vs;
  const int32_t* page_table;
  Rows rows;
  uint32_t nqh, nkh, hd, page_size, max_pages, num_pages, window;
  float scale;
  float* out;
};

// One workgroup per row and query head: 256 positions at a time, one score a
// thread, then one or two output dims a thread.
__global__ __launch_bounds__(NT) void attn8_kernel(Args a) {
  __shared__ float s_q[512], s_p[NT], s_red[8];
  __shared__ int s_pg[NT];
  const uint32_t row = blockIdx.y, head = blockIdx.x, kvh = head / (a.nqh / a.nkh), t = threadIdx.x;
  const uint32_t s = seq_of_row(a.rows, row);
  if (s >= a.rows.num_seqs) return;
  const Seq sq = seq_rows(a.rows, s);
  if (!sq.n) return;
  float* out = a.out + ((size_t)row * a.nqh + head) * a.hd;
  const uint32_t end = sq.len ? sq.base + (row - sq.first) + 1 : 0u;
  const uint32_t lo = a.window && end > a.window ? end - a.window : 0u;
  for (uint32_t d = t; d < a.hd; d += NT) s_q[d] = a.q[((size_t)row * a.nqh + head) * a.hd + d];
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (uint32_t p0 = lo; p0 < end; p0 += NT) {
    const uint32_t pos = min(p0 + t, end - 1);
    int32_t pg = a.page_table[(size_t)s * a.max_pages + pos / a.page_size];
    pg = pg < 0 ? 0 : (pg >= (int32_t)a.num_pages ? (int32_t)a.num_pages - 1 : pg);
    __syncthreads();
    s_pg[t] = pg;
    const int8_t* k = a.kp + (((size_t)pg * a.page_size + pos % a.page_size) * a.nkh + kvh) * a.hd;
    float x = 0.f;
    for (uint32_t d = 0; d < a.hd; ++d) x = fmaf(s_q[d], (float)k[d], x);
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
      const int8_t* v = a.vp + (((size_t)g * a.page_size + (p0 + i) % a.page_size) * a.nkh + kvh) * a.hd;
      const float w = s_p[i] * a.vs[(size_t)g * a.nkh + kvh];
      if (t < a.hd) o0 = fmaf(w, (float)v[t], o0);
      if (t + NT < a.hd) o1 = fmaf(w, (float)v[t + NT], o1);
    }
  }
  if (t < a.hd) out[t] = end ? o0 / l : 0.f;
  if (t + NT < a.hd) out[t + NT] = end ? o1 / l : 0.f;
}

}  // namespace

extern "C" {

int g4_pagedAttn8_workspace_size(g4_kv8_params p, size_t* bytes) {
  G4_REQUIRE(bytes, "g4_pagedAttn8_workspace_size: null out");
  int rc = g4_internal_kv8_check(__func__, p, p.max_rows == 1 && p.num_rows == p.num_seqs ? nullptr : &p.num_rows);
  if (rc) return rc;
  *bytes = 16;
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
  const Args a{q, k_pool, v_pool, k_scale, v_scale, page_table,
               {seq_lens, row_starts, p.num_seqs, p.num_rows, p.max_rows, p.max_seq_len},
               p.num_q_heads, p.num_kv_heads, p.head_dim, p.page_size, p.max_pages, p.num_pages, p.sliding_window,
               p.scale, output};
  hipLaunchKernelGGL(attn8_kernel, dim3(p.num_q_heads, p.num_rows), dim3(NT), 0, ctx->stream, a);
  G4_LAUNCHED(ctx, "attn8");
  return G4_OK;
}

}  // extern "C"
