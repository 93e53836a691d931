// Attention of drafted-tree rows over the 8-bit KV cache (hg_op_kv8_attn).
#include "hg_kv8.cuh"

namespace hg {

// One CTA per (row, q head), four warps; a warp takes every fourth visible slot (the context's, then the
// row's path) and keeps a running maximum, sum and weighted value row; lanes own neighbouring dims.
template <int HD>
__global__ void __launch_bounds__(128) k_kv8_attn(hg_kv8_cache C, hg_rows R, int nh, const float* __restrict__ q,
                                                  float* __restrict__ out) {
  constexpr int E = HD / 32;
  const int row = blockIdx.x, h = blockIdx.y, g = nh / C.n_kv_heads, kvh = h / g;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int s = -1;
  SeqSpan sp{};
  for (int i = 0; i < R.n_seqs; i++)
    if (R.row_off[i] <= row && row < R.row_off[i + 1]) s = i;
  if (s < 0) return;
  sp = kv8_span(R, s, true);
  const int j = row - sp.r0;
  if (j >= sp.n) return;
  float x[E], acc[E], m = -INFINITY, l = 0.0f;
  const float scale = 1.0f / sqrtf((float)HD);
#pragma unroll
  for (int e = 0; e < E; e++) {
    x[e] = q[((size_t)row * nh + h) * HD + lane * E + e] * scale;
    acc[e] = 0.0f;
  }
  auto attend = [&](long long slot) {
    const uint8_t* b = kv8_block(C, s, slot, kvh);
    if (!b) {
      kv8_flag(R.err, HG_ERR_CONTEXT);
      return;
    }
    const int w = (int)(slot % KV8_PAGE);
    float d = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++)
      d = __fmaf_rn(x[e], (float)(int8_t)b[kv8_k_off(HD, w, lane * E + e)], d);
    d = warp_sum(d) * *reinterpret_cast<const float*>(b + kv8_ks_off(HD, w));
    const float mn = fmaxf(m, d), al = m == -INFINITY ? 0.0f : expf(m - mn), p = expf(d - mn);
    const float pv = p * *reinterpret_cast<const float*>(b + kv8_vs_off(HD, w));
    l = l * al + p;
#pragma unroll
    for (int e = 0; e < E; e++)
      acc[e] = __fmaf_rn(pv, (float)(int8_t)b[kv8_v_off(HD, w, lane * E + e)], acc[e] * al);
    m = mn;
  };
  const int par = kv8_parent(R, sp, j);
  if (par != -2) {
    const long long cap = (long long)C.bt_stride * KV8_PAGE;
    if (sp.start > cap) kv8_flag(R.err, HG_ERR_CONTEXT);
    for (long long t = warp; t < min((long long)sp.start, cap); t += 4) attend(t);
    int at = j, k = 0;
    while (at >= 0) {
      const int up = kv8_parent(R, sp, at);
      if (up == -2) break;
      if ((k++ & 3) == warp) attend((long long)sp.start + at);
      at = up;
    }
  }
  __shared__ float ms[4], ls[4], os[4][HD];
  if (lane == 0) ms[warp] = m, ls[warp] = l;
#pragma unroll
  for (int e = 0; e < E; e++) os[warp][lane * E + e] = acc[e];
  __syncthreads();
  for (int i = threadIdx.x; i < HD; i += 128) {
    const float mx = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
    float o = 0.0f, tot = 0.0f;
    for (int w = 0; w < 4; w++) {
      const float f = ms[w] == -INFINITY && ls[w] == 0.0f ? 0.0f : expf(ms[w] - mx);
      tot += f * ls[w];
      o += f * os[w][i];
    }
    out[((size_t)row * nh + h) * HD + i] = tot == 0.0f ? 0.0f : o / tot;
  }
}

}  // namespace hg

using namespace hg;

namespace {

void check_attn(const hg_kv8_cache* c, const hg_rows* r, int n_heads) {
  kv8_check_cache(c);
  kv8_check_rows(r, true);
  kv8_need(n_heads > 0 && n_heads % c->n_kv_heads == 0, "bad head counts");
  kv8_need(n_heads / c->n_kv_heads <= KV8_MAX_GROUP, "more than 32 q heads per kv head");
}

}  // namespace

extern "C" size_t hg_op_kv8_attn_scratch_bytes(const hg_kv8_cache* c, const hg_rows* r, int n_heads) {
  try {
    check_attn(c, r, n_heads);
    return 256;
  } catch (const std::exception&) {
    return 0;
  }
}

extern "C" int hg_op_kv8_attn(const hg_kv8_cache* c, const hg_rows* r, int n_heads, const float* q, float* out,
                              void* scratch, void* stream) {
  KV8_API({
    check_attn(c, r, n_heads);
    if (r->n_seqs == 0 || r->n_rows == 0) return HG_OK;
    kv8_need(q && out && scratch, "null argument");
    kv8_need(kv8_aligned(q, 16) && kv8_aligned(out, 16) && kv8_aligned(scratch, 16),
             "q, out and scratch must be 16-byte aligned");
    Kv8Device dev(c->pool);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const dim3 grid(r->n_rows, n_heads);
    if (c->head_dim == 64) k_kv8_attn<64><<<grid, 128, 0, st>>>(*c, *r, n_heads, q, out);
    else k_kv8_attn<128><<<grid, 128, 0, st>>>(*c, *r, n_heads, q, out);
    kv8_launched(cudaGetLastError());
  })
}
