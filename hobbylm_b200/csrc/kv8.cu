// The 8-bit KV cache: rows are quantised as they are written (hg_op_kv8_append) and read back as f32
// (hg_op_kv8_read). Layout: hobbygpu.h (hg_kv8_cache).
//
// One scale per (slot, kv head): the attention folds a K scale into the score and a V scale into the
// probability, one multiplication each, where scales per 32 dims (the weights' format) would need four
// score accumulators and four sets of probabilities. 2 * (hd + 4) bytes a slot and head instead of 8 hd.
#include "hg_kv8.cuh"

namespace hg {

constexpr int KV8_WARPS = 16;

// round-half-even(y * inv) clamped to the codes: adding 1.5 * 2^52 leaves the rounded integer in the
// low word of the sum.
__device__ __forceinline__ int kv8_code(double y, double inv) {
  const int q = __double2loint(__dadd_rn(__dmul_rn(y, inv), 6755399441055744.0));
  return min(max(q, -127), 127);
}

// Scale of a row whose greatest magnitude is amax (any NaN or infinity: NaN), and 1 / scale.
__device__ __forceinline__ float kv8_scale(double amax, double* inv) {
  const float sc = amax <= 3.402823466385288598e38 ? (float)(amax / 127.0) : __int_as_float(0x7fffffff);
  *inv = sc > 0.0f ? 1.0 / (double)sc : 0.0;  // a zero or NaN scale: codes 0
  return sc;
}

// Greatest of the lanes' non-negative doubles (NaN greatest of all): their bit patterns are ordered.
__device__ __forceinline__ double warp_max_abs(double v) {
  const uint32_t hi = (uint32_t)__double2hiint(v), lo = (uint32_t)__double2loint(v);
  const uint32_t mh = __reduce_max_sync(0xffffffffu, hi);
  const uint32_t ml = __reduce_max_sync(0xffffffffu, hi == mh ? lo : 0u);
  return __hiloint2double((int)mh, (int)ml);
}

// One CTA per (page, sequence); its warps take the (row, head) pairs of the rows that the page holds.
// A lane owns HD / 32 neighbouring dims, so loads, q rows and K codes move as whole words, and the
// rotation's partner dim is 16 lanes away. The norm, rotation and quantisation of k run in f64: a code
// sits at a rounding border of its row's scale, and f32 sums in another order would move codes by one.
template <int HD>
__global__ void __launch_bounds__(32 * KV8_WARPS) k_kv8_append(hg_kv8_cache C, hg_rows R, hg_kv8_append_args A) {
  constexpr int E = HD / 32;
  const int s = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ int pos_s[KV8_PAGE];  // position of the page's row in slot w; -1: dropped or padding
  const SeqSpan sp = kv8_span(R, s, true);
  const long long base = ((long long)(sp.start / KV8_PAGE) + blockIdx.x) * KV8_PAGE;  // the page's first slot
  const int j0 = (int)max(0ll, base - sp.start);
  const int nr = (int)min((long long)sp.n, base + KV8_PAGE - sp.start) - j0;
  if (nr <= 0) return;
  const int w0 = (int)(sp.start + (long long)j0 - base);
  const uint8_t* page = kv8_block(C, s, base, 0);
  if (threadIdx.x < nr) {
    const int j = j0 + threadIdx.x;
    long long pos = (long long)sp.start + j;
    int up = kv8_parent(R, sp, j);
    if (R.parent) {
      if (up == -2) {
        pos = -1;
      } else {
        pos = sp.start;
        while (up >= 0) {  // strictly down: at most j steps; a padding ancestor ends the path
          const int q = kv8_parent(R, sp, up);
          if (q == -2) break;
          pos++;
          up = q;
        }
      }
    }
    if (pos >= 0 && (pos >= A.max_pos || !page)) {
      kv8_flag(R.err, HG_ERR_CONTEXT);
      pos = -1;
    }
    pos_s[threadIdx.x] = (int)pos;
  }
  __syncthreads();
  const int nh = A.n_heads, nkv = C.n_kv_heads, heads = nh + 2 * nkv;
  for (int t = warp; t < nr * heads; t += KV8_WARPS) {
    const int r = t / heads, h = t - r * heads, w = w0 + r, row = sp.r0 + j0 + r, pos = pos_s[r];
    const float* src = A.qkv + ((size_t)row * heads + h) * HD + lane * E;
    float x[E];
    if (E == 4) {
      const float4 v = *reinterpret_cast<const float4*>(src);
      x[0] = v.x, x[1] = v.y, x[E - 2] = v.z, x[E - 1] = v.w;
    } else {
      const float2 v = *reinterpret_cast<const float2*>(src);
      x[0] = v.x, x[1] = v.y;
    }
    if (h < nh) {
      if (!A.q_out) continue;
      float* dst = A.q_out + ((size_t)row * nh + h) * HD + lane * E;
      float y[E];
      if (pos < 0) {
#pragma unroll
        for (int e = 0; e < E; e++) y[e] = 0.0f;
      } else {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) ss = __fmaf_rn(x[e], x[e], ss);
        const float rs = __fdiv_rn(1.0f, __fsqrt_rn(warp_sum(ss) / HD + A.eps));
#pragma unroll
        for (int e = 0; e < E; e++) {
          const int i = lane * E + e, ci = i & (HD / 2 - 1);
          const float n = x[e] * rs * A.q_norm[i], o = __shfl_xor_sync(0xffffffffu, n, 16);
          const float c = A.rope_cos[(size_t)pos * (HD / 2) + ci], sn = A.rope_sin[(size_t)pos * (HD / 2) + ci];
          y[e] = lane < 16 ? n * c - o * sn : n * c + o * sn;
        }
      }
      if (E == 4) *reinterpret_cast<float4*>(dst) = make_float4(y[0], y[1], y[E - 2], y[E - 1]);
      else *reinterpret_cast<float2*>(dst) = make_float2(y[0], y[1]);
      continue;
    }
    if (pos < 0) continue;
    const bool is_v = h >= nh + nkv;
    const int kvh = h - nh - (is_v ? nkv : 0);
    uint8_t* blk = const_cast<uint8_t*>(page) + (long long)kvh * kv8_block_bytes(HD);
    double y[E], amax = 0.0, inv;
    if (is_v) {
#pragma unroll
      for (int e = 0; e < E; e++) y[e] = (double)x[e];
    } else {
      double ss = 0.0;
#pragma unroll
      for (int e = 0; e < E; e++) ss = fma((double)x[e], (double)x[e], ss);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const double rs = 1.0 / sqrt(ss / HD + (double)A.eps);
#pragma unroll
      for (int e = 0; e < E; e++) {
        const int i = lane * E + e, ci = i & (HD / 2 - 1);
        const double n = (double)x[e] * rs * (double)A.k_norm[i], o = __shfl_xor_sync(0xffffffffu, n, 16);
        const double c = (double)A.rope_cos[(size_t)pos * (HD / 2) + ci];
        const double sn = (double)A.rope_sin[(size_t)pos * (HD / 2) + ci];
        y[e] = lane < 16 ? n * c - o * sn : n * c + o * sn;
      }
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
      const double m = fabs(y[e]);
      amax = (m > amax || m != m) ? m : amax;  // a NaN stays
    }
    const float sc = kv8_scale(warp_max_abs(amax), &inv);
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < E; e++) word |= (uint32_t)(inv > 0.0 ? kv8_code(y[e], inv) & 255 : 0) << (8 * e);
    if (is_v) {
#pragma unroll
      for (int e = 0; e < E; e++) blk[kv8_v_off(HD, w, lane * E + e)] = (uint8_t)(word >> (8 * e));
      if (lane == 0) *reinterpret_cast<float*>(blk + kv8_vs_off(HD, w)) = sc;
    } else {
      uint8_t* d = blk + kv8_k_off(HD, w, lane * E);
      if (E == 4) *reinterpret_cast<uint32_t*>(d) = word;
      else *reinterpret_cast<uint16_t*>(d) = (uint16_t)word;
      if (lane == 0) *reinterpret_cast<float*>(blk + kv8_ks_off(HD, w)) = sc;
    }
  }
}

// One CTA per (page, sequence). K: a thread turns four neighbouring codes of one slot into a float4.
// V: a thread holds one dim's 16 slots (one 16-byte load) and writes a float to each row; neighbouring
// threads hold neighbouring dims, so both write whole lines.
template <int HD>
__global__ void __launch_bounds__(256) k_kv8_read(hg_kv8_cache C, hg_rows R, float* __restrict__ ko,
                                                  float* __restrict__ vo) {
  const int s = blockIdx.y, tid = threadIdx.x, nkv = C.n_kv_heads;
  const SeqSpan sp = kv8_span(R, s, true);
  const long long base = ((long long)(sp.start / KV8_PAGE) + blockIdx.x) * KV8_PAGE;
  const int j0 = (int)max(0ll, base - sp.start);
  const int nr = (int)min((long long)sp.n, base + KV8_PAGE - sp.start) - j0;
  if (nr <= 0) return;
  const int w0 = (int)(sp.start + (long long)j0 - base);
  const uint8_t* page = kv8_block(C, s, base, 0);
  if (!page && tid == 0) kv8_flag(R.err, HG_ERR_CONTEXT);
  const size_t row0 = (size_t)sp.r0 + j0, rs = (size_t)nkv * HD;
  if (ko) {
    for (int t = tid; t < nr * nkv * (HD / 4); t += blockDim.x) {
      const int i = (t % (HD / 4)) * 4, kvh = (t / (HD / 4)) % nkv, r = t / (HD / 4) / nkv, w = w0 + r;
      float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (page) {
        const uint8_t* blk = page + (long long)kvh * kv8_block_bytes(HD);
        const char4 c = *reinterpret_cast<const char4*>(blk + kv8_k_off(HD, w, i));
        const float sc = *reinterpret_cast<const float*>(blk + kv8_ks_off(HD, w));
        y = make_float4(c.x * sc, c.y * sc, c.z * sc, c.w * sc);
      }
      *reinterpret_cast<float4*>(ko + (row0 + r) * rs + kvh * HD + i) = y;
    }
  }
  if (vo) {
    for (int t = tid; t < nkv * HD; t += blockDim.x) {
      const int i = t % HD, kvh = t / HD;
      alignas(16) signed char c[16] = {};
      float sc[16] = {};
      if (page) {
        const uint8_t* blk = page + (long long)kvh * kv8_block_bytes(HD);
        *reinterpret_cast<int4*>(c) = *reinterpret_cast<const int4*>(blk + kv8_v_off(HD, 0, i));
#pragma unroll
        for (int q = 0; q < 4; q++)
          *reinterpret_cast<float4*>(sc + 4 * q) = *reinterpret_cast<const float4*>(blk + kv8_vs_off(HD, 4 * q));
      }
#pragma unroll
      for (int w = 0; w < 16; w++)
        if (w >= w0 && w < w0 + nr) vo[(row0 + w - w0) * rs + t] = c[w] * sc[w];
    }
  }
}

}  // namespace hg

using namespace hg;

extern "C" int64_t hg_kv8_block_bytes(int head_dim) {
  return head_dim == 64 || head_dim == 128 ? kv8_block_bytes(head_dim) : 0;
}

extern "C" int hg_op_kv8_append(const hg_kv8_cache* c, const hg_rows* r, const hg_kv8_append_args* a, void* stream) {
  KV8_API({
    kv8_check_cache(c);
    kv8_check_rows(r, true);
    kv8_need(a, "null argument");
    kv8_need(a->n_heads > 0 && a->n_heads <= 32768 && a->n_heads % c->n_kv_heads == 0, "bad head counts");
    kv8_need(a->max_pos > 0, "max_pos must be positive");
    kv8_need(a->qkv && a->q_norm && a->k_norm && a->rope_cos && a->rope_sin, "null argument");
    kv8_need(kv8_aligned(a->qkv, 16) && kv8_aligned(a->q_out, 16), "qkv and q_out must be 16-byte aligned");
    kv8_need(kv8_aligned(a->q_norm, 4) && kv8_aligned(a->k_norm, 4) && kv8_aligned(a->rope_cos, 4) &&
                 kv8_aligned(a->rope_sin, 4),
             "gains and RoPE tables must be 4-byte aligned");
    if (r->n_seqs == 0 || r->n_rows == 0) return HG_OK;
    Kv8Device dev(c->pool);
    const int rows = min(r->max_rows, r->n_rows);
    const dim3 grid((rows + KV8_PAGE - 2) / KV8_PAGE + 1, r->n_seqs);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (c->head_dim == 64) k_kv8_append<64><<<grid, 32 * KV8_WARPS, 0, st>>>(*c, *r, *a);
    else k_kv8_append<128><<<grid, 32 * KV8_WARPS, 0, st>>>(*c, *r, *a);
    kv8_launched(cudaGetLastError());
  })
}

extern "C" int hg_op_kv8_read(const hg_kv8_cache* c, const hg_rows* r, float* k_out, float* v_out, void* stream) {
  KV8_API({
    kv8_check_cache(c);
    kv8_check_rows(r, true);
    kv8_need(k_out || v_out, "null argument");
    kv8_need(kv8_aligned(k_out, 16) && kv8_aligned(v_out, 16), "k_out and v_out must be 16-byte aligned");
    if (r->n_seqs == 0 || r->n_rows == 0) return HG_OK;
    Kv8Device dev(c->pool);
    const int rows = min(r->max_rows, r->n_rows);
    const dim3 grid((rows + KV8_PAGE - 2) / KV8_PAGE + 1, r->n_seqs);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (c->head_dim == 64) k_kv8_read<64><<<grid, 256, 0, st>>>(*c, *r, k_out, v_out);
    else k_kv8_read<128><<<grid, 256, 0, st>>>(*c, *r, k_out, v_out);
    kv8_launched(cudaGetLastError());
  })
}
