// The 8-bit KV cache: rows are quantised as they are written (hg_op_kv8_append) and read back as f32
// (hg_op_kv8_read). Layout: hobbygpu.h (hg_kv8_cache).
//
// One scale per (slot, kv head): the attention folds a K scale into the score and a V scale into the
// probability, one multiplication each, where scales per 32 dims (the weights' format) would need four
// score accumulators and four sets of probabilities. 2 * (hd + 4) bytes a slot and head instead of 8 hd.
#include "hg_kv8.cuh"

namespace hg {

constexpr int KV8_WARPS = 8;   // most warps of an append CTA: three CTAs of them fit an SM's registers
constexpr int KV8_HEADS = 4;   // heads that a warp takes at a time
constexpr int KV8_STAGE_DIMS = 2048;  // most V dims (heads x head_dim) of a page that are staged
constexpr int KV8_PITCH = KV8_PAGE + 4;  // bytes of a staged V dim: 5 words, so that neighbouring dims spread over the banks

// round-half-even(v): adding 1.5 * 2^52 leaves the rounded integer in the low word of the sum.
__device__ __forceinline__ int kv8_round(double v) { return __double2loint(__dadd_rn(v, 6755399441055744.0)); }

// Scale of a row whose greatest magnitude is amax (any NaN or infinity: NaN), and 1 / scale. The
// quotient by 127 is amax * (1 / 127) and one correction.
__device__ __forceinline__ float kv8_scale(double amax, double* inv) {
  const double r = 1.0 / 127.0, q = __dmul_rn(amax, r);
  const float sc = amax <= 3.402823466385288598e38 ? (float)fma(fma(-127.0, q, amax), r, q) : __int_as_float(0x7fffffff);
  *inv = sc > 0.0f ? __drcp_rn((double)sc) : 0.0;  // a zero or NaN scale: codes 0
  return sc;
}

// The greatest magnitude of a row (an infinity or a NaN if it holds one): bit patterns of magnitudes are
// ordered, the upper words meet first.
template <int E>
__device__ __forceinline__ double row_max(const double (&y)[E]) {
  uint32_t hi = 0, lo = 0;
#pragma unroll
  for (int e = 0; e < E; e++) hi = max(hi, (uint32_t)__double2hiint(y[e]) & 0x7fffffffu);
  hi = __reduce_max_sync(0xffffffffu, hi);
#pragma unroll
  for (int e = 0; e < E; e++)
    if (((uint32_t)__double2hiint(y[e]) & 0x7fffffffu) == hi) lo = max(lo, (uint32_t)__double2loint(y[e]));
  return __hiloint2double((int)hi, (int)__reduce_max_sync(0xffffffffu, lo));
}
template <int E>
__device__ __forceinline__ double row_max(const float (&x)[E]) {  // NaN patterns lie above the infinities
  uint32_t a = 0;
#pragma unroll
  for (int e = 0; e < E; e++) a = max(a, __float_as_uint(x[e]) & 0x7fffffffu);
  return (double)__uint_as_float(__reduce_max_sync(0xffffffffu, a));
}

// the most that an append CTA takes: two tasks' rows per warp and a page's V codes
constexpr size_t KV8_APPEND_SMEM = (size_t)KV8_WARPS * 2 * KV8_HEADS * 128 * 4 + (size_t)KV8_STAGE_DIMS * KV8_PITCH;

// A head's row as a warp holds it: lane l has dims l H .. l H + H - 1 of each half (H = HD / 64), so a
// dim and its rotation partner are in the same lane.
template <int HD>
struct HeadRow {
  static constexpr int H = HD / 64;
  __device__ static __forceinline__ void load(const float* p, float (&x)[2 * H]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int half = 0; half < 2; half++) {
      if constexpr (H == 2) {
        const float2 v = *reinterpret_cast<const float2*>(p + half * (HD / 2) + lane * 2);
        x[half * 2] = v.x, x[half * 2 + 1] = v.y;
      } else {
        x[half] = p[half * (HD / 2) + lane];
      }
    }
  }
  __device__ static __forceinline__ void store(float* p, const float (&x)[2 * H]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int half = 0; half < 2; half++) {
      if constexpr (H == 2) *reinterpret_cast<float2*>(p + half * (HD / 2) + lane * 2) = make_float2(x[half * 2], x[half * 2 + 1]);
      else p[half * (HD / 2) + lane] = x[half];
    }
  }
  // dim of element e
  __device__ static __forceinline__ int dim(int e) { return (e / H) * (HD / 2) + (threadIdx.x & 31) * H + e % H; }
};

// The codes of `count` heads' rows y into slot w of a page: K as 2 H bytes per lane, V as bytes 16 apart
// or, staged, into shared memory. Lane g < count works out head g's scale and its inverse.
template <int HD, bool V, class T>
__device__ __forceinline__ void kv8_put(const T (&y)[KV8_HEADS][HD / 32], int count, uint8_t* blk, int w,
                                        uint8_t* stage) {
  constexpr int E = HD / 32, H = HD / 64;
  const int lane = threadIdx.x & 31;
  double amax = 0.0, inv;
#pragma unroll
  for (int g = 0; g < KV8_HEADS; g++) {
    const double a = row_max(y[g]);
    if ((lane & 3) == g) amax = a;
  }
  const float sc = kv8_scale(amax, &inv);
  if (lane < count) *reinterpret_cast<float*>(blk + lane * kv8_block_bytes(HD) + (V ? kv8_vs_off(HD, w) : kv8_ks_off(HD, w))) = sc;
  // only the rounding of a subnormal scale is coarse enough to leave a quotient above 127
  const bool tiny = __any_sync(0xffffffffu, sc < 1.17549435e-38f && sc > 0.0f);
  const bool odd = tiny || __any_sync(0xffffffffu, !(sc >= 0.0f));  // or a NaN among them
  const int i0 = HeadRow<HD>::dim(0);
  uint8_t* bk = blk + (V ? kv8_v_off(HD, w, i0) : kv8_k_off(HD, w, i0));
#pragma unroll
  for (int g = 0; g < KV8_HEADS; g++) {
    if (g >= count) break;
    uint8_t* to = bk + g * kv8_block_bytes(HD);
    int q[E];
    // y / scale, correctly rounded: the product with the rounded inverse is an ulp off at times, which moves
    // what lies half-way between two codes (Markstein's correction, "Computation of elementary functions on
    // the IBM RISC System/6000 processor", 1990). inv = 0: codes 0.
    auto quotients = [&]() {
      const double s = __shfl_sync(0xffffffffu, inv, g), sg = (double)__shfl_sync(0xffffffffu, sc, g), by = s > 0.0 ? sg : 0.0;
#pragma unroll
      for (int e = 0; e < E; e++) {
        const double v = (double)y[g][e], t = __dmul_rn(v, s);
        q[e] = kv8_round(fma(fma(-t, by, v), s, t));
      }
    };
    if constexpr (V) {
      // In f32 the quotient is off by 2 * 2^-24 * 127 < 1e-4 at most: the code is sure where it lies further
      // than that from half-way between two, which leaves one head's row in 40.
      const float s1 = __shfl_sync(0xffffffffu, (float)inv, g);
      const f32x2 s2 = pack2(s1, s1), up2 = pack2(12582912.0f, 12582912.0f), down2 = pack2(-12582912.0f, -12582912.0f);
      float off = 0.0f;
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        // + 1.5 * 2^23: the integer in the low bits
        const f32x2 t = mul2(pack2((float)y[g][e], (float)y[g][e + 1]), s2), r = add2(t, up2);
        float a, b;
        unpack2(r, a, b);
        q[e] = __float_as_int(a), q[e + 1] = __float_as_int(b);
        unpack2(fma2(add2(r, down2), pack2(-1.0f, -1.0f), t), a, b);
        off = fmaxf(off, fmaxf(fabsf(a), fabsf(b)));
      }
      if (odd || __any_sync(0xffffffffu, off > 0.4999f)) quotients();
    } else {
      quotients();
    }
    if (tiny) {
#pragma unroll
      for (int e = 0; e < E; e++) q[e] = min(max(q[e], -127), 127);
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int di = (e / H) * (HD / 2) + e % H;  // from the lane's first dim
      if constexpr (V) {
        if (stage) stage[(g * HD + i0 + di) * KV8_PITCH + w] = (uint8_t)q[e];
        else to[di * KV8_PAGE] = (uint8_t)q[e];
      } else if constexpr (H == 1) {
        to[di * 8] = (uint8_t)q[e];  // 16 dims on are 128 bytes on
      } else if (e % 2 == 0) {
        *reinterpret_cast<uint16_t*>(to + (e / H) * (HD / 2) * 8) = (uint16_t)((q[e] & 255) | (q[e + 1] & 255) << 8);
      }
    }
  }
}

// One CTA per (page, sequence); its warps take the page's rows in groups of up to four heads, whose
// loads are in flight together and whose sums, roots and divisions share the lanes (lane g finishes head
// g). k runs in f64: a code sits at a rounding border of its row's scale, and f32 sums in another order
// would move codes by one. The next task's rows come by asynchronous copies meanwhile. The V codes of a
// full page are turned round in shared memory, so that they leave as 16-byte columns; a page that the call
// fills in part gets its bytes one by one. 21,000 rows of 16 q and 8 kv heads of 128 dims take 110 us, 560
// MB, 0.78 of measured HBM: issue slots are 72% busy, most of it with the f64 work on k and the codes.
template <int HD>
__global__ void __launch_bounds__(32 * KV8_WARPS, 3) k_kv8_append(const __grid_constant__ hg_kv8_cache C,
                                                              const __grid_constant__ hg_rows R,
                                                              const __grid_constant__ hg_kv8_append_args A) {
  constexpr int E = HD / 32, H = HD / 64;
  extern __shared__ __align__(16) float rows_s[];  // per warp, two tasks' rows: [warp][2][KV8_HEADS * HD]; the staged V
  __shared__ int pos_s[KV8_PAGE];  // position of the page's row in slot w; -1: dropped or padding
  pdl_wait();
  pdl_trigger();
  const int s = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const SeqSpan sp = kv8_span(R, s, true);
  const long long base = ((long long)(sp.start / KV8_PAGE) + blockIdx.x) * KV8_PAGE;  // the page's first slot
  const int j0 = (int)max(0ll, base - sp.start);
  const int nr = (int)min((long long)sp.n, base + KV8_PAGE - sp.start) - j0;
  if (nr <= 0) return;
  const int w0 = (int)(sp.start + (long long)j0 - base);
  const int nh = A.n_heads, nkv = C.n_kv_heads, heads = nh + 2 * nkv;
  const int qg = A.q_out ? (nh + KV8_HEADS - 1) / KV8_HEADS : 0, kg = (nkv + KV8_HEADS - 1) / KV8_HEADS;
  const float* rows = A.qkv + ((size_t)sp.r0 + j0) * heads * HD;  // of the page: at most 16, fewer than 2^31 floats
  float* mine = rows_s + warp * 2 * KV8_HEADS * HD;
  // a task: row r's heads h0 .. h0 + count - 1 of q, k or v (kind 0, 1, 2)
  struct Task {
    int group, r, kind, h0, count;
    const float* src;
  };
  auto place = [&](Task& k) {
    while (k.r >= nr) k.r -= nr, k.group++;
    const int first = k.group < qg ? 0 : k.group < qg + kg ? qg : qg + kg;
    k.kind = k.group < qg ? 0 : k.group < qg + kg ? 1 : 2;
    k.h0 = (k.group - first) * KV8_HEADS;
    k.count = min(KV8_HEADS, (k.kind == 0 ? nh : nkv) - k.h0);
    k.src = rows + (k.r * heads + (k.kind == 0 ? 0 : k.kind == 1 ? nh : nh + nkv) + k.h0) * HD;
  };
  // its rows on their way into shared memory while the task before is worked on
  auto fetch = [&](const Task& k, float* dst) {
    if (k.group < qg + 2 * kg) {
      const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst + lane * 4);
      const float* src = k.src + lane * 4;
#pragma unroll
      for (int i = 0; i < KV8_HEADS * HD / 128; i++)
        if ((i * 32 + lane) * 4 < k.count * HD)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d + i * 512), "l"(src + i * 128) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  Task next{0, warp, 0, 0, 0, nullptr};
  place(next);
  fetch(next, mine);
  uint8_t* page = kv8_block(C, s, base, 0);
  auto put_pos = [&](int r, long long pos) {
    if (pos >= 0 && (pos >= A.max_pos || !page)) {
      kv8_flag(R.err, HG_ERR_CONTEXT);
      pos = -1;
    }
    pos_s[r] = (int)pos;
  };
  if (!R.parent) {
    if (threadIdx.x < nr) put_pos(threadIdx.x, (long long)sp.start + j0 + threadIdx.x);
  } else {
    for (int r = threadIdx.x >> 4; r < nr; r += blockDim.x >> 4) {  // half a warp a row
      int depth = -1;  // a padding ancestor ends the path
      for (int at = j0 + r; at >= 0;) {
        const PathRun run = kv8_run<16>(R, sp, at);
        depth += run.len;
        at = run.next;
      }
      if ((lane & 15) == 0) put_pos(r, depth < 0 ? -1 : (long long)sp.start + depth);
    }
  }
  __syncthreads();
  uint8_t* v_stage = reinterpret_cast<uint8_t*>(rows_s + warps * 2 * KV8_HEADS * HD);
  bool staged = nr == KV8_PAGE && nkv * HD <= KV8_STAGE_DIMS;
  for (int r = 0; staged && r < nr; r++) staged = pos_s[r] >= 0;
  for (int odd = 0; next.group < qg + 2 * kg; odd ^= 1) {
    const Task k = next;
    next.r += warps;
    place(next);
    fetch(next, mine + (odd ^ 1) * KV8_HEADS * HD);
    const int kind = k.kind, h0 = k.h0, count = k.count, w = w0 + k.r, pos = pos_s[k.r];
    const size_t row = (size_t)sp.r0 + j0 + k.r;
    if (pos < 0) {
      if (kind == 0) {
        const float zero[E] = {};
        for (int g = 0; g < count; g++) HeadRow<HD>::store(A.q_out + (row * nh + h0 + g) * HD, zero);
      }
      // The next fetch writes where this row's copies go, and copies of two groups land in any order: they
      // are waited for although nobody reads them (a lane's copies always go to the same places).
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      continue;
    }
    float gain[E], c[H], sn[H];
    if (kind != 2) {
      const float* g = kind == 0 ? A.q_norm : A.k_norm;
#pragma unroll
      for (int e = 0; e < E; e++) gain[e] = g[HeadRow<HD>::dim(e)];
      const float *cp = A.rope_cos + (size_t)pos * (HD / 2) + lane * H, *np = A.rope_sin + (size_t)pos * (HD / 2) + lane * H;
#pragma unroll
      for (int e = 0; e < H; e++) c[e] = cp[e], sn[e] = np[e];
    }
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    float x[KV8_HEADS][E];
#pragma unroll
    for (int g = 0; g < KV8_HEADS; g++)
      HeadRow<HD>::load(mine + odd * KV8_HEADS * HD + min(g, count - 1) * HD, x[g]);
    __syncwarp();  // read before the next fetch fills this half
    uint8_t* blk = page + (long long)h0 * kv8_block_bytes(HD);
    if (kind == 2) {
      kv8_put<HD, true>(x, count, blk, w, staged ? v_stage + (size_t)h0 * HD * KV8_PITCH : nullptr);
      continue;
    }
    if (kind == 0) {
      float ss[KV8_HEADS];
#pragma unroll
      for (int g = 0; g < KV8_HEADS; g++) {
        ss[g] = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) ss[g] = __fmaf_rn(x[g][e], x[g][e], ss[g]);
      }
      const float rs = rsqrtf(warp_sums(ss) * (1.0f / HD) + A.eps);  // head lane % 4; 2 ulp
#pragma unroll
      for (int g = 0; g < KV8_HEADS; g++) {
        if (g >= count) break;
        const float f = __shfl_sync(0xffffffffu, rs, g);
        float y[E];
#pragma unroll
        for (int e = 0; e < H; e++) {
          const float a = x[g][e] * f * gain[e], b = x[g][H + e] * f * gain[H + e];
          y[e] = __fmaf_rn(a, c[e], -(b * sn[e]));
          y[H + e] = __fmaf_rn(b, c[e], a * sn[e]);
        }
        HeadRow<HD>::store(A.q_out + (row * nh + h0 + g) * HD, y);
      }
    } else {
      double y[KV8_HEADS][E], ss[KV8_HEADS];
#pragma unroll
      for (int g = 0; g < KV8_HEADS; g++) {
        ss[g] = 0.0;
#pragma unroll
        for (int e = 0; e < E; e++) {
          y[g][e] = (double)x[g][e];
          ss[g] = fma(y[g][e], y[g][e], ss[g]);
        }
      }
      const double rs = rsqrt(warp_sums(ss) * (1.0 / HD) + (double)A.eps);
#pragma unroll
      for (int g = 0; g < KV8_HEADS; g++) {
        const double f = __shfl_sync(0xffffffffu, rs, g);
#pragma unroll
        for (int e = 0; e < H; e++) {
          const double a = y[g][e] * f * (double)gain[e], b = y[g][H + e] * f * (double)gain[H + e];
          y[g][e] = fma(a, (double)c[e], -(b * (double)sn[e]));
          y[g][H + e] = fma(b, (double)c[e], a * (double)sn[e]);
        }
      }
      kv8_put<HD, false>(y, count, blk, w, nullptr);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (!staged) return;
  __syncthreads();
  for (int t = threadIdx.x; t < nkv * HD; t += blockDim.x) {
    const uint32_t* v = reinterpret_cast<const uint32_t*>(v_stage + (size_t)t * KV8_PITCH);
    *reinterpret_cast<uint4*>(page + (long long)(t / HD) * kv8_block_bytes(HD) + kv8_v_off(HD, 0, t % HD)) =
        make_uint4(v[0], v[1], v[2], v[3]);
  }
}

// One CTA per `pages` neighbouring pages of a sequence for K and one for V, its work the pages' (page,
// head) blocks. K: a thread turns four neighbouring codes of a slot into a float4. V: a thread loads one
// dim's 16 slots; four neighbouring threads exchange their words, so that each holds four slots of four
// dims and writes a float4 to each. Bound by the f32 rows it writes; the codes come from the L2 cache, for
// which a CTA's pages are asked for at its start. 129,000 rows of 3 heads of 128 dims each way: 83 us, 0.91
// of measured HBM (two or eight pages a CTA: 91 and 92).
constexpr int KV8_READ = 4;        // blocks of a thread in flight
constexpr int KV8_READ_PAGES = 4;  // most pages of a CTA

__device__ __forceinline__ float4 kv8_values(uint32_t codes, float sc) {
  return make_float4((float)(int8_t)codes * sc, (float)(int8_t)(codes >> 8) * sc, (float)(int8_t)(codes >> 16) * sc,
                     (float)(int8_t)(codes >> 24) * sc);
}

template <int HD>
__global__ void __launch_bounds__(256) k_kv8_read(const __grid_constant__ hg_kv8_cache C,
                                                  const __grid_constant__ hg_rows R, float* __restrict__ ko,
                                                  float* __restrict__ vo, int pages, int kinds) {
  __shared__ const uint8_t* page_s[KV8_READ_PAGES];
  pdl_wait();
  pdl_trigger();
  // K's and V's CTA of the same pages side by side (kinds = 2), so that they meet in the L2 cache
  const int s = blockIdx.y, tid = threadIdx.x, nkv = C.n_kv_heads, chunk = blockIdx.x / kinds, kind = blockIdx.x % kinds;
  const SeqSpan sp = kv8_span(R, s, true);
  // the CTA's slots: base .. base + 16 pages - 1, of which its rows j0 .. j0 + nr - 1
  const long long base = ((long long)(sp.start / KV8_PAGE) + (long long)chunk * pages) * KV8_PAGE;
  const int j0 = (int)max(0ll, base - sp.start);
  const int nr = (int)min((long long)sp.n, base + pages * KV8_PAGE - sp.start) - j0;
  if (nr <= 0) return;
  const int w0 = (int)(sp.start + (long long)j0 - base), used = (w0 + nr + KV8_PAGE - 1) / KV8_PAGE;
  if (tid < used) {
    page_s[tid] = kv8_block(C, s, base + tid * KV8_PAGE, 0);
    if (!page_s[tid]) kv8_flag(R.err, HG_ERR_CONTEXT);
    else if (pages > 1 && kind == 0)
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(page_s[tid]), "r"(nkv * kv8_block_bytes(HD)) : "memory");
  }
  __syncthreads();
  const size_t rs = (size_t)nkv * HD;
  const int blocks = used * nkv;
  const uint32_t inv = nkv == 1 ? 0u : 0xffffffffu / nkv + 1;  // q / nkv = high word of q * inv: q * nkv < 2^32
  auto page_of = [&](int q) { return nkv == 1 ? q : (int)__umulhi(q, inv); };
  if (ko && kind == 0) {
    constexpr int T = HD / 4, RT = HD / 64;  // threads of a row; rows of a block per thread, eight apart
    const int i = tid % T * 4, wa = tid / T;
    float* out = ko + ((size_t)sp.r0 + j0) * rs + i;
    for (int q0 = 0; q0 < blocks; q0 += KV8_READ) {
      uint32_t c[KV8_READ][RT];
      float sc[KV8_READ][RT];
#pragma unroll
      for (int u = 0; u < KV8_READ; u++) {
        const int q = min(q0 + u, blocks - 1), g = page_of(q);
        const uint8_t *page = page_s[g], *blk = page + (long long)(q - g * nkv) * kv8_block_bytes(HD);
#pragma unroll
        for (int r = 0; r < RT; r++) {
          c[u][r] = page ? *reinterpret_cast<const uint32_t*>(blk + kv8_k_off(HD, wa + 8 * r, i)) : 0u;
          sc[u][r] = page ? *reinterpret_cast<const float*>(blk + kv8_ks_off(HD, wa + 8 * r)) : 0.0f;
        }
      }
#pragma unroll
      for (int u = 0; u < KV8_READ; u++) {
        const int q = q0 + u, g = page_of(q);
        if (q >= blocks) break;
#pragma unroll
        for (int r = 0; r < RT; r++) {
          const int row = g * KV8_PAGE + wa + 8 * r - w0;  // of the CTA's rows
          if (row >= 0 && row < nr)
            *reinterpret_cast<float4*>(out + (size_t)row * rs + (q - g * nkv) * HD) = kv8_values(c[u][r], sc[u][r]);
        }
      }
    }
  }
  if (vo && kind == kinds - 1) {
    constexpr int B = 256 / HD;  // blocks at once
    const int i = tid % HD, a = tid & 3;
    float* out = vo + ((size_t)sp.r0 + j0) * rs + (i & ~3);
    for (int q0 = 0; q0 < blocks; q0 += B * KV8_READ) {  // whole warps: the exchange needs every lane
      uint4 c[KV8_READ];
      float4 sc[KV8_READ];
#pragma unroll
      for (int u = 0; u < KV8_READ; u++) {
        const int q = min(q0 + u * B + tid / HD, blocks - 1), g = page_of(q);
        const uint8_t *page = page_s[g], *blk = page + (long long)(q - g * nkv) * kv8_block_bytes(HD);
        c[u] = page ? *reinterpret_cast<const uint4*>(blk + kv8_v_off(HD, 0, i)) : make_uint4(0, 0, 0, 0);
        sc[u] = page ? *reinterpret_cast<const float4*>(blk + kv8_vs_off(HD, 4 * a)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
#pragma unroll
      for (int u = 0; u < KV8_READ; u++) {
        const int q = q0 + u * B + tid / HD, g = page_of(q);
        // word b (slots 4 b .. 4 b + 3) of thread a to word a of thread b
        uint32_t w[4] = {c[u].x, c[u].y, c[u].z, c[u].w};
#pragma unroll
        for (int step = 1; step <= 2; step *= 2) {
#pragma unroll
          for (int p = 0; p < 2; p++) {
            const int lo = step == 1 ? 2 * p : p, hi = lo + step;
            const uint32_t got = __shfl_xor_sync(0xffffffffu, a & step ? w[lo] : w[hi], step);
            if (a & step) w[lo] = got;
            else w[hi] = got;
          }
        }
        const float s4[4] = {sc[u].x, sc[u].y, sc[u].z, sc[u].w};
        const int row0 = g * KV8_PAGE + 4 * a - w0;
        float* dst = out + (long long)row0 * (long long)rs + (q - g * nkv) * HD;
#pragma unroll
        for (int e = 0; e < 4; e++) {
          // slot e's byte of the four dims
          const uint32_t lo = __byte_perm(w[0], w[1], e | (4 + e) << 4), hi = __byte_perm(w[2], w[3], e | (4 + e) << 4);
          if (q < blocks && row0 + e >= 0 && row0 + e < nr)
            *reinterpret_cast<float4*>(dst) = kv8_values(__byte_perm(lo, hi, 0x5410), s4[e]);
          dst += rs;
        }
      }
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
    // a warp per group of heads of the rows that a page can get
    const int groups = (a->n_heads + KV8_HEADS - 1) / KV8_HEADS + 2 * ((c->n_kv_heads + KV8_HEADS - 1) / KV8_HEADS);
    const int warps = min((long long)KV8_WARPS, (long long)min(rows, KV8_PAGE) * groups);
    const int dims = c->n_kv_heads * c->head_dim;
    const size_t smem = (size_t)warps * 2 * KV8_HEADS * c->head_dim * 4 +
                        (rows >= KV8_PAGE && dims <= KV8_STAGE_DIMS ? (size_t)dims * KV8_PITCH : 0);
    auto kern = c->head_dim == 64 ? k_kv8_append<64> : k_kv8_append<128>;
    kv8_smem_limit(kern, dev.device, KV8_APPEND_SMEM);
    kv8_launch_pdl(kern, grid, 32 * warps, smem, stream, *c, *r, *a);
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
    const int most = (rows + KV8_PAGE - 2) / KV8_PAGE + 1;  // pages that a sequence's rows can touch
    // four pages a CTA once that leaves every SM several, else one
    const int pages = (long long)most * r->n_seqs >= 148 * 4 * KV8_READ_PAGES ? KV8_READ_PAGES : 1;
    const int kinds = k_out && v_out ? 2 : 1;
    const dim3 grid((most + pages - 1) / pages * kinds, r->n_seqs);
    kv8_launch_pdl(c->head_dim == 64 ? k_kv8_read<64> : k_kv8_read<128>, grid, 256, 0, stream, *c, *r, k_out, v_out, pages, kinds);
  })
}
