// Attention of chains and drafted trees over the 8-bit KV cache (hg_op_kv8_attn).
//
// For a row's q head and the slots t that it sees: p_t = exp(q . k_t / sqrt(hd) - m), out =
// sum p_t v_t / sum p_t, with k_t = ks_t K_t and v_t = vs_t V_t, K and V int8 codes. Both contractions
// are integer: q and p_t vs_t are written in fixed point as three signed base-256 digits, so the
// tensor cores (tcgen05.mma kind::i8) multiply the cache's bytes as they lie in HBM, exactly, and only
// the rounding to 23 fraction bits of q and of the probabilities (2^-24 of the greatest, what f32
// rounding costs) and the f32 sums across tiles remain. No code is converted, no K or V value is formed.
//
// A tile is 128 slots (8 pages) of one kv head, and the slots are the MMA's M:
//   S[slot][digit * R + r] = sum_i K[slot][i] qdigit[r][i]           (A = K pages, B = q digits)
//   O[dim][digit * R + r]  = sum_slot V[dim][slot] pdigit[r][slot]   (A = V pages, stored [dim][slot])
// for R = up to 32 rows (q heads of the group x nodes of the tree) at a time. The accumulators come
// back from tensor memory with one slot (S) or one dim (O) per thread, so the softmax needs one
// maximum across the CTA per tile and row, and the digits of the probabilities go to shared memory as
// bytes. The running maximum, sum and output rows stay in registers from tile to tile.
//
// Work split: all tiles of all (sequence, kv head, row block) units lie on one line that is cut into
// equal runs, one per resident CTA, whatever the lengths; a unit that is cut is joined by
// k_kv8_join from at most two partial results per CTA, in tile order (no atomics).
//
// A copy warp keeps the stages of a ring full: per page 16 hd bytes of K, as many of V and 128 of
// scales, three bulk copies that need no rearranging (hg_kv8.cuh). Every mbarrier wait is bounded; when
// one gives up, the CTA reports HG_ERR_TIMEOUT, waits for nothing more but its copies and MMAs
// (bounded again), frees its tensor memory and returns.
#include <algorithm>
#include <atomic>

#include "hg_kv8.cuh"
#include "hg_tc.cuh"

namespace hg {

constexpr int KA_TILE = 128;                      // slots of a tile: the MMA's M
constexpr int KA_PAGES = KA_TILE / KV8_PAGE;      // pages of a tile
constexpr int KA_COMPUTE = 128;                   // threads that hold a slot (S) or a dim (O)
constexpr int KA_THREADS = KA_COMPUTE + 32;       // and the copy warp
constexpr int KA_SMS = 148;
constexpr int KA_MAX_CTAS = 3 * KA_SMS;
constexpr float KA_FIX = 8323072.0f;              // 2^23 - 2^16: the greatest fixed-point value, three digits

// Shared memory of one CTA, in order: the ring, the digits of q and of the probabilities, small arrays.
template <int HD, int R>
struct KaShape {
  static constexpr int N = (3 * R + 15) / 16 * 16;  // MMA N: digit columns
  static constexpr int NB = (3 * R + 7) / 8 * 8;    // digit rows kept (what N reads past them stays unread)
  static constexpr int KBYTES = KA_TILE * HD, STAGE = 2 * KBYTES + KA_PAGES * 128;
  static constexpr int STAGES = HD == 128 ? 2 : 4;
  static constexpr int OFF_BQ = STAGES * STAGE, OFF_BP = OFF_BQ + NB * HD, OFF_SMALL = OFF_BP + NB * KA_TILE;
  // tensor-memory columns: S at 0, O behind it; a power of two of at least 32
  static constexpr int COL_O = N <= 16 ? 16 : N <= 32 ? 32 : N <= 64 ? 64 : 128;
  static constexpr int COLS = 2 * COL_O;
  static constexpr int RC = R < 16 ? R : 16;  // rows per tensor-memory read
};

template <int R>
struct KaSmall {
  uint64_t full[4], empty[4], sbar, obar;
  float wmax[R][4];          // per warp maxima of a tile's scores
  float wsum[R][4];          // per warp sums at a unit's end
  float qs[R];               // row r: log2(e) / sqrt(hd) * q scale
  int lim[R];                // row r sees the slots below, and the tree slots of `vis`
  uint32_t vis[R][4];        // slots of the current tile that row r's path holds
  float wsv[4];
  uint32_t pages[4];         // per stage: which of the tile's pages are there
  uint32_t tmem;
  int fail;
};

struct KaArgs {
  hg_kv8_cache C;
  hg_rows R;
  int nh, g, npb;  // q heads, q heads per kv head, nodes per row block
  const float* q;
  float* out;
  float* part;     // [CTA][2][R * (hd + 2)] partial results: rows of hd sums, then maxima, then sums of p
  int4* head;      // [CTA][2] of the joins: {sequence, kv head * 65536.. (see k_kv8_join)}
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float warp_fmax(float v) {  // NaN only if every lane's is
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ void bar_compute() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void mbar_arrive_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
// The three base-256 digits of a rounded sum, exact in f32 each, put together with one rounding each.
__device__ __forceinline__ float digits(uint32_t d0, uint32_t d1, uint32_t d2) {
  return __fmaf_rn(tc_isum(d2), 65536.0f, __fmaf_rn(tc_isum(d1), 256.0f, tc_isum(d0)));
}
// Fixed point v (|v| <= KA_FIX) as signed digits v = b0 + 256 b1 + 65536 b2, one per byte.
__device__ __forceinline__ uint32_t to_digits(uint32_t v) { return (v + 0x808080u) ^ 0x808080u; }

template <int RC>
__device__ __forceinline__ void tmem_rows(uint32_t t, uint32_t stride, uint32_t (&d)[3][RC]) {
  if constexpr (RC == 16) {
#pragma unroll
    for (int i = 0; i < 3; i++) tmem_ld16(t + i * stride, d[i]);
  } else {
    uint32_t v[32];
    tmem_ld16(t, v);
    if (RC == 8) tmem_ld16(t + 16, v + 16);
#pragma unroll
    for (int i = 0; i < 3 * RC; i++) d[i / RC][i % RC] = v[i];
  }
  tmem_ld_wait();
}

// A run of tiles of one unit, as both the copy warp and the compute warps walk it.
struct KaPiece {
  int s, kvh, blk, u0, tiles, lo, hi;  // unit's first tile on the line and tile count; this CTA's share
  SeqSpan sp;
  int j0, nodes;                       // the block's first node and node count
  int seen;                            // slots that any of its rows can see: 0 .. seen - 1
};

__device__ __forceinline__ int ka_cap(const hg_kv8_cache& C) { return C.bt_stride * KV8_PAGE; }
__device__ __forceinline__ int ka_tiles(const hg_kv8_cache& C, const SeqSpan& sp) {
  return (int)((min((long long)sp.start + sp.n, (long long)ka_cap(C)) + KA_TILE - 1) / KA_TILE);
}

__device__ __forceinline__ KaPiece ka_piece(const KaArgs& A, const uint32_t* pre, int t, int end) {
  KaPiece u;
  int a = 0, b = A.R.n_seqs - 1;
  while (a < b) {
    const int mid = (a + b + 1) >> 1;
    if (pre[mid] <= (uint32_t)t) a = mid;
    else b = mid - 1;
  }
  u.s = a;
  u.sp = kv8_span(A.R, a, true);
  u.tiles = ka_tiles(A.C, u.sp);
  const int blocks = (u.sp.n + A.npb - 1) / A.npb, k = (t - (int)pre[a]) / u.tiles;
  u.kvh = k / blocks;
  u.blk = k - u.kvh * blocks;
  u.u0 = (int)pre[a] + k * u.tiles;
  u.j0 = u.blk * A.npb;
  u.nodes = min(A.npb, u.sp.n - u.j0);
  u.seen = (int)min((long long)u.sp.start + u.j0 + u.nodes, (long long)ka_cap(A.C));
  u.lo = t - u.u0;
  u.hi = min(end - u.u0, u.tiles);
  return u;
}
// Tiles from here on show nothing to the block's rows.
__device__ __forceinline__ int ka_last(const KaPiece& u) { return min(u.hi, (u.seen + KA_TILE - 1) / KA_TILE); }

__device__ __forceinline__ bool ka_wait(uint64_t* bar, uint32_t parity, int* fail) {
  if (*reinterpret_cast<volatile int*>(fail)) return false;
  if (mbar_wait(bar, parity)) return true;
  *reinterpret_cast<volatile int*>(fail) = 1;
  return false;
}

template <int HD, int R>
__global__ void __launch_bounds__(KA_THREADS, R == 32 ? 2 : 3) k_kv8_attn(const __grid_constant__ KaArgs A) {
  using S = KaShape<HD, R>;
  constexpr int STAGES = S::STAGES, E = HD / 32;
  extern __shared__ __align__(128) unsigned char ka_raw[];
  unsigned char* bq = ka_raw + S::OFF_BQ;
  unsigned char* bp = ka_raw + S::OFF_BP;
  KaSmall<R>& sm = *reinterpret_cast<KaSmall<R>*>(ka_raw + S::OFF_SMALL);
  uint32_t* pre = reinterpret_cast<uint32_t*>(ka_raw + S::OFF_SMALL + sizeof(KaSmall<R>));  // [n_seqs + 1]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n_seqs = A.R.n_seqs;
  pdl_wait();
  pdl_trigger();

  // ---- the line of tiles: first tile of each sequence ----
  for (int s = tid; s < n_seqs; s += KA_THREADS) {
    const SeqSpan sp = kv8_span(A.R, s, true);
    if ((long long)sp.start + sp.n > ka_cap(A.C)) kv8_flag(A.R.err, HG_ERR_CONTEXT);
    pre[s + 1] = (uint32_t)ka_tiles(A.C, sp) * A.C.n_kv_heads * ((sp.n + A.npb - 1) / A.npb);
  }
  if (tid == 0) {
    pre[0] = 0;
    for (int k = 0; k < STAGES; k++) {
      mbar_init(&sm.full[k], KA_PAGES);
      mbar_init(&sm.empty[k], 1);
    }
    mbar_init(&sm.sbar, 1);
    mbar_init(&sm.obar, 1);
    sm.fail = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (warp == 0) {
    uint32_t run = 0;
    for (int s0 = 0; s0 < n_seqs; s0 += 32) {
      const int s = s0 + lane;
      uint32_t v = s < n_seqs ? pre[s + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t w = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += w;
      }
      if (s < n_seqs) pre[s + 1] = run + v;
      run += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
  const long long T = pre[n_seqs];
  const int G = (int)min((long long)gridDim.x, T), cta = blockIdx.x;
  if (tid == 0) A.head[cta] = make_int4(-1, 0, 0, 0);
  if (cta >= G) return;
  const int begin = (int)(T * cta / G), end = (int)(T * (cta + 1) / G);

  if (warp == KA_COMPUTE / 32) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)),
                 "r"(S::COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = sm.tmem;

  if (warp == KA_COMPUTE / 32) {
    // =================== copy warp: lanes 0..7 fetch a page of the tile each ===================
    int n = 0;
    for (int t = begin; t < end;) {
      const KaPiece u = ka_piece(A, pre, t, end);
      const int last = ka_last(u);
      auto page_of = [&](int tile) -> const uint8_t* {
        const long long slot = (long long)tile * KA_TILE + lane * KV8_PAGE;
        if (lane >= KA_PAGES || tile >= last || slot >= u.seen) return nullptr;
        const uint8_t* b = kv8_block(A.C, u.s, slot, u.kvh);
        if (!b) kv8_flag(A.R.err, HG_ERR_CONTEXT);
        return b;
      };
      const uint8_t* src = page_of(u.lo);
      for (int tile = u.lo; tile < last; tile++, n++) {
        const int k = n % STAGES;
        if (n >= STAGES) ka_wait(&sm.empty[k], (n / STAGES - 1) & 1, &sm.fail);
        const uint32_t there = __ballot_sync(0xffffffffu, src != nullptr);
        if (lane == 0) sm.pages[k] = there;
        __syncwarp();
        if (lane < KA_PAGES) {
          unsigned char* st = ka_raw + k * S::STAGE;
          if (src) {
            mbar_arrive_tx(&sm.full[k], kv8_block_bytes(HD));
            bulk_copy(st + lane * 16 * HD, src, 16 * HD, &sm.full[k]);
            bulk_copy(st + S::KBYTES + lane * 16 * HD, src + 16 * HD, 16 * HD, &sm.full[k]);
            bulk_copy(st + 2 * S::KBYTES + lane * 128, src + 32 * HD, 128, &sm.full[k]);
          } else {
            mbar_arrive(&sm.full[k]);
          }
        }
        src = page_of(tile + 1);
      }
      t = u.u0 + u.hi;
    }
    for (int i = max(0, n - STAGES); i < n; i++) mbar_wait(&sm.full[i % STAGES], (i / STAGES) & 1);
  } else {
    // =================== compute warps ===================
    const uint32_t tq = tm + ((uint32_t)(warp * 32) << 16);
    unsigned char* bp_mine = bp + (tid >> 4) * (S::NB * 16) + (tid & 15);
    const uint32_t bq_a = smem_u32(bq), bp_a = smem_u32(bp), ring_a = smem_u32(ka_raw);
    constexpr uint32_t IDESC = tc_idesc(KA_TILE, S::N);
    int n = 0;  // tiles done by this CTA
    auto issue_scores = [&](int k) {  // thread 0: S = K . q digits
      const uint32_t a = ring_a + k * S::STAGE;
#pragma unroll
      for (int i = 0; i < HD / 32; i++)
        tc_mma_acc(tm, tc_desc(a + i * 256, 128, 8 * HD, 0), tc_desc(bq_a + i * 2 * S::NB * 16, S::NB * 16, 128, 0),
                   IDESC, i > 0);
      tc_commit(&sm.sbar);
    };
    for (int t = begin; t < end;) {
      const KaPiece u = ka_piece(A, pre, t, end);
      const int last = ka_last(u);
      // ---- the block's queries as digits, and what its rows see ----
      for (int r = warp; r < R; r += 4) {
        const int node = r / A.g, h = u.kvh * A.g + r - node * A.g;
        const bool on = node < u.nodes;
        float x[E], amax = 0.0f, poison = 0.0f;
        if (on) {
          const float* src = A.q + ((size_t)(u.sp.r0 + u.j0 + node) * A.nh + h) * HD + lane * E;
          if constexpr (E == 4) {
            const float4 v = *reinterpret_cast<const float4*>(src);
            x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
          } else {
            const float2 v = *reinterpret_cast<const float2*>(src);
            x[0] = v.x, x[1] = v.y;
          }
        } else {
#pragma unroll
          for (int e = 0; e < E; e++) x[e] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < E; e++) {
          amax = fmaxf(amax, fabsf(x[e]));
          poison = __fmaf_rn(x[e], 0.0f, poison);  // NaN for a NaN or an infinity
        }
        amax = warp_fmax(amax);
        const float inv = amax > 1e-30f ? __fdiv_rn(KA_FIX, amax) : 0.0f;  // below: the scores are zero
        uint32_t w[3] = {0, 0, 0};
#pragma unroll
        for (int e = 0; e < E; e++) {
          const uint32_t d = to_digits((uint32_t)__float2int_rn(fminf(fmaxf(x[e] * inv, -KA_FIX), KA_FIX)));
#pragma unroll
          for (int i = 0; i < 3; i++) w[i] |= ((d >> (8 * i)) & 255u) << (8 * e);
        }
#pragma unroll
        for (int i = 0; i < 3; i++) {
          const int row = i * R + r, kb = lane * E;
          unsigned char* d = bq + (kb >> 4) * (S::NB * 16) + (row >> 3) * 128 + (row & 7) * 16 + (kb & 15);
          if constexpr (E == 4) *reinterpret_cast<uint32_t*>(d) = w[i];
          else *reinterpret_cast<uint16_t*>(d) = (uint16_t)w[i];
        }
        const bool bad = __any_sync(0xffffffffu, poison != poison);
        if (lane == 0) {
          sm.qs[r] = bad ? __int_as_float(0x7fffffff)
                         : (float)((double)amax / KA_FIX * (1.4426950408889634 / sqrt((double)HD)));
          int lim = 0;
          if (on) {
            const int par = kv8_parent(A.R, u.sp, u.j0 + node);
            const long long up_to = A.R.parent ? u.sp.start : (long long)u.sp.start + u.j0 + node + 1;
            lim = par == -2 ? 0 : (int)min(up_to, (long long)ka_cap(A.C));
          }
          sm.lim[r] = lim;
        }
      }
      fence_async_smem();
      bar_compute();
      float acc[R], l[R], m[R], c_run = 0.0f;
#pragma unroll
      for (int r = 0; r < R; r++) acc[r] = 0.0f, l[r] = 0.0f, m[r] = -INFINITY;
      if (tid == 0 && u.lo < last) {
        ka_wait(&sm.full[n % STAGES], (n / STAGES) & 1, &sm.fail);
        tc_fence_after();
        issue_scores(n % STAGES);
      }
      for (int tile = u.lo; tile < last; tile++, n++) {
        const int k = n % STAGES;
        const int slot = tile * KA_TILE + tid;
        unsigned char* st = ka_raw + k * S::STAGE;
        ka_wait(&sm.full[k], (n / STAGES) & 1, &sm.fail);  // the scales (the codes are the MMAs')
        const float* sc = reinterpret_cast<const float*>(st + 2 * S::KBYTES + (tid >> 4) * 128) + (tid & 15);
        const float ks = sc[0];
        float vs = sc[16];
        const uint32_t there = sm.pages[k];
        // every slot is context of every row and its page is there: nothing to mask
        const bool whole = there == (1u << KA_PAGES) - 1 && (tile + 1) * KA_TILE <= u.sp.start;
        if (!whole) {
          const bool tree = A.R.parent && (tile + 1) * KA_TILE > u.sp.start;
          if (tree) {
            // the path of each node, as bits of this tile
            if (tid < R) {
              uint32_t v[4] = {0, 0, 0, 0};
              const int node = tid / A.g;
              if (node < u.nodes) {
                for (int at = u.j0 + node; at >= 0;) {
                  const int up = kv8_parent(A.R, u.sp, at);
                  if (up == -2) break;
                  const long long b = (long long)u.sp.start + at - (long long)tile * KA_TILE;
                  if (b < 0) break;  // ancestors lie below
                  if (b < KA_TILE) {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                      if ((b >> 5) == i) v[i] |= 1u << (b & 31);
                  }
                  at = up;
                }
              }
#pragma unroll
              for (int i = 0; i < 4; i++) sm.vis[tid][i] = v[i];
            }
            bar_compute();
          }
        }
        ka_wait(&sm.sbar, n & 1, &sm.fail);
        __syncwarp();
        tc_fence_after();
        float s[R];
#pragma unroll
        for (int r0 = 0; r0 < R; r0 += S::RC) {
          uint32_t d[3][S::RC];
          tmem_rows<S::RC>(tq + r0, R, d);
#pragma unroll
          for (int r = 0; r < S::RC; r++) s[r0 + r] = digits(d[0][r], d[1][r], d[2][r]) * sm.qs[r0 + r] * ks;
        }
        if (!whole) {
          const bool in = (there >> (tid >> 4)) & 1u;
          const bool tree = A.R.parent && (tile + 1) * KA_TILE > u.sp.start;
          bool any = false;
#pragma unroll
          for (int r = 0; r < R; r++) {
            bool see = slot < sm.lim[r];
            if (tree) see = see || ((sm.vis[r][warp] >> lane) & 1u);
            if (see && in) any = true;
            else s[r] = -INFINITY;
          }
          if (!any) vs = 0.0f;  // what lies in an unseen slot counts nowhere, not for the scales' maximum either
        }
        // ---- the tile's maximum per row, and of the V scales ----
        float mine = 0.0f;
#pragma unroll
        for (int r = 0; r < R; r++) {
          const float v = warp_fmax(s[r]);
          if (lane == r) mine = v;
        }
        if (lane < R) sm.wmax[lane][warp] = mine;
        const float vfin = vs <= 3.402823466e38f ? vs : 0.0f;  // a NaN or infinite V scale: see `bad`
        const float bad = __fmul_rn(vs, 0.0f);                 // NaN then, else 0
        const float vm = warp_fmax(vfin);
        if (lane == 0) sm.wsv[warp] = vm;
        bar_compute();
        c_run = fmaxf(fmaxf(c_run, fmaxf(sm.wsv[0], sm.wsv[1])), fmaxf(sm.wsv[2], sm.wsv[3]));
        const float pf = c_run > 0.0f ? __fdiv_rn(vfin, c_run) * KA_FIX : 0.0f;
#pragma unroll
        for (int r = 0; r < R; r++) {
          const float4 w4 = *reinterpret_cast<const float4*>(sm.wmax[r]);
          const float mt = fmaxf(fmaxf(w4.x, w4.y), fmaxf(w4.z, w4.w));
          if (mt > m[r]) {  // the same for every thread
            const float al = m[r] == -INFINITY ? 0.0f : ex2(m[r] - mt);
            acc[r] *= al;
            l[r] *= al;
            m[r] = mt;
          }
          const float p = ex2(s[r] - (m[r] == -INFINITY ? 0.0f : m[r]));
          const bool see = s[r] != -INFINITY;  // a NaN score is seen
          l[r] += see ? p + bad : 0.0f;
          // p * pf in [0, KA_FIX], rounded into the low bits of 2^23 + v
          const uint32_t v = __float_as_uint(__fmaf_rn(see ? p : 0.0f, pf, 8388608.0f)) & 0x7fffffu;
          const uint32_t d = to_digits(v);
#pragma unroll
          for (int i = 0; i < 3; i++) {
            const int row = i * R + r;
            bp_mine[(row >> 3) * 128 + (row & 7) * 16] = (unsigned char)(d >> (8 * i));
          }
        }
        fence_async_smem();
        tc_fence_before();
        bar_compute();
        if (tid == 0) {
          tc_fence_after();
          const uint32_t a = ring_a + k * S::STAGE + S::KBYTES;
#pragma unroll
          for (int i = 0; i < KA_TILE / 32; i++)
            tc_mma_acc(tm + S::COL_O, tc_desc(a + i * 32 * HD, 16 * HD, 128, 0),
                       tc_desc(bp_a + i * 2 * S::NB * 16, S::NB * 16, 128, 0), IDESC, i > 0);
          tc_commit(&sm.obar);
          if (tile + 1 < last) {  // the next tile's scores meanwhile
            ka_wait(&sm.full[(n + 1) % STAGES], ((n + 1) / STAGES) & 1, &sm.fail);
            issue_scores((n + 1) % STAGES);
          }
        }
        __syncwarp();
        ka_wait(&sm.obar, n & 1, &sm.fail);
        __syncwarp();
        tc_fence_after();
        if (tid == 0) mbar_arrive(&sm.empty[k]);  // V was read, K and the scales long before
        const float of = c_run * (1.0f / KA_FIX);
#pragma unroll
        for (int r0 = 0; r0 < R; r0 += S::RC) {
          uint32_t d[3][S::RC];
          tmem_rows<S::RC>(tq + S::COL_O + r0, R, d);
#pragma unroll
          for (int r = 0; r < S::RC; r++) acc[r0 + r] = __fmaf_rn(digits(d[0][r], d[1][r], d[2][r]), of, acc[r0 + r]);
        }
        tc_fence_before();
      }
      // ---- the unit's (or its share's) end ----
#pragma unroll
      for (int r = 0; r < R; r++) {
        const float v = warp_sum(l[r]);
        if (lane == 0) sm.wsum[r][warp] = v;
      }
      bar_compute();
      const bool from0 = u.lo == 0, to_end = u.hi == u.tiles;
      float* part = A.part + ((size_t)cta * 2 + (from0 ? 1 : 0)) * R * (HD + 2);
#pragma unroll
      for (int r = 0; r < R; r++) {
        const int node = r / A.g, h = u.kvh * A.g + r - node * A.g;
        const float4 w4 = *reinterpret_cast<const float4*>(sm.wsum[r]);
        const bool dead = kv8_parent(A.R, u.sp, u.j0 + min(node, u.nodes - 1)) == -2;
        const float tot = dead ? 0.0f : (w4.x + w4.y) + (w4.z + w4.w);
        if (from0 && to_end) {
          if (node < u.nodes && tid < HD)
            A.out[((size_t)(u.sp.r0 + u.j0 + node) * A.nh + h) * HD + tid] = tot == 0.0f ? 0.0f : __fdiv_rn(acc[r], tot);
        } else {
          if (tid < HD) part[r * HD + tid] = acc[r];
          if (tid == 0) {
            part[R * HD + r] = m[r];
            part[R * HD + R + r] = tot;
          }
        }
      }
      if (from0 && !to_end && tid == 0) {
        // this CTA's share is the first: the join goes on to the CTA that holds the unit's last tile
        const int lt = u.u0 + u.tiles - 1;
        A.head[cta] = make_int4(u.sp.r0 + u.j0, u.kvh, u.nodes, (int)((((long long)lt + 1) * G - 1) / T));
      }
      bar_compute();
      t = u.u0 + u.hi;
    }
  }
  // ---- wind-down: every MMA was waited for (bounded) by its tile; free the columns ----
  tc_fence_before();
  __syncthreads();
  if (warp == KA_COMPUTE / 32)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(S::COLS));
  if (tid == 0 && sm.fail) kv8_flag(A.R.err, HG_ERR_TIMEOUT);
}

// The partial results of a unit whose tiles lie in several CTAs, added up in tile order: one CTA per
// first share and row.
template <int HD, int R>
__global__ void __launch_bounds__(HD) k_kv8_join(const __grid_constant__ KaArgs A) {
  pdl_wait();
  pdl_trigger();
  const int c0 = blockIdx.x, r = blockIdx.y;
  const int4 h = A.head[c0];
  if (h.x < 0) return;
  const int node = r / A.g;
  if (node >= h.z) return;
  constexpr int P = R * (HD + 2);
  auto part = [&](int c) { return A.part + ((size_t)c * 2 + (c == c0 ? 1 : 0)) * P; };
  float mx = -INFINITY;
  for (int c = c0; c <= h.w; c++) mx = fmaxf(mx, part(c)[R * HD + r]);
  float o = 0.0f, tot = 0.0f;
  for (int c = c0; c <= h.w; c++) {
    const float* p = part(c);
    const float m = p[R * HD + r], f = m == -INFINITY ? 0.0f : ex2(m - mx);
    o = __fmaf_rn(p[r * HD + threadIdx.x], f, o);
    tot = __fmaf_rn(p[R * HD + R + r], f, tot);
  }
  A.out[((size_t)(h.x + node) * A.nh + h.y * A.g + r - node * A.g) * HD + threadIdx.x] =
      tot == 0.0f ? 0.0f : __fdiv_rn(o, tot);
}

// ---- host ----
namespace {

void check_attn(const hg_kv8_cache* c, const hg_rows* r, int n_heads) {
  kv8_check_cache(c);
  kv8_check_rows(r, true);
  kv8_need(n_heads > 0 && n_heads % c->n_kv_heads == 0, "bad head counts");
  kv8_need(n_heads / c->n_kv_heads <= KV8_MAX_GROUP, "more than 32 q heads per kv head");
}

// Rows of a block: the fewest of 4, 8, 16 or 32 that hold a sequence's rows for one kv head, so that a
// single token pays for one node and a tree reads the cache as few times as possible.
int block_rows(const hg_rows* r, int g) {
  const long long want = (long long)std::min(r->max_rows, r->n_rows) * g;
  return want <= 4 ? 4 : want <= 8 ? 8 : want <= 16 ? 16 : 32;
}

size_t part_bytes(int R, int hd) { return (size_t)KA_MAX_CTAS * 2 * R * (hd + 2) * 4; }

template <int HD, int R>
void launch(KaArgs& A, int device, cudaStream_t st) {
  using S = KaShape<HD, R>;
  const size_t smem = S::OFF_SMALL + sizeof(KaSmall<R>) + (A.R.n_seqs + 1) * sizeof(uint32_t);
  constexpr size_t most = S::OFF_SMALL + sizeof(KaSmall<R>) + (KV8_MAX_SEQS + 1) * sizeof(uint32_t);
  static std::atomic<uint64_t> ready{0};  // devices whose kernel has its shared-memory limit set
  const uint64_t bit = 1ull << (device & 63);
  if (device > 63 || !(ready.load() & bit)) {
    const cudaError_t e =
        cudaFuncSetAttribute(k_kv8_attn<HD, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    if (e != cudaSuccess) throw Error(HG_ERR_CUDA, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
    if (device <= 63) ready.fetch_or(bit);
  }
  const int per_sm = (int)std::min<size_t>(std::min(3, 512 / S::COLS), (228 * 1024) / (smem + 1024));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(KA_SMS * per_sm);
  cfg.blockDim = dim3(KA_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  kv8_launched(cudaLaunchKernelEx(&cfg, k_kv8_attn<HD, R>, A));
  cfg.gridDim = dim3(KA_SMS * per_sm, R);
  cfg.blockDim = dim3(HD);
  cfg.dynamicSmemBytes = 0;
  kv8_launched(cudaLaunchKernelEx(&cfg, k_kv8_join<HD, R>, A));
}

}  // namespace
}  // namespace hg

using namespace hg;

extern "C" size_t hg_op_kv8_attn_scratch_bytes(const hg_kv8_cache* c, const hg_rows* r, int n_heads) {
  try {
    check_attn(c, r, n_heads);
    if (r->n_seqs == 0 || r->n_rows == 0) return 256;
    return part_bytes(block_rows(r, n_heads / c->n_kv_heads), c->head_dim) + KA_MAX_CTAS * sizeof(int4);
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
    KaArgs A{};
    A.C = *c;
    A.R = *r;
    A.nh = n_heads;
    A.g = n_heads / c->n_kv_heads;
    const int R = block_rows(r, A.g);
    A.npb = R / A.g;
    // tiles are numbered with 32 bits: the most that the arguments allow
    const double tiles = ((double)r->n_rows / A.npb + r->n_seqs) * ((double)c->bt_stride / KA_PAGES + 1) * c->n_kv_heads;
    kv8_need(tiles < 2147483647.0, "rows x table entries x kv heads out of range for one call");
    A.q = q;
    A.out = out;
    A.part = static_cast<float*>(scratch);
    A.head = reinterpret_cast<int4*>(static_cast<char*>(scratch) + part_bytes(R, c->head_dim));
    Kv8Device dev(c->pool);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const int d = dev.device;
    if (c->head_dim == 64) {
      if (R == 4) launch<64, 4>(A, d, st);
      else if (R == 8) launch<64, 8>(A, d, st);
      else if (R == 16) launch<64, 16>(A, d, st);
      else launch<64, 32>(A, d, st);
    } else {
      if (R == 4) launch<128, 4>(A, d, st);
      else if (R == 8) launch<128, 8>(A, d, st);
      else if (R == 16) launch<128, 16>(A, d, st);
      else launch<128, 32>(A, d, st);
    }
  })
}
