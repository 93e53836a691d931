// Attention of chains and drafted trees over the 8-bit KV cache (hg_op_kv8_attn).
//
// For a row's q head and the slots t that it sees: p_t = exp(q . k_t / sqrt(hd) - m), out =
// sum p_t v_t / sum p_t, with k_t = ks_t K_t and v_t = vs_t V_t, K and V int8 codes. Both contractions
// are integer: q and p_t vs_t are written in fixed point as signed base-256 digits, so the tensor cores
// (tcgen05.mma kind::i8) multiply the cache's bytes as they lie in HBM, exactly, and only the rounding of
// q and of the probabilities and the f32 sums across tiles remain. q has four digits, 30 bits from its
// row's greatest down: with three (23 bits) a q of 1 beside one of 1000 in a channel where K is small would
// be off by 2^-14. No code is converted, no K or V value is formed.
//
// The values' digits have to hold p_t vs_t and not p_t: what a slot adds goes by both, and the greatest p
// and the greatest vs may stand in different slots, or the latter where only another row sees it. So with
// vs_t = 2^e_t f_t, f_t from 1 to 2, a row's running maximum is that of y_t = log2 p_t + e_t (e_t an integer,
// so that nothing is lost by putting it there), the digits are those of 2^(y_t - max) f_t, three of them,
// 2^-23 of the row's own greatest product, and the sum of p takes 2^(y_t - max) 2^-e_t, exact powers of
// two. e_t is -60 at least: V scales below 2^-60, zeros among them, count with f_t < 1. Measured against
// 64-bit attention over the same codes, V scales equal, spread lognormally (sigma 1 and 3), or with one in
// 100 being 100 or 1000 times the rest, seen by a row or not: off by 3e-7 to 1.3e-6 (root mean square,
// relative), plain f32 arithmetic by 2e-7 to 9e-7.
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
// equal runs, one per resident CTA, whatever the lengths; a unit that is cut is joined by k_kv8_join from
// at most two partial results per CTA, in tile order (no atomics). Where the page tables are so short
// that a unit has few tiles, each unit has a cluster of 1 to 16 CTAs instead, joined over distributed
// shared memory: one launch, which is what a small call costs (one sequence of 2100 slots: 8.9 us a call
// against 10.4).
//
// A copy warp keeps two rings full, K tiles with the scales of both and V tiles: per page 16 hd bytes of
// K, 128 of scales and 16 hd of V, bulk copies that need no rearranging (hg_kv8.cuh). One thread issues
// the MMAs: a tile's value product and the next tile's scores together, so that the compute warps find
// scores ready; a tile's value sums are read back while the next tile's maxima meet. Every mbarrier wait
// is bounded; when one gives up, the CTA reports HG_ERR_TIMEOUT, its other waits give up soon too, and it
// waits (bounded) for its copies and last MMAs before it frees its tensor memory and returns.
//
// Measured: 256 sequences of 1024 to 8192 slots (12 q heads, 3 kv heads, 128 dims) 150 us, 5.9 TB/s
// of cache, 0.90 of measured HBM (R = 4, three CTAs an SM: bound by HBM). 32 trees of 64 nodes over 900
// to 7000 slots 264 us, 190 TFLOP/s of f32-like products (R = 32, two CTAs of 288 threads an SM): bound
// by the instructions between the products, about 50 per (slot, row): put four digits together, scale,
// maximum, exponential, sum, three digits again, add the value sums. Issue slots are 57% busy at 17 warps
// an SM, the tensor pipe 16%. The ninth warp leaves the others 96 registers, and some are spilled (52 bytes
// a thread at R = 32, 8 at 16).
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

#include "hg_kv8.cuh"
#include "hg_tc.cuh"

namespace hg {

namespace cg = cooperative_groups;

constexpr int KA_TILE = 128;                      // slots of a tile: the MMA's M
constexpr int KA_PAGES = KA_TILE / KV8_PAGE;      // pages of a tile
constexpr int KA_SMS = 148;
constexpr int KA_MAX_CTAS = 3 * KA_SMS;
constexpr int KA_CLUSTER = 16;                    // most CTAs of a unit's cluster
constexpr float KA_NONE = -3e38f;                 // maximum of a row that has seen nothing: finite, below any score
constexpr float KA_FIX = 8323072.0f;              // 2^23 - 2^16: the greatest fixed-point value, three digits
constexpr float KA_UNIT = 2.0f / KA_FIX;          // a unit of the probabilities' digits

// Shared memory of one CTA, in order: the ring, the digits of q and of the probabilities, small arrays.
template <int HD, int R>
struct KaShape {
  static constexpr int NS = 4 * R;                  // MMA N of the scores: columns of q's digits
  static constexpr int N = (3 * R + 15) / 16 * 16;  // and of the values: columns of the probabilities' digits
  static constexpr int NB = (3 * R + 7) / 8 * 8;    // digit rows kept (what N reads past them stays unread)
  // bytes between 16-byte columns of the digit operands: 16 more than the rows take, so that the two
  // columns that a warp's 32 slots lie in use different banks
  static constexpr int PITCH_Q = NS * 16 + 16, PITCH = NB * 16 + 16;
  // the rings: V tiles, then K tiles with the scales of both (what a 64-dim V operand reads past its
  // tile, for M = 128, is the next tile)
  static constexpr int VSTAGE = KA_TILE * HD, KSTAGE = VSTAGE + KA_PAGES * 128;
  static constexpr int STAGES = HD == 128 ? 2 : 4;
  static constexpr int OFF_K = STAGES * VSTAGE, OFF_BQ = OFF_K + STAGES * KSTAGE, OFF_BP = OFF_BQ + PITCH_Q * (HD / 16),
                       OFF_SMALL = OFF_BP + PITCH * (KA_TILE / 16);
  // tensor-memory columns: S at 0, O behind it; a power of two of at least 32
  static constexpr int COL_O = NS;
  static constexpr int COLS = 2 * COL_O;
  // Compute warps: groups of 128 threads, one slot (S) or dim (O) per thread and RT rows per group; and
  // the copy warp.
  static constexpr int GROUPS = R > 8 ? 2 : 1, RT = R / GROUPS, COMPUTE = 128 * GROUPS, THREADS = COMPUTE + 32;
  static constexpr int RC = RT < 8 ? RT : 8;  // rows per tensor-memory read
  static constexpr int PER_SM = R > 8 ? 2 : 3;
};

template <int R>
struct KaSmall {
  uint64_t full_k[4], empty_k[4], full_v[4], empty_v[4], sbar, obar;
  float wmax[4][R];          // per warp maxima of a tile's scores, and sums at a unit's end
  float m[2][R];             // running maxima of score + exponent of the V scale (log2), by the tile's parity
  float qs[R];               // row r: log2(e) / sqrt(hd) * 2^(exponent of its greatest q)
  int lim[R];                // row r sees the slots below, and the tree slots of `vis`; -1: padding
  int node[R], off[R];       // row r's node within its block, its q head's place behind the block's first
  uint32_t vis[R][4];        // slots of the current tile that row r's path holds
  int at[R];                 // where a node's path goes on below the tiles looked at
  uint32_t pages[4];         // per stage: which of the tile's pages are there
  uint32_t tmem;
  int fail;
  int first_row, kvh, nodes;  // the unit of a cluster (nodes 0: none)
};

struct KaArgs {
  hg_kv8_cache C;
  hg_rows R;
  int nh, g, npb;  // q heads, q heads per kv head, nodes per row block
  int cl;          // CTAs of a unit's cluster, or 0: units on the line
  int take;        // places on the line for taking a unit up
  const float* q;
  float* out;
  float* part;     // [CTA][2][R * (hd + 2)] partial results: rows of hd sums, then maxima, then sums of p
  int4* head;      // [CTA] of a join: first row (-1: none), kv head, nodes, the CTA of the unit's last place
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
template <int N>
__device__ __forceinline__ void bar_named(int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(N) : "memory"); }
__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void mbar_arrive_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
// Sums whose base-256 digits are d0 .. d3, each below 2^21.01 in magnitude, of two rows, / 65536. The upper
// two digits are put together as integers and converted with one rounding, d1 + d0 / 256 exactly, and one
// rounding joins them: like f32 also where the sum is small beside its terms.
__device__ __forceinline__ f32x2 ka_score(float hi0, float hi1, uint32_t d1, uint32_t e1, uint32_t d0, uint32_t e0) {
  const f32x2 lo = add2(pack2(__uint_as_float(d1 + (uint32_t)((int)d0 >> 8) + TC_BIAS),
                              __uint_as_float(e1 + (uint32_t)((int)e0 >> 8) + TC_BIAS)),
                        pack2(-TC_BIAS_F, -TC_BIAS_F));
  return fma2(lo, pack2(0.00390625f, 0.00390625f), pack2(hi0, hi1));
}
// Adds sums of three such digits to acc.
__device__ __forceinline__ f32x2 ka_add(const uint32_t (&d)[3][2], f32x2 acc) {
  const f32x2 hi = pack2(__int2float_rn((int)((d[2][0] << 8) + d[1][0])), __int2float_rn((int)((d[2][1] << 8) + d[1][1])));
  return fma2(hi, pack2(256.0f, 256.0f), add2(pack2(__int2float_rn((int)d[0][0]), __int2float_rn((int)d[0][1])), acc));
}
// Fixed point v (|v| <= 2^30) as signed digits v = b0 + 256 b1 + 65536 b2 + 2^24 b3, one per byte.
__device__ __forceinline__ uint32_t to_digits(uint32_t v) { return (v + 0x80808080u) ^ 0x80808080u; }

// 8 consecutive tensor-memory columns of this warp's 32 lanes.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(taddr));
}
// The loads before are over; their registers pass through, so that nothing reads them earlier.
template <int N>
__device__ __forceinline__ void tmem_wait(uint32_t (&v)[N]) {
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < N; i++) asm volatile("" : "+r"(v[i]));
}
// The sums of RC rows' scores / 65536, digit i of row r in column i * stride + r (d0 in the first).
template <int RC>
__device__ __forceinline__ void tmem_scores(uint32_t t, uint32_t stride, f32x2* s) {
  uint32_t u[16], v[16];
  if constexpr (RC == 8) {
    tmem_ld8(t + 3 * stride, u);
    tmem_ld8(t + 2 * stride, u + 8);
    tmem_wait(u);
    tmem_ld8(t + stride, v);
    tmem_ld8(t, v + 8);
  } else {
    tmem_ld16(t, v);  // the stride is 4: one read has them all
    tmem_wait(v);
#pragma unroll
    for (int i = 0; i < 4; i++) u[i] = v[12 + i], u[4 + i] = v[8 + i];
  }
  float hi[RC];
#pragma unroll
  for (int r = 0; r < RC; r++) hi[r] = __int2float_rn((int)((u[r] << 8) + u[RC + r]));
  if constexpr (RC == 8) tmem_wait(v);
  const uint32_t *d1 = RC == 8 ? v : v + 4, *d0 = RC == 8 ? v + 8 : v;
#pragma unroll
  for (int r = 0; r < RC; r += 2) s[r / 2] = ka_score(hi[r], hi[r + 1], d1[r], d1[r + 1], d0[r], d0[r + 1]);
}
// The three digit columns of RC rows: digit i of row r is column i * stride + r.
template <int RC>
__device__ __forceinline__ void tmem_rows(uint32_t t, uint32_t stride, uint32_t (&d)[3][RC]) {
  if constexpr (RC == 8) {
#pragma unroll
    for (int i = 0; i < 3; i++) tmem_ld8(t + i * stride, d[i]);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 24; i++) asm volatile("" : "+r"(d[i / 8][i % 8]));
  } else {
    uint32_t v[16];  // the stride is RC: one read has them all
    tmem_ld16(t, v);
    tmem_wait(v);
#pragma unroll
    for (int i = 0; i < 3 * RC; i++) d[i / RC][i % RC] = v[i];
  }
}

// A run of tiles of one unit, as both the copy warp and the compute warps walk it.
struct KaPiece {
  int s, kvh, blk, u0, next, tiles, lo, hi;  // the unit's place on the line, its tiles; this CTA's share of them
  SeqSpan sp;
  int j0, nodes;                       // the block's first node and node count
  int seen;                            // slots that any of its rows can see: 0 .. seen - 1
};

__device__ __forceinline__ int ka_cap(const hg_kv8_cache& C) { return C.bt_stride * KV8_PAGE; }
__device__ __forceinline__ int ka_tiles(const hg_kv8_cache& C, const SeqSpan& sp) {
  return (int)((min((long long)sp.start + sp.n, (long long)ka_cap(C)) + KA_TILE - 1) / KA_TILE);
}

// A unit's length on the line: its tiles and what taking it up (the digits of its q rows, a first tile
// with nothing before it, rows written or handed to the join) costs, about as much as `take` tiles.
// Measured with 1, 2, 3, 4 and 6 places, us: 4 rows, 256 sequences 146.5, 147.8, 148.5, 149.0, 150.5; 16
// rows, 200 short sequences 79.4, 72.6, 69.8, 70.4, 73.3; 32 rows, wide trees 283, 276, 271, 264, 269.
constexpr int ka_take(int R) { return R == 4 ? 1 : R == 32 ? 4 : 3; }
__device__ __forceinline__ int ka_line(const KaArgs& A, const SeqSpan& sp) { return ka_tiles(A.C, sp) + A.take; }

// Row blocks of a sequence.
__device__ __forceinline__ int ka_blocks(const KaArgs& A, const SeqSpan& sp) {
  return sp.n <= A.npb ? (sp.n > 0 ? 1 : 0) : (sp.n + A.npb - 1) / A.npb;
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
  const int len = A.cl ? 1 : u.tiles + A.take, blocks = ka_blocks(A, u.sp);
  const int k = A.cl ? t - (int)pre[a] : (int)((uint32_t)(t - (int)pre[a]) / (uint32_t)len);
  u.kvh = blocks == 1 ? k : k / blocks;
  u.blk = k - u.kvh * blocks;
  u.u0 = (int)pre[a] + k * len;
  u.j0 = u.blk * A.npb;
  u.nodes = min(A.npb, u.sp.n - u.j0);
  u.seen = (int)min((long long)u.sp.start + u.j0 + u.nodes, (long long)ka_cap(A.C));
  u.next = u.u0 + len;
  if (A.cl) {  // this CTA's part of the tiles that show something
    const int tiles = (u.seen + KA_TILE - 1) / KA_TILE, rank = blockIdx.x % A.cl;
    u.lo = tiles * rank / A.cl;
    u.hi = tiles * (rank + 1) / A.cl;
    return u;
  }
  // the tiles come behind the places for taking the unit up; a share of those alone is empty (hi <= lo)
  u.lo = max(t - u.u0 - A.take, 0);
  u.hi = min(end - u.u0 - A.take, u.tiles);
  return u;
}
// Tiles from here on show nothing to the block's rows.
__device__ __forceinline__ int ka_last(const KaPiece& u) { return min(u.hi, (u.seen + KA_TILE - 1) / KA_TILE); }

// A bounded wait; after the first that gave up, every other gives up soon.
__device__ __forceinline__ void ka_wait(uint64_t* bar, uint32_t parity, int* fail) {
  const uint32_t a = smem_u32(bar);
  for (long long i = 1; i < TC_SPIN_LIMIT; i++) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(a), "r"(parity)
        : "memory");
    if (done) return;
    if (i % 1024 == 0 && *reinterpret_cast<volatile int*>(fail)) return;
  }
  *reinterpret_cast<volatile int*>(fail) = 1;
}

template <int HD, int R>
__global__ void __launch_bounds__(KaShape<HD, R>::THREADS, KaShape<HD, R>::PER_SM) k_kv8_attn(const __grid_constant__ KaArgs A) {
  using S = KaShape<HD, R>;
  constexpr int STAGES = S::STAGES, E = HD / 32, RT = S::RT, COPY = S::COMPUTE / 32;
  extern __shared__ __align__(128) unsigned char ka_raw[];
  unsigned char* bq = ka_raw + S::OFF_BQ;
  unsigned char* bp = ka_raw + S::OFF_BP;
  KaSmall<R>& sm = *reinterpret_cast<KaSmall<R>*>(ka_raw + S::OFF_SMALL);
  uint32_t* pre = reinterpret_cast<uint32_t*>(ka_raw + S::OFF_SMALL + sizeof(KaSmall<R>));  // [n_seqs + 1]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n_seqs = A.R.n_seqs;
  pdl_wait();
  pdl_trigger();

  // ---- the line of tiles: each sequence's first place (tensor memory and barriers meanwhile) ----
  if (warp == COPY) {
    // after pdl_wait, never before: a kernel still running may have to allocate before it can finish
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)),
                 "r"(S::COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else if (warp == 1) {
    if (lane < R) {
      sm.node[lane] = lane / A.g;
      sm.off[lane] = sm.node[lane] * A.nh + lane % A.g;
    }
    if (lane == 0) {
      for (int k = 0; k < STAGES; k++) {
        mbar_init(&sm.full_k[k], KA_PAGES);
        mbar_init(&sm.full_v[k], KA_PAGES);
        mbar_init(&sm.empty_k[k], 1);
        mbar_init(&sm.empty_v[k], 1);
      }
      mbar_init(&sm.sbar, 1);
      mbar_init(&sm.obar, 1);
      sm.fail = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
  }
  auto places = [&](int s) -> unsigned long long {
    const SeqSpan sp = kv8_span(A.R, s, true);
    if ((long long)sp.start + sp.n > ka_cap(A.C)) kv8_flag(A.R.err, HG_ERR_CONTEXT);
    return (unsigned long long)(A.cl ? 1 : ka_line(A, sp)) * A.C.n_kv_heads * ka_blocks(A, sp);
  };
  auto place32 = [](unsigned long long v) { return (uint32_t)min(v, (unsigned long long)INT_MAX); };
  if (n_seqs > 32) {  // many sequences: every warp loads, then warp 0 adds up
    for (int s = tid; s < n_seqs; s += S::THREADS) pre[s + 1] = place32(places(s));
    __syncthreads();
  }
  if (warp == 0) {
    if (lane == 0) pre[0] = 0;
    unsigned long long run = 0;
    for (int s0 = 0; s0 < n_seqs; s0 += 32) {
      const int s = s0 + lane;
      unsigned long long v = s >= n_seqs ? 0 : n_seqs > 32 ? pre[s + 1] : places(s);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long w = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += w;
      }
      if (s < n_seqs) pre[s + 1] = place32(run + v);
      run += __shfl_sync(0xffffffffu, v, 31);
    }
    // more than the host allowed for: offsets that give rows to several sequences
    if (run >= INT_MAX) {
      if (lane == 0) pre[n_seqs] = 0;
      kv8_flag(A.R.err, HG_ERR_INVALID);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = sm.tmem;
  const long long T = pre[n_seqs];
  const int G = (int)min((long long)gridDim.x, T), cta = blockIdx.x;
  int begin = 0, end = 0;  // places on the line; of a cluster: its unit
  if (A.cl) {
    if (cta / A.cl < T) begin = cta / A.cl, end = begin + 1;
    if (tid == 0) sm.nodes = 0;
  } else {
    if (tid == 0) A.head[cta] = make_int4(-1, 0, 0, 0);
    if (cta < G) begin = (int)(T * cta / G), end = (int)(T * (cta + 1) / G);
  }

  if (warp == COPY) {
    // =================== copy warp: lanes 0..7 fetch a page of the tile each ===================
    int n = 0;
    for (int t = begin; t < end;) {
      const KaPiece u = ka_piece(A, pre, t, end);
      const int last = ka_last(u);
      auto page_of = [&](int tile) -> const uint8_t* {
        const long long slot = (long long)tile * KA_TILE + lane * KV8_PAGE;
        if (lane >= KA_PAGES || tile < u.lo || slot >= u.seen) return nullptr;
        const uint8_t* b = kv8_block(A.C, u.s, slot, u.kvh);
        if (!b) kv8_flag(A.R.err, HG_ERR_CONTEXT);
        return b;
      };
      const uint8_t* src = page_of(last - 1);
      for (int tile = last - 1; tile >= u.lo; tile--, n++) {
        const int k = n % STAGES;
        const uint32_t past = (n / STAGES - 1) & 1;
        if (n >= STAGES) ka_wait(&sm.empty_k[k], past, &sm.fail);
        const uint32_t there = __ballot_sync(0xffffffffu, src != nullptr);
        if (lane == 0) sm.pages[k] = there;
        __syncwarp();
        if (lane < KA_PAGES) {
          if (src) {
            unsigned char* st = ka_raw + S::OFF_K + k * S::KSTAGE;
            mbar_arrive_tx(&sm.full_k[k], 16 * HD + 128);
            bulk_copy(st + lane * 16 * HD, src, 16 * HD, &sm.full_k[k]);
            bulk_copy(st + S::VSTAGE + lane * 128, src + 32 * HD, 128, &sm.full_k[k]);
          } else {
            mbar_arrive(&sm.full_k[k]);
          }
        }
        const uint8_t* next = page_of(tile - 1);
        if (n >= STAGES) ka_wait(&sm.empty_v[k], past, &sm.fail);
        if (lane < KA_PAGES) {
          if (src) {
            mbar_arrive_tx(&sm.full_v[k], 16 * HD);
            bulk_copy(ka_raw + k * S::VSTAGE + lane * 16 * HD, src + 16 * HD, 16 * HD, &sm.full_v[k]);
          } else {
            mbar_arrive(&sm.full_v[k]);
          }
        }
        src = next;
      }
      t = u.next;
    }
    for (int i = max(0, n - STAGES); i < n; i++) {
      mbar_wait(&sm.full_k[i % STAGES], (i / STAGES) & 1);
      mbar_wait(&sm.full_v[i % STAGES], (i / STAGES) & 1);
    }
  } else {
    // =================== compute warps ===================
    // this thread: slot / dim ti of the tile, rows rb .. rb + RT - 1
    const int ti = tid & 127, quad = warp & 3, grp = warp >> 2, rb = grp * RT;
    const uint32_t tq = tm + ((uint32_t)(quad * 32) << 16) + rb;
    unsigned char* bp_mine[3];  // its byte of the digit operand's rows rb, R + rb, 2 R + rb
#pragma unroll
    for (int b = 0; b < 3; b++)
      bp_mine[b] = bp + (ti >> 4) * S::PITCH + (ti & 15) + ((b * R + rb) >> 3) * 128 + ((b * R + rb) & 7) * 16;
    auto bar_all = [&]() { bar_named<S::COMPUTE>(1); };
    auto bar_group = [&]() {
      if constexpr (S::GROUPS == 1) bar_all();
      else bar_named<128>(2 + grp);
    };
    const uint32_t bq_a = smem_u32(bq), bp_a = smem_u32(bp), ring_a = smem_u32(ka_raw);
    constexpr uint32_t IDESC_S = tc_idesc(KA_TILE, S::NS), IDESC_O = tc_idesc(KA_TILE, S::N);
    int n = 0;  // tiles done by this CTA
    auto issue_scores = [&](int k) {  // thread 0: S = K . q digits
      const uint32_t a = ring_a + S::OFF_K + k * S::KSTAGE;
#pragma unroll
      for (int i = 0; i < HD / 32; i++)
        tc_mma_acc(tm, tc_desc(a + i * 256, 128, 8 * HD, 0), tc_desc(bq_a + i * 2 * S::PITCH_Q, S::PITCH_Q, 128, 0),
                   IDESC_S, i > 0);
      tc_commit(&sm.sbar);
    };
    for (int t = begin; t < end;) {
      const KaPiece u = ka_piece(A, pre, t, end);
      if (!A.cl && u.hi <= u.lo) break;  // the next CTA takes the unit up
      const int last = ka_last(u);
      // ---- the block's queries as digits, and what its rows see ----
      constexpr int W = S::COMPUTE / 32;
      float x[R / W][E];
#pragma unroll
      for (int i = 0; i < R / W; i++) {  // warp w: rows w, w + W, ...
        const int r = warp + W * i;
        const float* src = A.q + ((size_t)(u.sp.r0 + u.j0) * A.nh + u.kvh * A.g + sm.off[r]) * HD + lane * E;
#pragma unroll
        for (int e = 0; e < E; e++) x[i][e] = 0.0f;
        if (sm.node[r] < u.nodes) {
          if constexpr (E == 4) {
            const float4 v = *reinterpret_cast<const float4*>(src);
            x[i][0] = v.x, x[i][1] = v.y, x[i][2] = v.z, x[i][3] = v.w;
          } else {
            const float2 v = *reinterpret_cast<const float2*>(src);
            x[i][0] = v.x, x[i][1] = v.y;
          }
        }
      }
      if (tid < R) {
        int lim = 0;
        if (sm.node[tid] < u.nodes) {
          const int j = u.j0 + sm.node[tid];
          const long long up_to = A.R.parent ? u.sp.start : (long long)u.sp.start + j + 1;
          lim = kv8_parent(A.R, u.sp, j) == -2 ? -1 : (int)min(up_to, (long long)ka_cap(A.C));
        }
        sm.lim[tid] = lim;
        sm.at[tid] = u.j0 + tid;
        *reinterpret_cast<uint4*>(sm.vis[tid]) = make_uint4(0, 0, 0, 0);
        sm.m[0][tid] = sm.m[1][tid] = KA_NONE;
      }
#pragma unroll
      for (int i = 0; i < R / W; i++) {
        const int r = warp + W * i;
        float amax = 0.0f, poison = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) {
          amax = fmaxf(amax, fabsf(x[i][e]));
          poison = __fmaf_rn(x[i][e], 0.0f, poison);  // NaN for a NaN or an infinity
        }
        amax = warp_fmax(amax);
        // units of 2^(ex - 29), so that |v| < 2^30: a power of two, so that what lies within 2^6 of the greatest is exact
        const int ex = min(max((int)(__float_as_uint(amax) >> 23) - 127, -97), 127);
        const float inv = __uint_as_float((uint32_t)(156 - ex) << 23);
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < E; e++) {
          const uint32_t d = to_digits((uint32_t)__float2int_rn(x[i][e] * inv));
#pragma unroll
          for (int b = 0; b < 4; b++) w[b] |= ((d >> (8 * b)) & 255u) << (8 * e);
        }
#pragma unroll
        for (int b = 0; b < 4; b++) {
          const int row = b * R + r, kb = lane * E;
          unsigned char* d = bq + (kb >> 4) * S::PITCH_Q + (row >> 3) * 128 + (row & 7) * 16 + (kb & 15);
          if constexpr (E == 4) *reinterpret_cast<uint32_t*>(d) = w[b];
          else *reinterpret_cast<uint16_t*>(d) = (uint16_t)w[b];
        }
        const bool bad = __any_sync(0xffffffffu, poison != poison);
        if (lane == 0)
          sm.qs[r] = bad ? __int_as_float(0x7fffffff)
                         : (float)(1.4426950408889634 / (HD == 64 ? 8.0 : 11.313708498984761)) * __uint_as_float((uint32_t)(ex + 127) << 23);
      }
      fence_async_smem();
      bar_all();
      f32x2 acc[RT / 2], l[RT / 2];
#pragma unroll
      for (int r = 0; r < RT / 2; r++) acc[r] = l[r] = 0ull;
      // the sums over the dims that the MMAs of tile n - 1 left in tensor memory
      auto add_out = [&](int n_of) {
        ka_wait(&sm.obar, n_of & 1, &sm.fail);
        __syncwarp();
        tc_fence_after();
        if (tid == 0) mbar_arrive(&sm.empty_v[n_of % STAGES]);
#pragma unroll
        for (int r0 = 0; r0 < RT; r0 += S::RC) {
          uint32_t d[3][S::RC];
          tmem_rows<S::RC>(tq + S::COL_O + r0, R, d);
#pragma unroll
          for (int r = 0; r < S::RC; r += 2) {
            const uint32_t e[3][2] = {{d[0][r], d[0][r + 1]}, {d[1][r], d[1][r + 1]}, {d[2][r], d[2][r + 1]}};
            acc[(r0 + r) / 2] = ka_add(e, acc[(r0 + r) / 2]);
          }
        }
        tc_fence_before();
      };
      if (tid == 0 && u.lo < last) {
        ka_wait(&sm.full_k[n % STAGES], (n / STAGES) & 1, &sm.fail);
        tc_fence_after();
        issue_scores(n % STAGES);
      }
      // from the last tile down, so that a path is walked once and not from its row again for every tile
      for (int tile = last - 1; tile >= u.lo; tile--, n++) {
        const int k = n % STAGES;
        const int slot = tile * KA_TILE + ti;
        ka_wait(&sm.full_k[k], (n / STAGES) & 1, &sm.fail);  // the scales (the codes are the MMAs')
        const float* sc =
            reinterpret_cast<const float*>(ka_raw + S::OFF_K + k * S::KSTAGE + S::VSTAGE + (ti >> 4) * 128) + (ti & 15);
        // the V scale as 2^e times 1 to 2 (below 2^-60, or 0: times less than 1); a NaN, an infinity or what is
        // below zero is nothing, and poisons the rows that see the slot
        const float ks = fabsf(sc[0]) <= 3.402823466e38f ? sc[0] : __int_as_float(0x7fffffff), vs = sc[16];
        const bool fine = vs >= 0.0f && vs < 1.7014118346e38f;
        const uint32_t ve = fine ? max((__float_as_uint(vs) & 0x7fffffffu) >> 23, 67u) : 127u;
        const float e = (float)((int)ve - 127), inv = __uint_as_float((254u - ve) << 23);
        const float pf = fine ? vs * inv * (KA_FIX * 0.5f) : 0.0f;
        const uint32_t there = sm.pages[k];
        // every slot is context of every row and its page is there: nothing to mask
        const bool whole = there == (1u << KA_PAGES) - 1 && (tile + 1) * KA_TILE <= u.sp.start;
        const bool tree = A.R.parent && (tile + 1) * KA_TILE > u.sp.start;
        if (tree) {
          // the path of each node, as bits of this tile: half a warp a node, lanes 0..3 a word each
          for (int node = tid >> 4; node < u.nodes; node += S::COMPUTE / 16) {
            const int word = lane & 15;
            uint32_t v = 0;
            int at = sm.at[node];
            while (at >= 0) {
              const long long b = (long long)u.sp.start + at - (long long)tile * KA_TILE;  // bit of row `at`
              if (b < 0) break;  // the path goes on in a tile below
              const PathRun run = kv8_run<16>(A.R, u.sp, at);
              const int hi = (int)min(b - 32 * word, 31ll), lo = (int)max(b - run.len + 1 - 32 * word, 0ll);
              if (word < 4 && lo <= hi) v |= (0xffffffffu >> (31 - (hi - lo))) << lo;
              at = run.len > b + 1 ? at - (int)b - 1 : run.next;
            }
            if (word < 4)
              for (int r = node * A.g; r < (node + 1) * A.g; r++) sm.vis[r][word] = v;
            if (word == 0) sm.at[node] = at;
          }
          bar_all();
        }
        ka_wait(&sm.sbar, n & 1, &sm.fail);
        __syncwarp();
        tc_fence_after();
        f32x2 s[RT / 2];
        const float ks13 = ks * 0.0001220703125f;  // 2^-13: 2^-29 of q's units, 2^16 of the sums'
        const f32x2 ks2 = pack2(ks13, ks13), e2 = pack2(e, e);
#pragma unroll
        for (int r0 = 0; r0 < RT; r0 += S::RC) {
          tmem_scores<S::RC>(tq + r0, R, s + r0 / 2);
#pragma unroll
          for (int r = 0; r < S::RC; r += 4) {
            const float4 q = *reinterpret_cast<const float4*>(&sm.qs[rb + r0 + r]);
            f32x2* x = s + (r0 + r) / 2;
            x[0] = fma2(mul2(x[0], ks2), pack2(q.x, q.y), e2);
            x[1] = fma2(mul2(x[1], ks2), pack2(q.z, q.w), e2);
          }
        }
        if (!whole) {
          const bool in = (there >> (ti >> 4)) & 1u;
#pragma unroll
          for (int r = 0; r < RT; r += 2) {
            float x[2];
            unpack2(s[r / 2], x[0], x[1]);
#pragma unroll
            for (int i = 0; i < 2; i++) {
              bool see = slot < sm.lim[rb + r + i];
              if (tree) see = see || ((sm.vis[rb + r + i][quad] >> lane) & 1u);
              if (!(see && in)) x[i] = -INFINITY;
            }
            s[r / 2] = pack2(x[0], x[1]);
          }
        }
        // ---- the tile's maximum per row ----
#pragma unroll
        for (int r = 0; r < RT; r += 4) {
          float x[4];
          unpack2(s[r / 2], x[0], x[1]);
          unpack2(s[r / 2 + 1], x[2], x[3]);
          const float4 v = make_float4(warp_fmax(x[0]), warp_fmax(x[1]), warp_fmax(x[2]), warp_fmax(x[3]));
          if (lane == 0) *reinterpret_cast<float4*>(&sm.wmax[quad][rb + r]) = v;
        }
        if (tile < last - 1) add_out(n - 1);  // the previous tile's sums, while the others get here
        bar_group();
        const int now = n & 1;
        if (__any_sync(0xffffffffu, !fine)) {
          const float bad = fine ? 0.0f : __int_as_float(0x7fffffff);
#pragma unroll
          for (int r = 0; r < RT; r += 2) {
            float x[2];
            unpack2(s[r / 2], x[0], x[1]);
            l[r / 2] = add2(l[r / 2], pack2(x[0] != -INFINITY ? bad : 0.0f, x[1] != -INFINITY ? bad : 0.0f));
          }
        }
        const f32x2 pf2 = pack2(pf, pf), inv2 = pack2(inv, inv), big = pack2(8388608.0f + 32896.0f, 8388608.0f + 32896.0f);
#pragma unroll
        for (int r0 = 0; r0 < RT; r0 += 4) {  // four rows at a time, so that their maxima need not stay in registers
          const float4 a = *reinterpret_cast<const float4*>(&sm.wmax[0][rb + r0]), b = *reinterpret_cast<const float4*>(&sm.wmax[1][rb + r0]);
          const float4 c = *reinterpret_cast<const float4*>(&sm.wmax[2][rb + r0]), d = *reinterpret_cast<const float4*>(&sm.wmax[3][rb + r0]);
          const float4 o = *reinterpret_cast<const float4*>(&sm.m[now ^ 1][rb + r0]);
          const float4 m4 = make_float4(fmaxf(fmaxf(fmaxf(a.x, b.x), fmaxf(c.x, d.x)), o.x), fmaxf(fmaxf(fmaxf(a.y, b.y), fmaxf(c.y, d.y)), o.y),
                                        fmaxf(fmaxf(fmaxf(a.z, b.z), fmaxf(c.z, d.z)), o.z), fmaxf(fmaxf(fmaxf(a.w, b.w), fmaxf(c.w, d.w)), o.w));
          if (ti == 0) *reinterpret_cast<float4*>(&sm.m[now][rb + r0]) = m4;
          const float m[4] = {m4.x, m4.y, m4.z, m4.w};
          if (m[0] > o.x || m[1] > o.y || m[2] > o.z || m[3] > o.w) {  // the same for every thread of the group
            const f32x2 al[2] = {pack2(ex2(o.x - m[0]), ex2(o.y - m[1])), pack2(ex2(o.z - m[2]), ex2(o.w - m[3]))};
#pragma unroll
            for (int i = 0; i < 2; i++) {
              acc[r0 / 2 + i] = mul2(acc[r0 / 2 + i], al[i]);
              l[r0 / 2 + i] = mul2(l[r0 / 2 + i], al[i]);
            }
          }
#pragma unroll
          for (int r = r0; r < r0 + 4; r += 2) {
            float x[2];
            unpack2(add2(s[r / 2], pack2(-m[r - r0], -m[r - r0 + 1])), x[0], x[1]);
            const f32x2 p = pack2(ex2(x[0]), ex2(x[1]));
            l[r / 2] = fma2(p, inv2, l[r / 2]);
            // p * pf in [0, KA_FIX], rounded into the low bits of 2^23 + 0x8080 + v: the lower digits' bytes
            // are 128 up, which the exclusive or takes back
            unpack2(fma2(p, pf2, big), x[0], x[1]);
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const uint32_t d = __float_as_uint(x[i]) ^ 0x8080u;
#pragma unroll
              for (int b = 0; b < 3; b++) {
                const int row = ((b * R) & 7) + r + i;  // rb is a multiple of 8
                // (byte 2's highest bit is the exponent's lowest, which is 0)
                bp_mine[b][((row >> 3) * 128 + (row & 7) * 16) - ((b * R) & 7) * 16] = (unsigned char)(d >> (8 * b));
              }
            }
          }
        }
        fence_async_smem();
        tc_fence_before();
        bar_all();
        if (tid == 0) {
          mbar_arrive(&sm.empty_k[k]);  // its scores are done, and every thread has its scales
          ka_wait(&sm.full_v[k], (n / STAGES) & 1, &sm.fail);
          tc_fence_after();
          const uint32_t a = ring_a + k * S::VSTAGE;
#pragma unroll
          for (int i = 0; i < KA_TILE / 32; i++)
            tc_mma_acc(tm + S::COL_O, tc_desc(a + i * 32 * HD, 16 * HD, 128, 0),
                       tc_desc(bp_a + i * 2 * S::PITCH, S::PITCH, 128, 0), IDESC_O, i > 0);
          tc_commit(&sm.obar);
          if (tile > u.lo) {  // the next tile's scores meanwhile
            ka_wait(&sm.full_k[(n + 1) % STAGES], ((n + 1) / STAGES) & 1, &sm.fail);
            issue_scores((n + 1) % STAGES);
          }
        }
        __syncwarp();
      }
      if (u.lo < last) add_out(n - 1);
      // ---- the unit's (or its share's) end ----
      float ls[RT], sums[RT];
#pragma unroll
      for (int r = 0; r < RT; r += 2) {
        unpack2(l[r / 2], ls[r], ls[r + 1]);
        unpack2(acc[r / 2], sums[r], sums[r + 1]);
      }
      const float mine = warp_sums(ls);
      if (lane < RT) sm.wmax[quad][rb + lane] = mine;
      bar_group();
      const bool from0 = A.cl ? A.cl == 1 : t <= u.u0 + A.take, to_end = u.next <= end;
      // where a share's sums go: of a cluster to its own shared memory (the ring is done with)
      float* part = A.cl ? reinterpret_cast<float*>(ka_raw) : A.part + ((size_t)cta * 2 + (from0 ? 1 : 0)) * R * (HD + 2);
      float* out = A.out + ((size_t)(u.sp.r0 + u.j0) * A.nh + u.kvh * A.g) * HD + ti;
#pragma unroll
      for (int r = 0; r < RT; r++) {
        const int row = rb + r;
        float tot = (sm.wmax[0][row] + sm.wmax[1][row]) + (sm.wmax[2][row] + sm.wmax[3][row]);
        if (sm.lim[row] < 0) tot = 0.0f;
        if (from0 && to_end) {
          if (sm.node[row] < u.nodes && ti < HD) out[sm.off[row] * HD] = tot == 0.0f ? 0.0f : __fdiv_rn(sums[r] * KA_UNIT, tot);
        } else {
          if (ti < HD) part[row * HD + ti] = sums[r];
          if (ti == 0) {
            part[R * HD + row] = sm.m[(n + 1) & 1][row];
            part[R * HD + R + row] = tot;
          }
        }
      }
      if (A.cl && tid == 0) sm.first_row = u.sp.r0 + u.j0, sm.kvh = u.kvh, sm.nodes = u.nodes;
      if (from0 && !to_end && tid == 0) {
        // this CTA's share is the first: the join goes on to the CTA that holds the unit's last tile
        const int lt = u.next - 1;
        A.head[cta] = make_int4(u.sp.r0 + u.j0, u.kvh, u.nodes, (int)((((long long)lt + 1) * G - 1) / T));
      }
      bar_all();
      t = u.next;
    }
    if (tid == 0 && sm.fail && n > 0) {  // waits were cut short: the last tile's MMAs (bounded)
      mbar_wait(&sm.sbar, (n - 1) & 1);
      mbar_wait(&sm.obar, (n - 1) & 1);
    }
  }
  if (A.cl > 1) {
    // ---- the unit's shares, each in its CTA's shared memory: row r by CTA r % cl, in tile order ----
    cg::this_cluster().sync();
    const int i = tid % HD;
    if (tid < S::COMPUTE) {
      for (int r = blockIdx.x % A.cl + A.cl * (tid / HD); r < R; r += A.cl * (S::COMPUTE / HD)) {
        if (sm.node[r] >= sm.nodes) continue;
        float m[KA_CLUSTER], l[KA_CLUSTER], v[KA_CLUSTER], mx = KA_NONE, o = 0.0f, tot = 0.0f;
#pragma unroll
        for (int c = 0; c < KA_CLUSTER; c++) {
          const float* p = cg::this_cluster().map_shared_rank(reinterpret_cast<const float*>(ka_raw), min(c, A.cl - 1));
          m[c] = c < A.cl ? p[R * HD + r] : KA_NONE;
          l[c] = c < A.cl ? p[R * HD + R + r] : 0.0f;
          v[c] = c < A.cl ? p[r * HD + i] : 0.0f;
        }
#pragma unroll
        for (int c = 0; c < KA_CLUSTER; c++) mx = fmaxf(mx, m[c]);
#pragma unroll
        for (int c = 0; c < KA_CLUSTER; c++) {
          const float f = ex2(m[c] - mx);
          o = __fmaf_rn(v[c], f, o);
          tot = __fmaf_rn(l[c], f, tot);
        }
        A.out[((size_t)sm.first_row * A.nh + sm.kvh * A.g + sm.off[r]) * HD + i] = tot == 0.0f ? 0.0f : __fdiv_rn(o * KA_UNIT, tot);
      }
    }
    cg::this_cluster().sync();  // nobody leaves while its shared memory is read
  }
  // ---- wind-down: every MMA was waited for; free the columns ----
  tc_fence_before();
  __syncthreads();
  if (warp == COPY)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(S::COLS));
  if (tid == 0 && sm.fail) kv8_flag(A.R.err, HG_ERR_TIMEOUT);
}

// The partial results of a unit whose tiles lie in several CTAs, added up in a fixed order: one CTA per
// first share and `rows` rows (1 or 4). Latency is all it costs. A row of many shares is split over four
// warps, each with eight shares' loads in flight at a time, that meet in shared memory; of few shares,
// each warp takes a row of the four. A lane has HD / 32 dims of a row.
constexpr int KA_STRANDS = 4, KA_BATCH = 8;
template <int HD, int R>
__global__ void __launch_bounds__(KA_STRANDS * 32) k_kv8_join(const __grid_constant__ KaArgs A, int rows) {
  constexpr int E = HD / 32;
  struct __align__(4 * E) Dims { float d[E]; };
  __shared__ float ms[KA_STRANDS], ls[KA_STRANDS];
  __shared__ Dims os[KA_STRANDS][32];
  pdl_wait();
  pdl_trigger();
  const int c0 = blockIdx.x, i = threadIdx.x, strand = threadIdx.y;
  const int4 h = A.head[c0];
  if (h.x < 0) return;
  constexpr int P = R * (HD + 2);
  const int n = h.w - c0 + 1;  // shares: the first in CTA c0's second place, the others in the first place
  // shares s0, s0 + step, ... of row r
  auto add = [&](int r, int s0, int step, float& mx, Dims& o, float& tot) {
    mx = KA_NONE;
    o = Dims{};
    tot = 0.0f;
    for (; s0 < n; s0 += step * KA_BATCH) {
      float m[KA_BATCH], l[KA_BATCH];
      Dims v[KA_BATCH];
#pragma unroll
      for (int b = 0; b < KA_BATCH; b++) {
        const int s = s0 + b * step, at = min(s, n - 1);
        const float* p = A.part + ((size_t)(c0 + at) * 2 + (at == 0 ? 1 : 0)) * P;
        m[b] = s < n ? p[R * HD + r] : KA_NONE;
        l[b] = s < n ? p[R * HD + R + r] : 0.0f;
        v[b] = s < n ? reinterpret_cast<const Dims*>(p + r * HD)[i] : Dims{};
      }
      float up = mx;
#pragma unroll
      for (int b = 0; b < KA_BATCH; b++) up = fmaxf(up, m[b]);
      const float al = ex2(mx - up);
#pragma unroll
      for (int e = 0; e < E; e++) o.d[e] *= al;
      tot *= al;
      mx = up;
#pragma unroll
      for (int b = 0; b < KA_BATCH; b++) {
        const float f = ex2(m[b] - mx);
#pragma unroll
        for (int e = 0; e < E; e++) o.d[e] = __fmaf_rn(v[b].d[e], f, o.d[e]);
        tot = __fmaf_rn(l[b], f, tot);
      }
    }
  };
  auto put = [&](int r, Dims o, float tot) {
    const int node = r / A.g;
#pragma unroll
    for (int e = 0; e < E; e++) o.d[e] = tot == 0.0f ? 0.0f : __fdiv_rn(o.d[e] * KA_UNIT, tot);
    reinterpret_cast<Dims*>(A.out + ((size_t)(h.x + node) * A.nh + h.y * A.g + r - node * A.g) * HD)[i] = o;
  };
  const int have = h.z * A.g;  // rows of the block
  float mx, tot;
  Dims o;
  if (rows > 1 && n <= KA_BATCH) {
    const int r = blockIdx.y * rows + strand;
    if (r >= have) return;
    add(r, 0, 1, mx, o, tot);
    put(r, o, tot);
    return;
  }
  for (int r = blockIdx.y * rows; r < min(have, (int)(blockIdx.y + 1) * rows); r++) {
    add(r, strand, KA_STRANDS, mx, o, tot);
    __syncthreads();
    os[strand][i] = o;
    if (i == 0) ms[strand] = mx, ls[strand] = tot;
    __syncthreads();
    if (strand != 0) continue;
#pragma unroll
    for (int k = 1; k < KA_STRANDS; k++) mx = fmaxf(mx, ms[k]);
    o = Dims{};
    tot = 0.0f;
#pragma unroll
    for (int k = 0; k < KA_STRANDS; k++) {
      const float f = ex2(ms[k] - mx);
#pragma unroll
      for (int e = 0; e < E; e++) o.d[e] = __fmaf_rn(os[k][i].d[e], f, o.d[e]);
      tot = __fmaf_rn(ls[k], f, tot);
    }
    put(r, o, tot);
  }
}

// ---- host ----
namespace {

void check_attn(const hg_kv8_cache* c, const hg_rows* r, int n_heads) {
  kv8_check_cache(c);
  kv8_check_rows(r, true);
  kv8_need(n_heads > 0 && n_heads % c->n_kv_heads == 0, "bad head counts");
  kv8_need(n_heads / c->n_kv_heads <= KV8_MAX_GROUP, "more than 32 q heads per kv head");
}

// Rows of a block: 4, 8, 16 or 32, whichever makes a ragged batch cheapest. A block's cost, the mean of
// the call's time per block at 64 and at 256 rows a kv head (32 sequences of 900 to 7000 slots, 12 q
// heads, 3 kv heads, 128 dims; us): 11.7, 13.8, 23.3 and 36.7. The whole calls took 752, 433, 363 and 267
// us at 256 rows, 31.1, 28.4, 34.0 and 48.0 us with the one block that the size just fills. (64 dims: by
// assumption the same.) The
// sequences' row counts lie between 1 and max_rows; they are taken as spread evenly around their mean.
int block_rows(const hg_rows* r, int g) {
  const double hi = std::min(r->max_rows, r->n_rows), mean = std::min(hi, (double)r->n_rows / r->n_seqs);
  const double lo = std::min(hi, std::max(1.0, 2 * mean - hi));
  constexpr double pass[4] = {11.7, 13.8, 23.3, 36.7};
  double least = 0.0;
  int best = 0;
  for (int i = 0; i < 4; i++) {
    const int R = 4 << i, npb = R / g;
    if (npb == 0) continue;
    double cost = 0.0;
    for (int k = 0; k < 8; k++) cost += std::ceil(std::round(lo + (hi - lo) * (k + 0.5) / 8) / npb) * pass[i];
    if (best == 0 || cost < least) best = R, least = cost;
  }
  return best;
}

size_t part_bytes(int R, int hd) { return (size_t)KA_MAX_CTAS * 2 * R * (hd + 2) * 4; }
// scratch for any rows: the largest block has the fewest CTAs
size_t scratch_bytes(int hd) { return part_bytes(32, hd) / KA_MAX_CTAS * 2 * KA_SMS + KA_MAX_CTAS * sizeof(int4); }

template <int HD, int R>
void launch(KaArgs& A, int device, double units, cudaStream_t st) {
  using S = KaShape<HD, R>;
  const size_t smem = S::OFF_SMALL + sizeof(KaSmall<R>) + (A.R.n_seqs + 1) * sizeof(uint32_t);
  constexpr size_t most = S::OFF_SMALL + sizeof(KaSmall<R>) + (KV8_MAX_SEQS + 1) * sizeof(uint32_t);
  kv8_smem_limit(k_kv8_attn<HD, R>, device, most);
  const int per_sm = (int)std::min<size_t>(std::min(3, 512 / S::COLS), (228 * 1024) / (smem + 1024));
  const int resident = KA_SMS * per_sm;
  // A unit per cluster, joined in it, where a table's row of pages makes so few tiles that a CTA gets
  // three at most: one launch instead of two.
  const int tiles = (A.C.bt_stride + KA_PAGES - 1) / KA_PAGES;
  int cl = 1;
  while (cl < KA_CLUSTER && tiles > 2 * cl && units * 2 * cl <= KA_SMS) cl *= 2;
  A.cl = tiles <= 3 * cl && units * cl <= resident ? cl : 0;
  // one CTA per place on the line is the most that can have work
  const int ctas = A.cl ? (int)units * A.cl : (int)std::min((double)resident, units * (tiles + A.take));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(S::THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = A.cl;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = A.cl > 1 ? 2 : 1;
  kv8_launched(cudaLaunchKernelEx(&cfg, k_kv8_attn<HD, R>, A));
  if (A.cl) return;
  // few places: latency, a CTA per row; many: four rows each, so that most find their share's row at once
  const int rows = ctas < resident ? 1 : 4;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3(ctas, (A.g * A.npb + rows - 1) / rows);
  cfg.blockDim = dim3(32, KA_STRANDS);
  cfg.dynamicSmemBytes = 0;
  kv8_launched(cudaLaunchKernelEx(&cfg, k_kv8_join<HD, R>, A, rows));
}

}  // namespace
}  // namespace hg

using namespace hg;

extern "C" size_t hg_op_kv8_attn_scratch_bytes(const hg_kv8_cache* c, const hg_rows* r, int n_heads) {
  try {
    check_attn(c, r, n_heads);
    return scratch_bytes(c->head_dim);
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
    A.take = ka_take(R);
    // the most units that ragged rows make; places on the line are numbered with 32 bits
    const double blocks = std::min(std::floor((double)r->n_rows / A.npb) + r->n_seqs,
                                   (double)r->n_seqs * ((std::min(r->max_rows, r->n_rows) + A.npb - 1) / A.npb));
    const double units = blocks * c->n_kv_heads, places = units * ((c->bt_stride + KA_PAGES - 1) / KA_PAGES + A.take);
    kv8_need(places < 2147483647.0, "rows x table entries x kv heads out of range for one call");
    A.q = q;
    A.out = out;
    A.head = static_cast<int4*>(scratch);
    A.part = reinterpret_cast<float*>(A.head + KA_MAX_CTAS);
    Kv8Device dev(c->pool);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const int d = dev.device;
    if (c->head_dim == 64) {
      if (R == 4) launch<64, 4>(A, d, units, st);
      else if (R == 8) launch<64, 8>(A, d, units, st);
      else if (R == 16) launch<64, 16>(A, d, units, st);
      else launch<64, 32>(A, d, units, st);
    } else {
      if (R == 4) launch<128, 4>(A, d, units, st);
      else if (R == 8) launch<128, 8>(A, d, units, st);
      else if (R == 16) launch<128, 16>(A, d, units, st);
      else launch<128, 32>(A, d, units, st);
    }
  })
}
