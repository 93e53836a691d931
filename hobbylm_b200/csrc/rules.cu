// Rules on a batch of logit rows (hg_op_logits_rules): penalties for ids that occurred, biases, the id
// bound and grammar masks, with a greedy pick per row.
//
// Bound by the row's bytes: 4 read and 4 written per id. Only ids in the row's lists need more than a mask
// bit, some hundreds of fifty thousand. A word per id in shared memory holds its occurrences and flags;
// the first list entry to claim an id's word puts it on a work list, from which it is gathered, worked on
// and written, and the stream over the row passes it by. The two touch different ids, so nothing waits
// between them: an id that occurs often, whose roundings wait for one another, holds up one warp.
//
// A row is one cluster of 1, 2, 4 or 8 CTAs, each with a run of its ids in chunks. Words have 16 bits,
// and 32 where the lists are long enough for a count to need them. Occurrences are counted with integer
// atomics, whose order does not matter. Lists are read four entries a thread at a time, before the run is
// asked for (behind it they took twice as long). The arithmetic per id is Engine::generate's (sampler.cpp,
// lib.rs:130-139): one f32 rounding per occurrence, so a pick equals the engine's own.
//
// 256 rows of 50304 ids with histories of up to 2000 ids and up to 300 biases take 44 us, of which the
// bytes need 16: all CTAs run at once, each through its lists (some 12 us of loads and atomics that wait
// for one another) and then its stream (about the 16), and too few rows follow to fill the one with the
// other. The same rows without lists take 27 us. Smaller CTAs (runs of an eighth), more of them an SM (48
// registers) and eight list entries a thread were slower.
#include <cooperative_groups.h>

#include <algorithm>

#include "hg_kv8.cuh"

namespace hg {

namespace cg = cooperative_groups;

constexpr int LR_THREADS = 256;
constexpr int LR_CHUNK = 25216;            // most ids of a chunk with 16-bit words (half as many with 32): half a
                                           // row of 50304, four CTAs of which fit an SM
constexpr int LR_SPARE = 32;               // bytes behind the words that whole lines reach into
constexpr int LR_LONG = 1 << 13;           // occurrences that a 16-bit word's 13 bits do not hold
constexpr int LR_PATH = 256;               // drafted tokens of a path in hand at a time
constexpr int LR_AHEAD = 4;                // 16-byte lines of a thread in flight
constexpr int LR_BATCH = 4;                // list entries of a thread in flight
constexpr int LR_WORK = 256;               // entries of a work list; what does not fit is done where it is claimed
constexpr int LR_OFTEN = 8;                // occurrences from which an id is for the warp that does those

// The sequence that a row belongs to (-1: none): every thread of the block gets it.
__device__ __forceinline__ int rules_seq(const hg_rows& R, int row) {
  int s = 0;
  for (int i0 = 0; i0 < R.n_seqs; i0 += LR_THREADS) {
    const int i = i0 + threadIdx.x;
    s += __syncthreads_count(i < R.n_seqs && R.row_off[i + 1] <= row);
  }
  return s < R.n_seqs ? s : -1;
}

// l after c occurrences: l / rep each while l > 0, else l * rep, every step rounded to f32
// (lib.rs:130-139). The steps wait for one another, so a quotient takes five dependent fused
// multiply-adds: y = RN(1 / rep), two refinements q += (l - q rep) y; after the first q is within an ulp,
// and then the second is the correctly rounded quotient (Markstein, "Computation of elementary functions
// on the IBM RISC System/6000 processor", 1990), as long as nothing comes near under- or overflow:
// checked every four steps, which change l by at most 2^16. Not inlined: one copy of it.
__device__ __noinline__ float rules_repeat(float l, float rep, int c) {
  int n = 0;
  if (rep >= 0.0625f && rep <= 16.0f) {
    if (l > 0.0f) {
      const float y = __frcp_rn(rep);
      for (; n < c && l > 8.6736174e-19f && l < 1.1529215e18f; n += 4) {  // 2^-60, 2^60
#pragma unroll
        for (int k = 0; k < 4; k++) {
          float q = __fmul_rn(l, y);
          q = __fmaf_rn(__fmaf_rn(-q, rep, l), y, q);
          q = __fmaf_rn(__fmaf_rn(-q, rep, l), y, q);
          if (n + k < c) l = q;
        }
      }
    } else {
      for (; n < c; n += 4) {
#pragma unroll
        for (int k = 0; k < 4; k++)
          if (n + k < c) l = __fmul_rn(l, rep);
      }
    }
  }
#pragma unroll 1
  for (; n < c; n++) {
    const float p = l > 0.0f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
    if (p == l) break;  // zero, infinity or the least subnormal: stays
    l = p;
  }
  return l;
}

// Words of a chunk's ids: 16 bits each, two to a 32-bit word, or 32. The three highest bits are flags.
template <bool WIDE>
struct RuleWords {
  static constexpr int BITS = WIDE ? 32 : 16;
  static constexpr uint32_t ALL = WIDE ? 0xffffffffu : 0xffffu;
  static constexpr uint32_t BIASED = 1u << (BITS - 1);   // the id has a bias
  static constexpr uint32_t TWICE = 1u << (BITS - 2);    // more than one entry of it
  static constexpr uint32_t CLAIMED = 1u << (BITS - 3);  // an entry does the id
  uint32_t* w;
  __device__ __forceinline__ uint32_t* at(int d) const { return w + (WIDE ? d : d >> 1); }
  __device__ __forceinline__ int shift(int d) const { return WIDE ? 0 : (d & 1) * 16; }
  __device__ __forceinline__ void count(int d) { atomicAdd(at(d), 1u << shift(d)); }
  // sets flags of the id's word and returns what it was
  __device__ __forceinline__ uint32_t set(int d, uint32_t flags) {
    return (atomicOr(at(d), flags << shift(d)) >> shift(d)) & ALL;
  }
  __device__ __forceinline__ uint32_t get(int d) const {
    return WIDE ? w[d] : reinterpret_cast<const uint16_t*>(w)[d];
  }
  // whether any of the four ids from d on (d a multiple of 4) is listed
  __device__ __forceinline__ bool four(int d) const {
    if (WIDE) {
      const uint4 v = *reinterpret_cast<const uint4*>(w + d);
      return (v.x | v.y | v.z | v.w) != 0;
    }
    const uint2 v = *reinterpret_cast<const uint2*>(w + d / 2);
    return (v.x | v.y) != 0;
  }
};

// A row as its CTAs see it.
struct RulesRow {
  const float* in;
  float* out;
  const uint32_t* mask;
  const int32_t *hist, *bias_id, *token;  // token: of the sequence's first row, or null
  const float* bias;
  int hn, bn, j, valid;
  float rep, freq, pres;
  SeqSpan sp;
};
struct RulesShared {
  int2 often[LR_WORK], once[LR_WORK];  // work lists: id, occurrences
  int often_n, once_n;
  int path[LR_PATH], path_n, path_at;
  unsigned long long red[LR_THREADS / 32], best[8];
};

// One CTA's ids lo .. hi - 1 of a row, with room for the 16-bit words of `room` ids (even); returns the thread's greatest as an argmax key.
template <bool VEC, bool WIDE>
__device__ __forceinline__ unsigned long long rules_run(const hg_rows& R, const RulesRow& A, RulesShared& sh,
                                                        uint32_t* words_s, int room, int lo, int hi) {
  using Words = RuleWords<WIDE>;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float* in = A.in;
  float* out = A.out;
  const uint32_t* mask = A.mask;
  const int valid = A.valid, bn = A.bn;
  const bool in_place = in == out;
  const bool counts = (A.hn > 0 || A.token) && (A.rep != 1.0f || A.freq != 0.0f || A.pres != 0.0f), listed = counts || bn > 0;
  const int lines = VEC ? (int)((reinterpret_cast<uintptr_t>(in) >> 2) & 3) : 0;  // floats before the row in its first line
  unsigned long long best = 0ull;
  Words words{words_s};

  auto allowed = [&](int i) { return i < valid && (!mask || (__ldg(mask + (i >> 5)) >> (i & 31)) & 1u); };
  // id i's logit after c occurrences
  auto penalised = [&](int i, int c) -> float {
    float l = in[i];
    if (c > 0) {
      if (A.rep != 1.0f) l = rules_repeat(l, A.rep, c);
      l = __fsub_rn(__fsub_rn(l, __fmul_rn(A.freq, (float)c)), A.pres);
    }
    return l;
  };
  auto finish = [&](int i, float l) {
    if (!allowed(i)) l = -INFINITY;
    out[i] = l;
    if (l > -INFINITY) best = max(best, argmax_key(l, (uint32_t)i));  // false for NaN
  };
  // f(ids) for a list of n ids, LR_BATCH of them per thread at a time (-1 past its end), whole warps
  auto each_id = [&](const int32_t* list, int n, auto f) {
    for (int i0 = 0; i0 < n; i0 += LR_BATCH * LR_THREADS) {
      int id[LR_BATCH];
#pragma unroll
      for (int k = 0; k < LR_BATCH; k++) {
        const int i = i0 + k * LR_THREADS + tid;
        id[k] = i < n ? list[i] : -1;
      }
      f(id);
    }
  };
  // the same for the history and the drafted tokens on the row's path
  auto each_counted = [&](auto f) {
    each_id(A.hist, A.hn, f);
    if (!A.token) return;
    if (!R.parent) {
      each_id(A.token, A.j + 1, f);
      return;
    }
    for (int at = A.j; at >= 0;) {  // the same for every thread
      __syncthreads();
      if (warp == 0) {
        int n = 0, up = at;
        while (up >= 0 && n + 32 <= LR_PATH) {
          const PathRun run = kv8_run<32>(R, A.sp, up);
          if (lane < run.len) sh.path[n + lane] = A.token[up - lane];
          n += run.len;
          up = run.next;
        }
        if (lane == 0) sh.path_n = n, sh.path_at = up;
      }
      __syncthreads();
      at = sh.path_at;
      each_id(sh.path, sh.path_n, f);
    }
  };

  const int chunk = WIDE ? room / 2 : room;
  for (int c0 = lo; c0 < hi; c0 += chunk) {
    // id i's word is number i - c1, so that a line of the row has its words together; c1 <= c0
    const int n = min(chunk, hi - c0), c1 = c0 - ((c0 + lines) & 3);
    // whole lines: ids ia .. ib - 1; at most three ids stand before and three behind them
    const int ia = VEC ? min(c0 + n, c1 + (c1 < c0 ? 4 : 0)) : c0 + n, ib = ia + (c0 + n - ia) / 4 * 4;
    auto inside = [&](int id) { return (uint32_t)id - (uint32_t)c0 < (uint32_t)n; };
    if (listed) {
      __syncthreads();
      if (tid == 0) sh.often_n = sh.once_n = 0;
      for (int i = tid * 4; i < (WIDE ? n + 4 : (n + 4) / 2 + 1); i += LR_THREADS * 4)
        *reinterpret_cast<uint4*>(words_s + i) = make_uint4(0, 0, 0, 0);
      __syncthreads();
      if (counts)
        each_counted([&](const int (&id)[LR_BATCH]) {
#pragma unroll
          for (int k = 0; k < LR_BATCH; k++)
            if (inside(id[k])) words.count(id[k] - c1);
        });
      each_id(A.bias_id, bn, [&](const int (&id)[LR_BATCH]) {
#pragma unroll
        for (int k = 0; k < LR_BATCH; k++)
          if (inside(id[k]) && words.set(id[k] - c1, Words::BIASED) & Words::BIASED) words.set(id[k] - c1, Words::TWICE);
      });
      __syncthreads();
      // ---- each listed id to one entry: one with a bias to an entry of the biases, else to a work list ----
      if (counts) {
        each_counted([&](const int (&id)[LR_BATCH]) {
#pragma unroll
          for (int k = 0; k < LR_BATCH; k++) {
            int c = 0;
            if (inside(id[k]) && !(words.get(id[k] - c1) & Words::BIASED)) {
              const uint32_t w = words.set(id[k] - c1, Words::CLAIMED);
              if (!(w & Words::CLAIMED)) c = (int)(w & (Words::CLAIMED - 1));
            }
            const unsigned a = __ballot_sync(0xffffffffu, c >= LR_OFTEN), b = __ballot_sync(0xffffffffu, c > 0 && c < LR_OFTEN);
            if (a | b) {
              int at = 0;
              if (lane < 2 && (lane ? b : a)) at = atomicAdd(lane ? &sh.once_n : &sh.often_n, __popc(lane ? b : a));
              const unsigned mine = c >= LR_OFTEN ? a : b;
              at = __shfl_sync(0xffffffffu, at, c >= LR_OFTEN ? 0 : 1) + __popc(mine & ((1u << lane) - 1));
              if (c > 0) {
                if (at < LR_WORK) (c >= LR_OFTEN ? sh.often : sh.once)[at] = make_int2(id[k], c);
                else finish(id[k], penalised(id[k], c));
              }
            }
          }
        });
        __syncthreads();
        if (VEC && tid == 0 && ib > ia)  // the run on its way to the L2 cache while the listed ids are worked on
          asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(in + ia), "r"((ib - ia) * 4) : "memory");
        const bool last = warp == LR_THREADS / 32 - 1;  // the warp for the ids that occur often
        const int2* list = last ? sh.often : sh.once;
        const int have = min(last ? sh.often_n : sh.once_n, LR_WORK);
#pragma unroll 1
        for (int k = last ? lane : tid; k < have; k += last ? 32 : LR_THREADS - 32)
          finish(list[k].x, penalised(list[k].x, list[k].y));
      }
#pragma unroll 1
      for (int i = tid; i < bn; i += LR_THREADS) {
        const int id = A.bias_id[i];
        if (!inside(id)) continue;
        const uint32_t w = words.set(id - c1, Words::CLAIMED);
        if (w & Words::CLAIMED) continue;
        float b = A.bias[i];
        if (w & Words::TWICE) {  // the entries of the id, added up in the list's order
          b = 0.0f;
          for (int e = 0; e < bn; e++)
            if (A.bias_id[e] == id) b = __fadd_rn(b, A.bias[e]);
        }
        finish(id, __fadd_rn(penalised(id, (int)(w & (Words::CLAIMED - 1))), b));
      }
    }
    // ---- the stream: all other ids ----
    float top = -INFINITY;
    int top_id = -1;
    auto pass = [&](float l, int i, bool ok) -> float {
      if (!ok) l = -INFINITY;
      if (l > top) top = l, top_id = i;  // a thread's ids ascend: the first of equals stays
      return l;
    };
    auto single = [&](int i) {
      if (!(listed && words.get(i - c1))) out[i] = pass(in[i], i, allowed(i));
    };
#pragma unroll 1
    for (int i = c0 + tid; i < (VEC ? ia : c0 + n); i += LR_THREADS) single(i);
    if (VEC) {
#pragma unroll 1
      for (int i0 = ia + tid * 4; i0 < ib; i0 += LR_AHEAD * LR_THREADS * 4) {
        float4 x[LR_AHEAD];
        uint32_t may[LR_AHEAD];
#pragma unroll
        for (int k = 0; k < LR_AHEAD; k++) {
          const int i = min(i0 + k * LR_THREADS * 4, ib - 4);  // past the end: the last line again, not used
          x[k] = *reinterpret_cast<const float4*>(in + i);
        }
#pragma unroll
        for (int k = 0; k < LR_AHEAD; k++) may[k] = 15u;
        if (mask) {
          uint32_t m1[LR_AHEAD];
#pragma unroll
          for (int k = 0; k < LR_AHEAD; k++) {
            const int i = min(i0 + k * LR_THREADS * 4, ib - 4);
            may[k] = __ldg(mask + (i >> 5));
            m1[k] = __ldg(mask + ((i + 3) >> 5));  // a line may have its bits in two words
          }
#pragma unroll
          for (int k = 0; k < LR_AHEAD; k++) may[k] = __funnelshift_r(may[k], m1[k], i0 + k * LR_THREADS * 4) & 15u;
        }
#pragma unroll
        for (int k = 0; k < LR_AHEAD; k++) {
          const int i = i0 + k * LR_THREADS * 4;
          if (i >= ib) break;
          if (i + 4 > valid) may[k] &= (1u << max(valid - i, 0)) - 1u;
          const float l[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
          if (listed && words.four(i - c1)) {
#pragma unroll
            for (int e = 0; e < 4; e++)
              if (!words.get(i - c1 + e)) out[i + e] = pass(l[e], i + e, (may[k] >> e) & 1u);
          } else {
            const float4 v = make_float4(pass(l[0], i, may[k] & 1u), pass(l[1], i + 1, may[k] & 2u),
                                         pass(l[2], i + 2, may[k] & 4u), pass(l[3], i + 3, may[k] & 8u));
            if (!in_place || may[k] != 15u) *reinterpret_cast<float4*>(out + i) = v;
          }
        }
      }
      if (ib + tid < c0 + n) single(ib + tid);
    }
    if (top_id >= 0) best = max(best, argmax_key(top, (uint32_t)top_id));
  }
  return best;
}

// VEC: logits and out lie alike in their 16-byte lines, so that a row moves in whole ones.
template <bool VEC>
__global__ void __launch_bounds__(LR_THREADS, 4) k_logits_rules(const __grid_constant__ hg_rows R,
                                                               const __grid_constant__ hg_logits_rules_args A, int nc,
                                                               int per, int room) {
  extern __shared__ __align__(16) uint32_t words_s[];
  __shared__ RulesShared sh;
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / nc, part = blockIdx.x - row * nc;
  const int s = rules_seq(R, row);
  if (s < 0) return;  // behind the last sequence (the whole cluster leaves)
  RulesRow w;
  const int h0 = A.hist_off ? A.hist_off[s] : 0, b0 = A.bias_off ? A.bias_off[s] : 0;
  // below 0 (no entries) where the offsets descend or are below 0 themselves
  w.hn = A.hist_off ? (int)((uint32_t)A.hist_off[s + 1] - (uint32_t)h0) | h0 >> 31 : 0;
  w.bn = A.bias_off ? (int)((uint32_t)A.bias_off[s + 1] - (uint32_t)b0) | b0 >> 31 : 0;
  w.rep = A.rep_penalty ? A.rep_penalty[s] : 1.0f;
  w.freq = A.freq_penalty ? A.freq_penalty[s] : 0.0f;
  w.pres = A.pres_penalty ? A.pres_penalty[s] : 0.0f;
  const int mr = A.mask ? (A.mask_row ? A.mask_row[row] : row) : -1;
  w.sp = kv8_span(R, s, false);
  w.j = row - w.sp.r0;
  if (w.j < 0 || w.j >= w.sp.n) return;
  if (R.parent && R.parent[row] <= -2) {
    if (A.next_ids && part == 0 && tid == 0) A.next_ids[row] = -1;
    return;
  }
  if (A.next_ids) cg::cluster_group::barrier_arrive();  // every CTA of the row has started: see below
  w.in = A.logits + (size_t)row * A.ld;
  w.out = A.out + (size_t)row * A.ld_out;
  w.mask = mr >= 0 ? A.mask + (size_t)mr * A.mask_words : nullptr;
  w.hist = A.hist + h0;
  w.bias_id = A.bias_id + b0;
  w.bias = A.bias + b0;
  w.token = A.token ? A.token + w.sp.r0 : nullptr;
  w.valid = A.valid > 0 ? min(A.valid, A.vocab) : A.vocab;
  const int lo = part * per, hi = min(A.vocab, lo + per);
  unsigned long long best = (long long)max(w.hn, 0) + w.j + 1 < LR_LONG ? rules_run<VEC, false>(R, w, sh, words_s, room, lo, hi)
                                                               : rules_run<VEC, true>(R, w, sh, words_s, room, lo, hi);
  if (tid == 0 && (w.hn | w.bn) < 0) kv8_flag(R.err, HG_ERR_INVALID);
  if (!A.next_ids) return;
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) sh.red[warp] = best;
  __syncthreads();
  if (tid == 0)
    for (int k = 1; k < LR_THREADS / 32; k++) best = max(best, sh.red[k]);
  cg::cluster_group::barrier_wait();  // CTA 0's shared memory is there to be written
  if (tid == 0) cg::this_cluster().map_shared_rank(sh.best, 0)[part] = best;
  cg::this_cluster().sync();
  if (part == 0 && tid == 0) {
    for (int c = 0; c < nc; c++) best = max(best, sh.best[c]);
    A.next_ids[row] = best ? (int32_t)(0xffffffffu - (uint32_t)best) : -1;
  }
}

}  // namespace hg

using namespace hg;

extern "C" int hg_op_logits_rules(const hg_rows* r, const hg_logits_rules_args* args, void* stream) {
  KV8_API({
    kv8_check_rows(r, false);
    kv8_need(args, "null argument");
    hg_logits_rules_args a = *args;
    kv8_need(a.vocab > 0 && a.vocab <= INT_MAX - 65536, "vocab out of range");
    if (a.ld == 0) a.ld = a.vocab;
    if (a.ld_out == 0) a.ld_out = a.vocab;
    kv8_need(a.ld >= a.vocab && a.ld_out >= a.vocab, "row strides must hold a row");
    kv8_need(a.logits && a.out, "null argument");
    kv8_need(a.logits != a.out || a.ld == a.ld_out, "in place, both row strides must be the same");
    kv8_need(!a.hist_off || a.hist, "null argument");
    kv8_need(!a.bias_off || (a.bias_id && a.bias), "null argument");
    kv8_need(!a.mask || a.mask_words >= (a.vocab + 31) / 32, "mask_words does not hold a row of the mask");
    for (const void* p : {(const void*)a.logits, (const void*)a.out, (const void*)a.next_ids, (const void*)a.token,
                          (const void*)a.hist_off, (const void*)a.hist, (const void*)a.rep_penalty,
                          (const void*)a.freq_penalty, (const void*)a.pres_penalty, (const void*)a.bias_off,
                          (const void*)a.bias_id, (const void*)a.bias, (const void*)a.mask, (const void*)a.mask_row})
      kv8_need(kv8_aligned(p, 4), "arrays must be 4-byte aligned");
    if (r->n_seqs == 0 || r->n_rows == 0) return HG_OK;
    Kv8Device dev(a.logits);
    // CTAs per row: a run of one chunk each where eight will do, and enough for every SM if the runs stay
    // at 2048 ids or more
    int nc = 1;
    while (nc < 8 && (a.vocab > nc * LR_CHUNK || ((long long)r->n_rows * nc < 2 * 148 && a.vocab / (2 * nc) >= 2048))) nc *= 2;
    const int per = (a.vocab + nc - 1) / nc;
    // rows move in 16-byte lines where both lie alike in them
    const bool vec = a.ld % 4 == a.ld_out % 4 && ((uintptr_t)a.logits & 15) == ((uintptr_t)a.out & 15);
    auto kern = vec ? k_logits_rules<true> : k_logits_rules<false>;
    const int room = std::min((per + 1) / 2 * 2, LR_CHUNK);
    const size_t smem = (size_t)room * 2 + LR_SPARE;
    kv8_smem_limit(kern, dev.device, LR_CHUNK * 2 + LR_SPARE);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)r->n_rows * nc);
    cfg.blockDim = dim3(LR_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = nc;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    kv8_launched(cudaLaunchKernelEx(&cfg, kern, *r, a, nc, per, room));
  })
}
