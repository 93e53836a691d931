// Rules on a batch of logit rows (hg_op_logits_rules): penalties for ids that occurred, biases, the id
// bound and grammar masks, with a greedy pick per row.
//
// Bound by the row's bytes (4 read, 4 written per id). A row is one cluster of 1, 2, 4 or 8 CTAs, each
// with a run of its ids; a CTA walks its run in chunks that have an occurrence count and a bias per id
// in shared memory, so one pass over the logits applies everything. Each chunk reads the sequence's
// whole lists and keeps what falls into it. The arithmetic per id is Engine::generate's (sampler.cpp,
// lib.rs:130-139): one f32 rounding per occurrence, so a pick equals the engine's own.
#include <cooperative_groups.h>

#include "hg_kv8.cuh"

namespace hg {

namespace cg = cooperative_groups;

constexpr int LR_THREADS = 512;
constexpr int LR_CHUNK = 8192;  // ids of a chunk: 32 KB of counts and 32 KB of biases
constexpr size_t LR_SMEM = (size_t)LR_CHUNK * 8;

// The sequence that a row belongs to (-1: none): every thread of the block gets it.
__device__ __forceinline__ int rules_seq(const hg_rows& R, int row) {
  int s = 0;
  for (int i0 = 0; i0 < R.n_seqs; i0 += LR_THREADS) {
    const int i = i0 + threadIdx.x;
    s += __syncthreads_count(i < R.n_seqs && R.row_off[i + 1] <= row);
  }
  return s < R.n_seqs ? s : -1;
}

template <bool VEC>
__global__ void __launch_bounds__(LR_THREADS) k_logits_rules(hg_rows R, hg_logits_rules_args A, int nc, int per) {
  extern __shared__ __align__(16) unsigned char lr_raw[];
  int* cnt = reinterpret_cast<int*>(lr_raw);
  float* bias = reinterpret_cast<float*>(lr_raw) + LR_CHUNK;
  __shared__ unsigned long long red[LR_THREADS / 32], best_s[8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / nc, part = blockIdx.x - row * nc;
  const int s = rules_seq(R, row);
  if (s < 0) return;  // behind the last sequence (the whole cluster leaves)
  const SeqSpan sp = kv8_span(R, s, false);
  const int j = row - sp.r0;
  if (j < 0 || j >= sp.n) return;
  if (kv8_parent(R, sp, j) == -2) {
    if (A.next_ids && part == 0 && tid == 0) A.next_ids[row] = -1;
    return;
  }
  if (A.next_ids) cg::cluster_group::barrier_arrive();  // every CTA of the row has started: see below
  const float* in = A.logits + (size_t)row * A.ld;
  float* out = A.out + (size_t)row * A.ld_out;
  const float rep = A.rep_penalty ? A.rep_penalty[s] : 1.0f;
  const float freq = A.freq_penalty ? A.freq_penalty[s] : 0.0f, pres = A.pres_penalty ? A.pres_penalty[s] : 0.0f;
  const int h0 = A.hist_off ? A.hist_off[s] : 0, hn = A.hist_off ? A.hist_off[s + 1] - h0 : 0;
  const int b0 = A.bias_off ? A.bias_off[s] : 0, bn = A.bias_off ? A.bias_off[s + 1] - b0 : 0;
  const bool counts = (hn > 0 || A.token) && (rep != 1.0f || freq != 0.0f || pres != 0.0f);
  const int valid = A.valid > 0 ? min(A.valid, A.vocab) : A.vocab;
  const int mr = A.mask ? (A.mask_row ? A.mask_row[row] : row) : -1;
  const uint32_t* mask = mr >= 0 ? A.mask + (size_t)mr * A.mask_words : nullptr;
  unsigned long long best = 0ull;

  auto rule = [&](float l, int i, int k) -> float {  // id i, the chunk's entry k
    if (counts) {
      const int c = cnt[k];
      if (c > 0) {
        if (rep != 1.0f)
          for (int n = 0; n < c; n++) {
            const float p = l > 0.0f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
            if (p == l) break;  // zero or infinity: stays
            l = p;
          }
        l = __fsub_rn(l, __fmul_rn(freq, (float)c));
        l = __fsub_rn(l, pres);
      }
    }
    if (bn > 0) l = __fadd_rn(l, bias[k]);
    if (i >= valid || (mask && !((mask[i >> 5] >> (i & 31)) & 1u))) l = -INFINITY;
    if (l > -INFINITY) best = max(best, argmax_key(l, (uint32_t)i));  // false for NaN
    return l;
  };

  const int lo = part * per, hi = min(A.vocab, lo + per);
  for (int c0 = lo; c0 < hi; c0 += LR_CHUNK) {
    const int n = min(LR_CHUNK, hi - c0);
    __syncthreads();
    if (counts)
      for (int i = tid; i < n; i += LR_THREADS) cnt[i] = 0;
    if (bn > 0)
      for (int i = tid; i < n; i += LR_THREADS) bias[i] = 0.0f;
    __syncthreads();
    if (counts) {
      for (int i = tid; i < hn; i += LR_THREADS) {
        const unsigned d = (unsigned)A.hist[(size_t)h0 + i] - (unsigned)c0;
        if (d < (unsigned)n) atomicAdd(&cnt[d], 1);
      }
      if (A.token && !R.parent) {
        for (int i = tid; i <= j; i += LR_THREADS) {
          const unsigned d = (unsigned)A.token[sp.r0 + i] - (unsigned)c0;
          if (d < (unsigned)n) atomicAdd(&cnt[d], 1);
        }
      } else if (A.token && tid == 0) {
        for (int at = j; at >= 0;) {
          const int up = kv8_parent(R, sp, at);
          if (up == -2) break;
          const unsigned d = (unsigned)A.token[sp.r0 + at] - (unsigned)c0;
          if (d < (unsigned)n) atomicAdd(&cnt[d], 1);
          at = up;
        }
      }
    }
    if (bn > 0 && warp == LR_THREADS / 32 - 1) {
      // one warp, 32 entries at a time; entries of one id add up in the list's order
      for (int i0 = 0; i0 < bn; i0 += 32) {
        const int i = i0 + lane;
        const unsigned d = i < bn ? (unsigned)A.bias_id[(size_t)b0 + i] - (unsigned)c0 : 0xffffffffu;
        const bool mine = d < (unsigned)n;
        const float b = mine ? A.bias[(size_t)b0 + i] : 0.0f;
        const unsigned same = __match_any_sync(0xffffffffu, mine ? (int)d : -1 - lane);
        const int rank = __popc(same & ((1u << lane) - 1));
        const int most = __reduce_max_sync(0xffffffffu, rank);
        for (int k = 0; k <= most; k++) {
          if (mine && rank == k) bias[d] = __fadd_rn(bias[d], b);
          __syncwarp();
        }
      }
    }
    __syncthreads();
    if (VEC) {
      for (int k = tid * 4; k < n; k += LR_THREADS * 4) {
        const float4 x = *reinterpret_cast<const float4*>(in + c0 + k);
        float4 y;
        y.x = rule(x.x, c0 + k, k);
        y.y = rule(x.y, c0 + k + 1, k + 1);
        y.z = rule(x.z, c0 + k + 2, k + 2);
        y.w = rule(x.w, c0 + k + 3, k + 3);
        *reinterpret_cast<float4*>(out + c0 + k) = y;
      }
    } else {
      for (int k = tid; k < n; k += LR_THREADS) out[c0 + k] = rule(in[c0 + k], c0 + k, k);
    }
  }
  if (!A.next_ids) return;
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) red[warp] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < LR_THREADS / 32; w++) best = max(best, red[w]);
  }
  cg::cluster_group::barrier_wait();  // CTA 0's shared memory is there to be written
  if (tid == 0) {
    cg::this_cluster().map_shared_rank(best_s, 0)[part] = best;
  }
  cg::this_cluster().sync();
  if (part == 0 && tid == 0) {
    for (int c = 0; c < nc; c++) best = max(best, best_s[c]);
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
    // CTAs per row: enough of them for every SM, a run of at least 2048 ids each
    int nc = 1;
    while (nc < 8 && (long long)r->n_rows * nc < 2 * 148 && a.vocab / (2 * nc) >= 2048) nc *= 2;
    const int per = ((a.vocab + nc - 1) / nc + 3) / 4 * 4;
    const bool vec = a.vocab % 4 == 0 && a.ld % 4 == 0 && a.ld_out % 4 == 0 && kv8_aligned(a.logits, 16) &&
                     kv8_aligned(a.out, 16);
    auto kern = vec ? k_logits_rules<true> : k_logits_rules<false>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)LR_SMEM);
    if (e != cudaSuccess) throw Error(HG_ERR_CUDA, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)r->n_rows * nc);
    cfg.blockDim = dim3(LR_THREADS);
    cfg.dynamicSmemBytes = LR_SMEM;
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = nc;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    kv8_launched(cudaLaunchKernelEx(&cfg, kern, *r, a, nc, per));
  })
}
