// Shared pieces of the 8-bit KV cache kernels (kv8.cu, kv8_attn.cu) and the logit rules (rules.cu):
// the argument structs as the kernels see them, the checks of row and page indices that come from
// device memory, and the host-side argument checks of the entry points.
#pragma once
#include <climits>
#include <mutex>
#include <set>
#include <string>
#include <utility>

#include "hg_device.cuh"
#include "hg_host.h"

namespace hg {

constexpr int KV8_PAGE = 16;           // slots of a page
constexpr int KV8_MAX_SEQS = 1024;     // sequences of one call
constexpr int KV8_MAX_GROUP = 32;      // q heads per kv head

__host__ __device__ constexpr int kv8_block_bytes(int hd) { return 32 * hd + 128; }

// Byte offsets inside a (page, kv head) block (hobbygpu.h, hg_kv8_cache). The K tile of 8 slots x 16
// bytes and the V column of 16 slots are the 128-byte core matrices that a tcgen05 operand without
// swizzle is made of, so a page goes into shared memory by plain bulk copies, ready for the MMA.
__host__ __device__ constexpr int kv8_k_off(int hd, int w, int i) {
  return (w >> 3) * 8 * hd + (i >> 4) * 128 + (w & 7) * 16 + (i & 15);
}
__host__ __device__ constexpr int kv8_v_off(int hd, int w, int i) { return 16 * hd + i * 16 + w; }
__host__ __device__ constexpr int kv8_ks_off(int hd, int w) { return 32 * hd + 4 * w; }
__host__ __device__ constexpr int kv8_vs_off(int hd, int w) { return 32 * hd + 64 + 4 * w; }

__device__ __forceinline__ void kv8_flag(int32_t* err, int code) {
  if (err) atomicExch(err, code);
}

// The rows of a sequence, with the offsets clamped to the row buffers: [r0, r0 + n), behind `start`.
struct SeqSpan {
  int r0, n, start;
};
__device__ __forceinline__ SeqSpan kv8_span(const hg_rows& R, int s, bool with_start) {
  SeqSpan p;
  const int a = R.row_off[s], b = R.row_off[s + 1];
  p.r0 = min(max(a, 0), R.n_rows);
  p.n = min(max(b, p.r0), R.n_rows) - p.r0;
  p.start = with_start ? R.start[s] : 0;
  if (p.start < 0 || p.n > R.max_rows || a < 0 || b < a || b > R.n_rows) {
    kv8_flag(R.err, HG_ERR_INVALID);
    p.n = p.start < 0 ? 0 : min(p.n, R.max_rows);
  }
  return p;
}

// The parent of row j of a span (-1: none, -2 and below: row j is padding, returned as -2); one that is
// not below j is none.
__device__ __forceinline__ int kv8_parent(const hg_rows& R, const SeqSpan& p, int j) {
  if (!R.parent) return j - 1;
  const int q = R.parent[p.r0 + j];
  if (q < j) return max(q, -2);
  kv8_flag(R.err, HG_ERR_INVALID);
  return -1;
}

// A stretch of a row's path, looked at by W neighbouring lanes at once: from row `at`, which is on the path or
// padding, the rows at, at - 1, ... at - len + 1 are on it, and it goes on at `next` (-1: ends). A chain
// given by its parents takes a load per W rows, where a walk from parent to parent waits for a load per
// row. (A chain of 2500 rows, 8 q heads, 2 kv heads, 64 dims: attended in 0.30 ms, 0.16 without parents.)
struct PathRun {
  int len, next;
};
template <int W>
__device__ __forceinline__ PathRun kv8_run(const hg_rows& R, const SeqSpan& p, int at) {
  const int lane = threadIdx.x & 31, l = lane & (W - 1), first = lane - l, i = at - l;
  const unsigned mask = (W == 32 ? 0xffffffffu : (1u << (W & 31)) - 1u) << first;
  const int up = i >= 0 ? R.parent[p.r0 + i] : INT_MIN;
  const int n = __ffs(~(__ballot_sync(mask, up == i - 1) >> first)) - 1;  // rows whose parent is the row before
  if (n < 0 || n >= W) return {W, at - W};
  const int q = __shfl_sync(mask, up, n, W);  // of the first that is not one of those
  if (at - n < 0 || q <= -2) return {n, -1};
  if (q < at - n) return {n + 1, q};
  if (l == 0) kv8_flag(R.err, HG_ERR_INVALID);
  return {n + 1, -1};
}

// Address of the block of (slot, kv head), or null where the sequence has no such page. Slots are
// 64-bit: start + j may pass the 32-bit range.
__device__ __forceinline__ uint8_t* kv8_block(const hg_kv8_cache& C, int s, long long slot, int kvh) {
  const long long pg = slot / KV8_PAGE;
  if (pg >= C.bt_stride) return nullptr;
  const int id = C.block_table[(size_t)s * C.bt_stride + pg];
  if ((unsigned)id >= (unsigned)C.n_pages) return nullptr;
  return static_cast<uint8_t*>(C.pool) + (long long)id * C.page_stride + (long long)kvh * kv8_block_bytes(C.head_dim);
}

// Sums over the warp of R values per lane: lane i gets value i % R's.
template <int R, class T>
__device__ __forceinline__ T warp_sums(T (&v)[R]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int half = R / 2; half > 0; half /= 2) {
#pragma unroll
    for (int i = 0; i < half; i++) {
      const bool up = lane & half;
      const T give = up ? v[i] : v[i + half], keep = up ? v[i + half] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, half);
    }
  }
#pragma unroll
  for (int x = R; x < 32; x *= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], x);
  return v[0];
}

// Two f32 values side by side: one instruction for both.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pack2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// ---- host ----
inline void kv8_need(bool ok, const char* what) {
  if (!ok) throw Error(HG_ERR_INVALID, what);
}
inline bool kv8_aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

inline void kv8_check_rows(const hg_rows* r, bool with_start) {
  kv8_need(r, "null argument");
  kv8_need(r->n_seqs >= 0 && r->n_seqs <= KV8_MAX_SEQS, "n_seqs must be in 0..1024");
  kv8_need(r->n_rows >= 0 && r->n_rows <= INT_MAX / 256, "n_rows out of range");
  if (r->n_seqs == 0 || r->n_rows == 0) return;
  kv8_need(r->max_rows > 0, "max_rows must be positive");
  kv8_need(r->row_off && (r->start || !with_start), "null argument");
  kv8_need(kv8_aligned(r->row_off, 4) && kv8_aligned(r->start, 4) && kv8_aligned(r->parent, 4) &&
               kv8_aligned(r->err, 4),
           "row arrays must be 4-byte aligned");
}

inline void kv8_check_cache(const hg_kv8_cache* c) {
  kv8_need(c, "null argument");
  kv8_need(c->head_dim == 64 || c->head_dim == 128, "head_dim must be 64 or 128");
  kv8_need(c->n_kv_heads > 0 && c->n_kv_heads <= 1024, "n_kv_heads must be in 1..1024");
  kv8_need(c->n_pages > 0, "n_pages must be positive");
  kv8_need(c->bt_stride > 0 && c->bt_stride <= 1 << 26, "bt_stride out of range");
  kv8_need(c->block_table && c->pool, "null argument");
  kv8_need(kv8_aligned(c->block_table, 4), "block_table must be 4-byte aligned");
  kv8_need(kv8_aligned(c->pool, 16), "pool must be 16-byte aligned");
  kv8_need(c->page_stride % 16 == 0 && c->page_stride >= (int64_t)c->n_kv_heads * kv8_block_bytes(c->head_dim),
           "page_stride must be a multiple of 16 and hold a page's blocks");
}

// The device that holds p becomes current for the call.
struct Kv8Device {
  int prev = -1, device = 0;
  explicit Kv8Device(const void* p) {
    cudaPointerAttributes at{};
    cudaError_t e = cudaPointerGetAttributes(&at, p);
    if (e != cudaSuccess) {
      cudaGetLastError();
      throw Error(HG_ERR_CUDA, std::string("cudaPointerGetAttributes: ") + cudaGetErrorString(e));
    }
    kv8_need(at.type == cudaMemoryTypeDevice || at.type == cudaMemoryTypeManaged, "not device memory");
    device = at.device;
    int cur = -1;
    cudaGetDevice(&cur);
    if (cur != at.device) {
      e = cudaSetDevice(at.device);
      if (e != cudaSuccess) {
        cudaGetLastError();
        throw Error(HG_ERR_CUDA, std::string("cudaSetDevice: ") + cudaGetErrorString(e));
      }
      prev = cur;
    }
  }
  ~Kv8Device() {
    if (prev >= 0) cudaSetDevice(prev);
  }
  Kv8Device(const Kv8Device&) = delete;
  Kv8Device& operator=(const Kv8Device&) = delete;
};

inline void kv8_launched(cudaError_t e) {
  if (e == cudaSuccess) return;
  cudaGetLastError();  // reported here, not to the next call that asks
  throw Error(HG_ERR_CUDA, std::string("kernel launch: ") + cudaGetErrorString(e));
}

// The kernel may use `most` bytes of dynamic shared memory, and clusters of up to 16 CTAs, on the device
// (told to the runtime once).
template <typename... P>
inline void kv8_smem_limit(void (*kern)(P...), int device, size_t most) {
  static std::mutex mu;
  static std::set<std::pair<const void*, int>> told;
  const std::pair<const void*, int> key(reinterpret_cast<const void*>(kern), device);
  std::lock_guard<std::mutex> lock(mu);
  if (told.count(key)) return;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) {
    cudaGetLastError();
    throw Error(HG_ERR_CUDA, std::string("cudaFuncSetAttribute: ") + cudaGetErrorString(e));
  }
  told.insert(key);
}

// Launch with programmatic stream serialization: the kernels wait (pdl_wait) before they touch memory.
template <typename... P, typename... Args>
inline void kv8_launch_pdl(void (*kern)(P...), dim3 grid, int threads, size_t smem, void* stream, Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  kv8_launched(cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...));
}

#define KV8_API(...)                                     \
  try {                                                  \
    __VA_ARGS__;                                         \
    return HG_OK;                                        \
  } catch (const ::hg::Error& ex_) {                     \
    ::hg::set_last_error(ex_.what());                    \
    return ex_.code;                                     \
  } catch (const std::exception& ex_) {                  \
    ::hg::set_last_error(ex_.what());                    \
    return HG_ERR_INVALID;                               \
  }

}  // namespace hg
