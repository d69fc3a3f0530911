// paged_attention.cuh — what the kernels of the attention over the paged
// cache share (paged_attention.cu: few rows per key/value head;
// paged_attention_mma.cu: many; tree_attention.cu: many of a tree's nodes).
#pragma once

#include <atomic>
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

#include "sm100_ptx.cuh"

namespace dwa {

struct PagedArgs {
  const uint16_t* q;
  uint16_t* out;
  int64_t q_ld, out_ld;  // elements between tokens
  const void *k, *v;
  const float *k_scale, *v_scale;
  int64_t ld_page, ld_scale_page;  // elements, scales
  int64_t n_pages;
  const int32_t* table;
  int64_t ld_table;
  int max_pages, page_log2;
  const int32_t* lengths;
  const int32_t* q_start;  // null: `even` rows per sequence
  int64_t T;
  int even, max_q;
  int B, H, H_kv, group;  // group = H / H_kv query heads per key/value head
  int d;
  float scale_log2;  // scale * log2(e)
  int32_t* status;
  // Trees: the nodes that a row's new token sees, tree_words words of 32 bits to a token.
  const uint32_t* tree;
  int tree_words;
};

// Rows per key/value head that paged_attention.cu takes; more go to a tcgen05 kernel.  At 20
// rows (16 sequences of 4096, 8 heads of 128, bf16) that one (paged_attention_mma.cu) takes 58 us, this one (in two passes) 165.
constexpr int kFewRows = 16;

// Rows that tree_attention.cu takes, and the blocks of rows of tree_attention_short.cu, which takes two.
constexpr int kTreeRows = 32;

// One sequence as the device finds it.
struct PagedSeq {
  int64_t row0;   // first row of q
  int n;          // new tokens
  int length;     // cached tokens, the new ones with them
  bool bad;       // its rows get NaN
};

__device__ __forceinline__ void paged_report(int32_t* status) {
  if (status != nullptr) atomicCAS(status, 0, 5 /* DWA_ERR_DEVICE_CHECK */);
}

// From its number and what q_start and lengths say of it (lo, hi: unless there is no q_start).
__device__ __forceinline__ PagedSeq paged_seq(const PagedArgs& a, int b, int64_t lo, int64_t hi, int length) {
  PagedSeq s;
  if (a.q_start != nullptr) {
    const bool fine = lo >= 0 && lo <= hi && hi <= a.T;
    s.row0 = fine ? lo : 0;
    s.n = fine ? static_cast<int>(hi - lo) : 0;  // rows that cannot be told apart stay as they are
    s.bad = !fine;
  } else {
    s.row0 = static_cast<int64_t>(b) * a.even;
    s.n = a.even;
    s.bad = false;
  }
  s.length = length;
  if (s.length < 0 || s.length > (static_cast<int64_t>(a.max_pages) << a.page_log2) ||
      s.n > a.max_q) {
    s.bad = true;
    s.length = 0;
  }
  return s;
}

__device__ __forceinline__ int q_start_at(const PagedArgs& a, int b) {
  return a.q_start != nullptr ? __ldg(a.q_start + b) : 0;
}
__device__ __forceinline__ PagedSeq paged_seq(const PagedArgs& a, int b) {
  return paged_seq(a, b, q_start_at(a, b), q_start_at(a, b + 1), __ldg(a.lengths + b));
}

// Blocks start in the order of their number, so the ones with the most keys should
// have the lowest: the index i < n whose cost(i) has this rank among all (equal costs by
// index).  Every block finds its own; `costs` and `found` are shared memory.
constexpr int kMostRanked = 128;  // more units than this even out by themselves
template <typename F>
__device__ __forceinline__ int ranked(int n, int rank, int* costs, int* found, F&& cost) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) costs[i] = cost(i);
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int own = costs[i];
    int before = 0;
    for (int j = 0; j < n; ++j) before += costs[j] > own || (costs[j] == own && j < i);
    if (before == rank) *found = i;
  }
  __syncthreads();
  return *found;
}

// Tokens that new token i may see.
__device__ __forceinline__ int paged_visible(const PagedSeq& s, int i) {
  return max(s.length - s.n + i + 1, 0);
}

// Trees.  Every new token of a sequence sees the tokens before the first of them, and of the new
// ones those that its mask names: node j is cached token length - n + j.
__device__ __forceinline__ int tree_prefix(const PagedSeq& s) { return s.length - s.n; }  // below 0: nodes without a place
// 32 keys from node `at` on that the token in row `row` of q sees, as bits; what lies before
// node 0 is seen by all.
__device__ __forceinline__ uint32_t tree_bits(const PagedArgs& a, int64_t row, int at) {
  if (at <= -32) return 0xFFFFFFFFu;
  const uint32_t* mask = a.tree + row * a.tree_words;
  const int w = at >> 5;  // -1 where bits before node 0 are among them
  const uint32_t lo = w < 0 ? 0xFFFFFFFFu : w < a.tree_words ? __ldg(mask + w) : 0u;
  const uint32_t hi = w + 1 < a.tree_words ? __ldg(mask + w + 1) : 0u;
  return __funnelshift_r(lo, hi, at & 31);
}
// Whether that token sees a node whose value is not finite: in channel ch of a bf16 cache, of an
// e4m3 one at all.  (Only where a block met such a value.)
template <bool kE4m3>
__device__ __noinline__ bool tree_sees_bad(const PagedArgs& a, const PagedSeq s, const int32_t* table, int hk,
                                           int64_t row, int ch) {
  const int prefix = tree_prefix(s);
  for (int node = max(-prefix, 0); node < s.n; ++node) {
    if (!(tree_bits(a, row, node) & 1u)) continue;
    const int key = prefix + node, page = __ldg(table + (key >> a.page_log2));
    if (page < 0 || page >= a.n_pages) continue;
    const int64_t at = (static_cast<int64_t>(hk) << a.page_log2) + (key & ((1 << a.page_log2) - 1));
    if constexpr (kE4m3) {
      if (!(fabsf(__ldg(a.v_scale + page * a.ld_scale_page + at)) < INFINITY)) return true;
    } else {
      const uint16_t x = __ldg(static_cast<const uint16_t*>(a.v) + page * a.ld_page + at * a.d + ch);
      if ((x & 0x7F80u) == 0x7F80u) return true;
    }
  }
  return false;
}

// The new token of a row (rows are token-major, `group` query heads to a token).
__device__ __forceinline__ uint32_t row_token(uint32_t row, int group) {
  return group == 1 ? row : row / static_cast<uint32_t>(group);
}

// ---------------------------------------------------------------- arithmetic
// ex2.approx: 2 ulp of f32, far below the probabilities' own rounding.
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two e4m3 codes (the low or high half of w) as a pair of fp16, exactly.
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint32_t w, int high) {
  uint32_t r;
  if (high)
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}"
        : "=r"(r) : "r"(w));
  else
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}"
        : "=r"(r) : "r"(w));
  return r;
}

// e4m3 caches: a code's weight in its row is its probability p <= 1 times its value's scale,
// in units of 2^v_exp / kPScale, chosen so that the row's largest weight lies between
// kLowWeight and kMostWeight: fp16 holds 11 bits of everything down to 2^-20 of it then.
constexpr float kPScale = 2048.f, kMostWeight = 32768.f, kLowWeight = 64.f;
constexpr int kLeastExp = -110;    // a scale of 2^-126 still makes 2^-5
constexpr float kAllRoom = 0x1p30f;  // of a row without weights so far
__device__ __forceinline__ float pow2(int n) {  // -126 to 127
  return __uint_as_float(static_cast<uint32_t>(127 + n) << 23);
}
// kPScale / 2^v_exp: v_exp is at most 127
__device__ __forceinline__ float exp_scale(int v_exp) { return pow2(11 - v_exp); }
// A scale as m 2^e, exactly, with 1 <= |m| < 2 (smaller for subnormal numbers); what is not
// finite becomes NaN.  Returns m.
__device__ __forceinline__ float scale_parts(float x, int* e) {
  const uint32_t w = __float_as_uint(x), field = (w >> 23) & 0xFFu;
  *e = field == 0u || field == 0xFFu ? -126 : static_cast<int>(field) - 127;
  return field == 0u      ? x * 0x1p126f
         : field == 0xFFu ? __uint_as_float(0x7FC00000u)
                          : __uint_as_float((w & 0x807FFFFFu) | 0x3F800000u);
}
__device__ __forceinline__ int exponent_of(float x) {  // x >= 0
  return static_cast<int>(__float_as_uint(x) >> 23) - 127;
}
// How far a unit has to rise so that weight x lies between 2^11 and 2^12 (an infinite one: 117).
__device__ __forceinline__ int exponent_above(float x) {
  return static_cast<int>(__float_as_uint(x) >> 23) - 127 - 11;
}

// A row of Q goes into fp16 times the power of two *up that puts its largest
// magnitude `top` (f32 bits) in [2^13, 2^14): what falls below fp16's range then is
// 2^-37 of it.  (2^126 is the largest power; smaller rows come out exact with it, bf16
// being multiples of 2^-133.)  Returns the factor of the row's scores (never 0: minus
// infinity times it has to stay that).
__device__ __forceinline__ float f16_row_scale(uint32_t top, float scale_log2, float* up) {
  const int e = top == 0 || top >= 0x7F800000u ? 13 : static_cast<int>(top >> 23) - 127;
  const int n = min(13 - e, 126);
  *up = __uint_as_float(static_cast<uint32_t>(127 + n) << 23);
  return fmaxf(scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - n) << 23), 0x1p-126f);
}

// ---------------------------------------------------------------- clusters
// The same variable in block `rank` of the cluster.
__device__ __forceinline__ float ld_cluster_f32(const float* local, int rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];"
               : "=f"(v)
               : "r"(map_to_cta(smem_u32(local), rank))
               : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster_f32x2(const float* local, int rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
               : "=f"(v.x), "=f"(v.y)
               : "r"(map_to_cta(smem_u32(local), rank))
               : "memory");
  return v;
}
__device__ __forceinline__ int ld_cluster_s32(const int* local, int rank) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];"
               : "=r"(v)
               : "r"(map_to_cta(smem_u32(local), rank))
               : "memory");
  return v;
}
// Stores into another block's shared memory, at an address of map_to_cta.
__device__ __forceinline__ void st_cluster_f32x4(uint32_t addr, float x, float y, float z, float w) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(x), "f"(y), "f"(z), "f"(w)
               : "memory");
}
__device__ __forceinline__ void st_cluster_f32x2(uint32_t addr, float x, float y) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(x), "f"(y) : "memory");
}
__device__ __forceinline__ void st_cluster_s32(uint32_t addr, int x) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(addr), "r"(x) : "memory");
}
__device__ __forceinline__ void min_cluster_s32(uint32_t addr, int x) {
  asm volatile("red.relaxed.cluster.shared::cluster.min.s32 [%0], %1;" ::"r"(addr), "r"(x) : "memory");
}

// Tensor map of one of the caches, (channel, token of the page, half of the channels, head,
// page): boxes of `row_bytes` by `box_rows` tokens of one page's head, 128-byte rows
// swizzled.  Channels beyond d arrive as zeros; two halves (64 bf16 each) only for d = 128.
bool make_page_map(CUtensorMap* map, const void* ptr, const PagedArgs& a, int row_bytes, int box_rows,
                   int box_halves);

// One box of it, at these coordinates.
__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x,
                                              int y, int half, int head, int page) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(half), "r"(head), "r"(page)
      : "memory");
}

// Lets a kernel have its dynamic shared memory, once per device.
template <auto kKernel>
cudaError_t allow_smem_once(int bytes) {
  static std::atomic<bool> done[64] = {};
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
  if (dev < 64 && done[dev].load(std::memory_order_acquire)) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) done[dev].store(true, std::memory_order_release);
  return e;
}

}  // namespace dwa
