// kv_keep.cu — the cached tokens of a tree's path that stood move to the places behind the
// sequence's earlier tokens: token start + path[i] to start + i, in every layer.
//
// Latency first (a few tokens per sequence): one launch for all layers, heads, keys and
// values.  Node numbers ascend along a path from 0 or more, so a place i is never above the number of the node
// that moves there (which every thread checks of its own nodes before it looks up their pages), and a token
// moves before its own place is needed: a thread that moves a
// vector's 16 bytes of one token after the other needs no second copy of them.  32 paths of up to 12 tokens in
// 12 layers of 16 8-bit heads of 128: 9.0 us, 2.3 TB/s of scattered 128-byte rows, two dependent rounds of loads
// (path and table, then the rows) before the stores.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "dwa_internal.h"
#include "kv_store.cuh"
#include "paged_attention.cuh"

namespace dwa {

namespace {

constexpr int kThreads = 256;
constexpr int kStaged = 256;  // moves whose pages and places are looked up together
constexpr int kBatch = 8;     // tokens under way together

struct KeepArgs {
  uint8_t *k, *v;
  float *k_scale, *v_scale;
  int64_t ld_layer, ld_scale_layer, ld_page, ld_scale_page;  // bytes, scales, bytes, scales
  int64_t n_pages;
  int H, page_log2, row_bytes;
  const int32_t* table;
  int64_t ld_table;
  int max_pages;
  const int32_t *start, *path, *n_accepted;
  int steps;  // path entries of a sequence
  int64_t columns;  // 16-byte pieces of a token: layers, keys and values, heads
  int64_t scales;   // scales of a token
  int parts;
  int32_t* status;
};

struct Move {  // a token's page and place in it, before and after
  int64_t from_page, to_page;
  int from, to;
};

// A thread's part of moves k0 .. k1 - 1, in their order.
template <typename T, typename F>
__device__ __forceinline__ void move(const Move* moves, int k0, int k1, F&& at) {
  for (int k = k0; k < k1; k += kBatch) {
    T held[kBatch];
#pragma unroll
    for (int e = 0; e < kBatch; ++e)
      if (k + e < k1) held[e] = *at(moves[k + e].from_page, moves[k + e].from);
#pragma unroll
    for (int e = 0; e < kBatch; ++e)
      if (k + e < k1) *at(moves[k + e].to_page, moves[k + e].to) = held[e];
  }
}

__global__ void __launch_bounds__(kThreads) kv_keep_kernel(const KeepArgs a) {
  __shared__ Move moves[kStaged];
  __shared__ int first;
  const int64_t b = blockIdx.x / a.parts;
  const int part = static_cast<int>(blockIdx.x % a.parts);
  const int n = __ldg(a.n_accepted + b);
  const int64_t start = __ldg(a.start + b);
  const int32_t* path = a.path + b * a.steps;
  const int32_t* table = a.table + b * a.ld_table;
  const int64_t tokens = static_cast<int64_t>(a.max_pages) << a.page_log2;
  // the path's start comes with its length, not behind it
  const int own = static_cast<int>(threadIdx.x), own_node = own < a.steps ? __ldg(path + own) : 0;
  const int own_before = own > 0 && own <= a.steps ? __ldg(path + own - 1) : -1;
  if (n < 0 || (n == 0 && __ldg(path) < 0)) return;  // nothing stood
  // nodes ascend: from the first that moves on all do
  if (threadIdx.x == 0) first = n + 1;
  __syncthreads();
  const int mask = (1 << a.page_log2) - 1;
  bool bad = n >= a.steps || start < 0;
  for (int i = threadIdx.x; i <= n && !bad; i += kThreads) {
    const int64_t node = i == own ? own_node : __ldg(path + i), before = i == own ? own_before : __ldg(path + i - 1);
    // With i <= node both lookups are inside the table, whatever the rest of the path says.
    bad = node <= before || node < i || start + node >= tokens;
    if (bad || node == i) continue;
    const int64_t p = __ldg(table + ((start + node) >> a.page_log2)), q = __ldg(table + ((start + i) >> a.page_log2));
    bad = p < 0 || p >= a.n_pages || q < 0 || q >= a.n_pages;
    atomicMin(&first, i);
    if (i < kStaged) moves[i] = Move{p, q, static_cast<int>((start + node) & mask), static_cast<int>((start + i) & mask)};
  }
  if (__syncthreads_or(bad)) {  // the sequence's tokens stay where they are
    if (part == 0 && threadIdx.x == 0) paged_report(a.status);
    return;
  }
  const int pieces = a.row_bytes >> 4;
  for (int i0 = 0; i0 <= n; i0 += kStaged) {
    if (i0 > 0) {  // the first are there already
      __syncthreads();
      const int i = i0 + threadIdx.x;
      if (i <= n && i >= first) {
        const int64_t old = start + __ldg(path + i), now = start + i;
        moves[threadIdx.x] = Move{__ldg(table + (old >> a.page_log2)), __ldg(table + (now >> a.page_log2)),
                                  static_cast<int>(old & mask), static_cast<int>(now & mask)};
      }
      __syncthreads();
    }
    const int k0 = max(first - i0, 0), k1 = min(n + 1 - i0, kStaged);
    if (k0 >= k1) continue;
    for (int64_t c = static_cast<int64_t>(part) * kThreads + threadIdx.x; c < a.columns + a.scales;
         c += static_cast<int64_t>(a.parts) * kThreads) {
      const bool scale = c >= a.columns;
      const int64_t vec = scale ? c - a.columns : c / pieces;  // (layer, keys or values, head)
      const int64_t side = vec / a.H;
      const int64_t head = (vec - side * a.H) << a.page_log2;
      if (scale) {
        float* const base = ((side & 1) ? a.v_scale : a.k_scale) + (side >> 1) * a.ld_scale_layer + head;
        move<float>(moves, k0, k1, [&](int64_t page, int at) { return base + page * a.ld_scale_page + at; });
      } else {
        uint8_t* const base = ((side & 1) ? a.v : a.k) + (side >> 1) * a.ld_layer + head * a.row_bytes + (c - vec * pieces) * 16;
        move<uint4>(moves, k0, k1, [&](int64_t page, int at) {
          return reinterpret_cast<uint4*>(base + page * a.ld_page + static_cast<int64_t>(at) * a.row_bytes);
        });
      }
    }
  }
}

}  // namespace

cudaError_t launch_kv_keep(const KvCacheView& c, int layers, int64_t ld_layer, int64_t ld_scale_layer,
                           const int32_t* table, int64_t ld_table, int max_pages, const int32_t* start,
                           const int32_t* path, const int32_t* n_accepted, int64_t B, int steps,
                           int32_t* status, cudaStream_t stream) {
  const bool e4m3 = c.k_scale != nullptr;
  const int es = e4m3 ? 1 : 2;
  KeepArgs a{};
  a.k = static_cast<uint8_t*>(const_cast<void*>(c.k)); a.v = static_cast<uint8_t*>(const_cast<void*>(c.v));
  a.k_scale = const_cast<float*>(c.k_scale); a.v_scale = const_cast<float*>(c.v_scale);
  a.ld_layer = ld_layer * es; a.ld_scale_layer = ld_scale_layer;
  a.ld_page = c.ld_page * es; a.ld_scale_page = c.ld_scale_page;
  a.n_pages = c.n_pages;
  a.H = c.H; a.page_log2 = log2_at_least(c.page_size); a.row_bytes = c.d * es;
  a.table = table; a.ld_table = ld_table; a.max_pages = max_pages;
  a.start = start; a.path = path; a.n_accepted = n_accepted; a.steps = steps;
  const int64_t vectors = static_cast<int64_t>(layers) * 2 * c.H;
  a.columns = vectors * (a.row_bytes / 16);
  a.scales = e4m3 ? vectors : 0;
  const int64_t most = (4 * static_cast<int64_t>(device_sm_count()) + B - 1) / B;  // blocks of a sequence
  a.parts = static_cast<int>(std::max<int64_t>(1, std::min((a.columns + a.scales + kThreads - 1) / kThreads, most)));
  a.status = status;
  kv_keep_kernel<<<static_cast<unsigned>(B * a.parts), kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace dwa
