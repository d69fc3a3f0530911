// draft_tree.cu — trees of drafted tokens: which nodes a node sees, and the walk through a
// verified tree.
//
// A tree is the n newest tokens of a sequence, parents before children; node 0 is the
// sequence's newest token, the others are drafts.
//
// Masks: a node's row has its own bit and its ancestors'.  Up to 128 nodes by doubling, in log2(depth) rounds;
// beyond, a thread per node walks up: since parents have lower numbers the bits come in
// descending order, a word at a time.  Latency: one tree of 16 nodes 2.1 us, 64 of 33 to 128 2.9 (walking up
// 6.4).
//
// Walk: at node 0 a token t is drawn from the node's row of probabilities; where a child has t
// the walk goes on from there, else it ends with t.  Given the tree t is distributed as
// the target's at every step, whatever proposed the drafts: they only decide how far one
// pass of the model reaches.  Running sums are 64-bit, good to 1e-16 of their total, so
// the outcome does not hang on their order.
//
// One row of V entries per step of the path is read.  A cluster of blocks shares it, each lane a
// contiguous chunk (32 entries of 64400: one round of loads); the warps' sums go through distributed shared memory, the
// warp whose piece holds the draw finds it and tells every block.
// Latency, a row after the other: one tree over 32000 entries 6.7 us, 32 over 64400 with up to nine draws 14 (18
// with a row's entries dealt out by single vectors).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>

#include "dwa_internal.h"
#include "paged_attention.cuh"
#include "sm100_ptx.cuh"

namespace dwa {

namespace {

// ---------------------------------------------------------------- masks
constexpr int kMaskThreads = 128;
constexpr int kMostNodes = 4096;  // of a tree
constexpr int kShortWords = 2;    // up to 128 nodes
constexpr int kRowBits = 8192;    // rows that are told apart at a time where a range is bad

struct MaskArgs {
  const int32_t *parents, *q_start;
  int64_t T;
  int even, max_q, B, words;
  uint64_t* mask;
  int32_t *depth, *status;
};

// Sequence b's rows; whether they are any.
__device__ __forceinline__ bool rows_of(const MaskArgs& a, int b, int64_t* lo, int64_t* hi) {
  *lo = __ldg(a.q_start + b);
  *hi = __ldg(a.q_start + b + 1);
  return *lo >= 0 && *lo <= *hi && *hi <= a.T;
}
// Whether one of sequences 0 .. n - 1 has a range that is none; the block together.
__device__ __forceinline__ bool any_bad_range(const MaskArgs& a, int n) {
  bool bad = false;
  for (int i = threadIdx.x; i < n && !bad; i += kMaskThreads) {
    int64_t lo, hi;
    bad = !rows_of(a, i, &lo, &hi);
  }
  return __syncthreads_or(bad);
}
// Zeros to the rows that no sequence has, wherever they are: kRowBits rows at a time the ranges set their bits.
__device__ __noinline__ void clear_free_rows(const MaskArgs& a) {
  __shared__ uint32_t taken[kRowBits / 32];
  for (int64_t first = 0; first < a.T; first += kRowBits) {
    for (int i = threadIdx.x; i < kRowBits / 32; i += kMaskThreads) taken[i] = 0;
    __syncthreads();
    for (int b = threadIdx.x; b < a.B; b += kMaskThreads) {
      int64_t lo, hi;
      if (!rows_of(a, b, &lo, &hi)) continue;
      const int from = static_cast<int>(min(max(lo - first, int64_t{0}), int64_t{kRowBits}));
      const int to = static_cast<int>(min(max(hi - first, int64_t{0}), int64_t{kRowBits}));
      for (int t = from; t < to; t = (t | 31) + 1) {
        const int n = min(to - t, 32 - (t & 31));
        atomicOr(&taken[t >> 5], (n == 32 ? 0xFFFFFFFFu : (1u << n) - 1u) << (t & 31));
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < min(a.T - first, int64_t{kRowBits}); i += kMaskThreads) {
      if ((taken[i >> 5] >> (i & 31)) & 1u) continue;
      for (int w = 0; w < a.words; ++w) a.mask[(first + i) * a.words + w] = 0;
      a.depth[first + i] = 0;
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kMaskThreads) tree_masks_kernel(const __grid_constant__ MaskArgs a) {
  extern __shared__ __align__(16) int32_t up[];  // this sequence's parents
  const int b = blockIdx.x;
  int64_t lo = static_cast<int64_t>(b) * a.even, hi = lo + a.even;
  auto clear = [&](int64_t from, int64_t to) {  // rows of no sequence see nothing
    for (int64_t t = from + threadIdx.x; t < to; t += kMaskThreads) {
      for (int w = 0; w < a.words; ++w) a.mask[t * a.words + w] = 0;
      a.depth[t] = 0;
    }
  };
  if (a.q_start != nullptr) {
    const bool fine = rows_of(a, b, &lo, &hi);
    if (!fine) {  // the first such sequence's block sees to all rows of no sequence
      if (threadIdx.x == 0) paged_report(a.status);
      if (!any_bad_range(a, b)) clear_free_rows(a);
      return;
    }
    const bool ends = (b == 0 && lo > 0) || (b == a.B - 1 && hi < a.T);
    if (ends && !any_bad_range(a, a.B)) {  // ranges follow one another: rows of no sequence are before and behind
      if (b == 0) clear(0, lo);
      if (b == a.B - 1) clear(hi, a.T);
    }
  }
  if (hi - lo > a.max_q) {
    if (threadIdx.x == 0) paged_report(a.status);
    clear(lo, hi);
    return;
  }
  const int n = static_cast<int>(hi - lo);
  bool bad = false;
  for (int i = threadIdx.x; i < n; i += kMaskThreads) {
    int p = __ldg(a.parents + lo + i);
    if (p < -1 || p >= i) {
      bad = true;
      p = -1;  // a root of its own
    }
    up[i] = p;
  }
  if (__syncthreads_or(bad) && threadIdx.x == 0) paged_report(a.status);
  if (a.words <= kShortWords) {
    // Few words: a node takes what the node that it has come to sees, twice as far each time.
    uint64_t* const seen = reinterpret_cast<uint64_t*>(up + ((a.max_q + 1) & ~1));
    static_assert(64 * kShortWords <= kMaskThreads, "a node to a thread");
    const int i = threadIdx.x;
    uint64_t bits[kShortWords];
    int at = i < n ? up[i] : -1;
#pragma unroll
    for (int w = 0; w < kShortWords; ++w) {
      bits[w] = i >> 6 == w ? 1ull << (i & 63) : 0;
      if (i < n) seen[i * kShortWords + w] = bits[w];
    }
    while (__syncthreads_or(at >= 0)) {
      if (at >= 0) {
#pragma unroll
        for (int w = 0; w < kShortWords; ++w) bits[w] |= seen[at * kShortWords + w];
        at = up[at];
      }
      __syncthreads();
      if (i < n) {
        up[i] = at;
#pragma unroll
        for (int w = 0; w < kShortWords; ++w) seen[i * kShortWords + w] = bits[w];
      }
    }
    if (i < n) {
      int depth = -1;
#pragma unroll
      for (int w = 0; w < kShortWords; ++w) {
        depth += __popcll(bits[w]);
        if (w < a.words) a.mask[(lo + i) * a.words + w] = bits[w];
      }
      a.depth[lo + i] = depth;
    }
    return;
  }
  for (int i = threadIdx.x; i < n; i += kMaskThreads) {
    uint64_t* row = a.mask + (lo + i) * a.words;
    int w = i >> 6, depth = -1;
    for (int k = w + 1; k < a.words; ++k) row[k] = 0;
    uint64_t bits = 0;
    for (int p = i; p >= 0; p = up[p]) {
      while (w > p >> 6) {
        row[w--] = bits;
        bits = 0;
      }
      bits |= 1ull << (p & 63);
      ++depth;
    }
    while (w >= 0) {
      row[w--] = bits;
      bits = 0;
    }
    a.depth[lo + i] = depth;
  }
}

// ---------------------------------------------------------------- the walk
constexpr int kWalkThreads = 256;
constexpr int kWalkWarps = kWalkThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBatch = 8;      // of four entries, under way together
constexpr int kHeldNodes = 2;  // of a lane

struct WalkArgs {
  const void* target;
  const int32_t *tokens, *parents, *q_start;
  const float* u;
  int64_t T;
  int even, B, steps, V;
  int chunk;  // entries per lane, a multiple of 4: a warp's lie side by side
  int wide;   // rows may be read four entries at a time
  int32_t *n_accepted, *out_tokens, *path;
};

// Entries i .. i + 3 of a row, zeros from `end` on; what is no positive finite number is nothing.
template <typename T>
__device__ __forceinline__ void weights4(const T* row, int i, int end, int wide, float (&x)[4]) {
  if (wide && i < end) {
    if constexpr (sizeof(T) == 2) {
      const uint2 w = __ldg(reinterpret_cast<const uint2*>(row + i));
      x[0] = __uint_as_float(w.x << 16); x[1] = __uint_as_float(w.x & 0xFFFF0000u);
      x[2] = __uint_as_float(w.y << 16); x[3] = __uint_as_float(w.y & 0xFFFF0000u);
    } else {
      const float4 w = __ldg(reinterpret_cast<const float4*>(row + i));
      x[0] = w.x; x[1] = w.y; x[2] = w.z; x[3] = w.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j] = 0.f;
      if (i + j < end) {
        if constexpr (sizeof(T) == 2) x[j] = __uint_as_float(static_cast<uint32_t>(__ldg(row + i + j)) << 16);
        else x[j] = __ldg(row + i + j);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[j] = fmaxf(x[j], 0.f);  // NaN too
    x[j] = x[j] < INFINITY ? x[j] : 0.f;
  }
}
__device__ __forceinline__ double sum4(const float (&x)[4]) {
  return (static_cast<double>(x[0]) + static_cast<double>(x[1])) +
         (static_cast<double>(x[2]) + static_cast<double>(x[3]));
}
template <typename T>
__device__ __forceinline__ double weight1(const T* at) {
  float x;
  if constexpr (sizeof(T) == 2) x = __uint_as_float(static_cast<uint32_t>(__ldg(at)) << 16);
  else x = __ldg(at);
  x = fmaxf(x, 0.f);  // NaN too
  return x < INFINITY ? static_cast<double>(x) : 0.0;
}
__device__ __forceinline__ double warp_scan(double x) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xFFFFFFFFu, x, o);
    if ((threadIdx.x & 31) >= o) x += y;
  }
  return x;
}
__device__ __forceinline__ double ld_cluster_f64(const double* local, int rank) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];"
               : "=d"(v)
               : "r"(map_to_cta(smem_u32(local), rank))
               : "memory");
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kWalkThreads, 4) verify_tree_kernel(const WalkArgs a, const int cluster) {
  __shared__ double sums[2][kWalkWarps];  // of this step and the last
  __shared__ int drawn[2];
  const int rank = static_cast<int>(blockIdx.x % cluster);
  const int64_t b = blockIdx.x / cluster;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int V = a.V;
  int64_t row0 = b * a.even;
  int n = a.even;
  if (a.q_start != nullptr) {
    const int64_t lo = __ldg(a.q_start + b), hi = __ldg(a.q_start + b + 1);
    row0 = lo;
    n = lo >= 0 && lo <= hi && hi <= a.T ? static_cast<int>(hi - lo) : 0;
  }
  const bool writes = rank == 0 && threadIdx.x == 0;
  const int pieces = cluster * kWalkWarps;
  const int lo = static_cast<int>(min((static_cast<int64_t>(rank * kWalkWarps + warp) * 32 + lane) * a.chunk, static_cast<int64_t>(V)));
  const int hi = min(lo + a.chunk, V);  // this lane's entries
  // The first nodes' parents and tokens, some to a lane, are there before the first draw.
  int held_parent[kHeldNodes], held_token[kHeldNodes];
#pragma unroll
  for (int k = 0; k < kHeldNodes; ++k) {
    const int i = 32 * k + lane;
    held_parent[k] = i < n ? __ldg(a.parents + row0 + i) : -1;
    held_token[k] = i < n ? __ldg(a.tokens + row0 + i) : -1;
  }
  int node = 0, kept = 0, step = 0;
  bool going = n > 0;
  for (; going; ++step) {
    const int set = step & 1;
    const T* p = static_cast<const T*>(a.target) + (row0 + node) * V;
    const double u = __ldg(a.u + b * a.steps + step);
    double own = 0.0;
    for (int i0 = lo; i0 < hi; i0 += 4 * kBatch) {
      float x[kBatch][4];
#pragma unroll
      for (int r = 0; r < kBatch; ++r) weights4(p, i0 + 4 * r, hi, a.wide, x[r]);
#pragma unroll
      for (int r = 0; r < kBatch; ++r) own += sum4(x[r]);
    }
    const double upto = warp_scan(own);  // of the warp's piece
    if (lane == 31) sums[set][warp] = upto;
    cluster_sync();
    // Lane l has the sums of pieces 2 l and 2 l + 1, and by a scan what lies before them;
    // every warp computes the same.
    double mine0 = 0.0, mine1 = 0.0;
    if (2 * lane < pieces) {
      const int c = 2 * lane / kWalkWarps, k = 2 * lane % kWalkWarps;
      mine0 = ld_cluster_f64(&sums[set][k], c);
      mine1 = ld_cluster_f64(&sums[set][k + 1], c);
    }
    double before = warp_scan(mine0 + mine1);
    const double total = __shfl_sync(0xFFFFFFFFu, before, 31);
    if (total > 0.0) {
      const double goal = u * total;
      before -= mine0 + mine1;  // within rounding: what this decides is decided once, below
      const double mid = before + mine0;
      // the first piece whose running sum passes the goal, or the last with any weight
      const uint32_t past = __ballot_sync(0xFFFFFFFFu, (mine0 > 0.0 && mid > goal) ||
                                                           (mine1 > 0.0 && mid + mine1 > goal));
      const uint32_t some = __ballot_sync(0xFFFFFFFFu, mine0 > 0.0 || mine1 > 0.0);
      const int src = past ? __ffs(past) - 1 : 31 - __clz(some);
      const bool early = past ? mine0 > 0.0 && mid > goal : !(mine1 > 0.0);
      const int at = __shfl_sync(0xFFFFFFFFu, 2 * lane + (early ? 0 : 1), src);
      double run = __shfl_sync(0xFFFFFFFFu, early ? before : mid, src);
      if (at == rank * kWalkWarps + warp) {
        // The first lane whose running sum passes the goal, or where rounding keeps it at the goal the last
        // with weight; then of its entries, again shared out among the lanes, the lane's; then the entry.
        auto lane_of = [&](double sum, double incl) -> int {
          const uint32_t hit = __ballot_sync(0xFFFFFFFFu, sum > 0.0 && run + incl > goal);
          const uint32_t any = __ballot_sync(0xFFFFFFFFu, sum > 0.0);
          return hit ? __ffs(hit) - 1 : 31 - __clz(any);
        };
        int l = lane_of(own, upto);
        run += __shfl_sync(0xFFFFFFFFu, upto - own, l);
        const int first = __shfl_sync(0xFFFFFFFFu, lo, l), end = __shfl_sync(0xFFFFFFFFu, hi, l);
        const int per = (a.chunk + 31) / 32, from = min(first + lane * per, end), to = min(from + per, end);
        double part = 0.0;
        for (int i = from; i < to; ++i) part += weight1(p + i);
        const double incl = warp_scan(part);
        l = lane_of(part, incl);
        int found = from;
        if (lane == l) {
          double c = run + (incl - part);
          int last = from;
          bool in = false;
          for (int i = from; i < to && !in; ++i) {
            const double w = weight1(p + i);
            c += w;
            if (w > 0.0) last = i;
            in = w > 0.0 && c > goal;
          }
          found = last;
        }
        const int token = __shfl_sync(0xFFFFFFFFu, found, l);
        if (lane < cluster) st_cluster_s32(map_to_cta(smem_u32(&drawn[set]), lane), token);
      }
    }
    cluster_sync();  // the draw is known, the sums have been read
    const int token = total > 0.0 ? *static_cast<volatile int*>(&drawn[set]) : -1;
    // the first child that has it: every warp for itself
    int child = INT_MAX;
    if (token >= 0 && step + 1 < a.steps) {
#pragma unroll
      for (int k = 0; k < kHeldNodes; ++k) {
        const int i = 32 * k + lane;
        const uint32_t all =
            __ballot_sync(0xFFFFFFFFu, i > node && held_parent[k] == node && held_token[k] == token);
        if (all && child == INT_MAX) child = 32 * k + __ffs(all) - 1;
      }
      for (int i0 = 32 * kHeldNodes; i0 < n && child == INT_MAX; i0 += 32) {
        const int i = i0 + lane;
        const bool fits = i < n && __ldg(a.parents + row0 + i) == node && i > node &&
                          __ldg(a.tokens + row0 + i) == token;
        const uint32_t all = __ballot_sync(0xFFFFFFFFu, fits);
        if (all) child = i0 + __ffs(all) - 1;
      }
    }
    if (writes) {
      a.out_tokens[b * a.steps + step] = token;
      a.path[b * a.steps + step] = node;
    }
    going = child != INT_MAX;
    if (going) {
      node = child;
      ++kept;
    }
  }
  if (writes) a.n_accepted[b] = kept;
  if (rank == 0)
    for (int i = step + threadIdx.x; i < a.steps; i += kWalkThreads)
      a.out_tokens[b * a.steps + i] = a.path[b * a.steps + i] = -1;
}

}  // namespace

int tree_most_nodes() { return kMostNodes; }

cudaError_t launch_tree_masks(const int32_t* parents, const int32_t* q_start, int64_t T, int B, int max_q,
                              int words, int64_t* mask, int32_t* depth, int32_t* status, cudaStream_t stream) {
  if (B == 0) {  // rows of no sequence
    if (cudaError_t e = cudaMemsetAsync(mask, 0, static_cast<size_t>(T) * words * 8, stream); e != cudaSuccess) return e;
    return cudaMemsetAsync(depth, 0, static_cast<size_t>(T) * 4, stream);
  }
  MaskArgs a{};
  a.parents = parents; a.q_start = q_start; a.T = T;
  a.even = q_start ? 0 : static_cast<int>(T / B);
  a.max_q = max_q; a.B = B; a.words = words;
  a.mask = reinterpret_cast<uint64_t*>(mask); a.depth = depth; a.status = status;
  const size_t smem = ((max_q + 1) & ~1) * sizeof(int32_t) + (words <= kShortWords ? max_q * kShortWords * 8 : 0);
  tree_masks_kernel<<<static_cast<unsigned>(B), kMaskThreads, smem, stream>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_verify_tree(const void* target, int probs_bf16, const int32_t* tokens, const int32_t* parents,
                               const int32_t* q_start, const float* u, int64_t T, int B, int steps, int V,
                               int32_t* n_accepted, int32_t* out_tokens, int32_t* path, cudaStream_t stream) {
  WalkArgs a{};
  a.target = target; a.tokens = tokens; a.parents = parents; a.q_start = q_start; a.u = u;
  a.T = T; a.even = q_start ? 0 : static_cast<int>(T / B);
  a.B = B; a.steps = steps; a.V = V;
  a.n_accepted = n_accepted; a.out_tokens = out_tokens; a.path = path;
  // one block per 2048 entries, up to the portable cluster size
  int cluster = 1;
  while (cluster < kMaxCluster && cluster * 2048 < V) cluster *= 2;
  const int lanes = cluster * kWalkThreads;
  a.chunk = (((V + lanes - 1) / lanes) + 3) & ~3;
  a.wide = V % 4 == 0 && reinterpret_cast<uintptr_t>(target) % (probs_bf16 ? 8 : 16) == 0;

  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(B) * cluster));
  cfg.blockDim = dim3(kWalkThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(cluster);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return probs_bf16 ? cudaLaunchKernelEx(&cfg, verify_tree_kernel<uint16_t>, a, cluster)
                    : cudaLaunchKernelEx(&cfg, verify_tree_kernel<float>, a, cluster);
}

}  // namespace dwa
