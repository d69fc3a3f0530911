// verify_drafts.cu — verification of drafted tokens against the target's
// probabilities, and the draw that follows them.
//
// With p the target's and q the drafter's distribution, keeping draft x with
// probability min(1, p(x) / q(x)) and otherwise drawing from max(p - q, 0)
// (normalised) gives tokens distributed as p.  All tests are made in 64 bits:
// u q and p are compared exactly (24-bit factors), and the running sums are
// good to 1e-16 of their total, so the outcome does not hang on the order of
// the sums.
//
// Per sequence this reads the few tested probabilities and one row of V (p,
// and q where a draft fell), 8 V bytes at most: latency for one sequence, HBM
// for many.  A cluster of blocks shares the row, each warp a contiguous piece;
// the piece sums go through distributed shared memory, every block finds the
// piece that holds the draw, and only its warp goes over its piece again, to the row of
// 128 that the draw is in.  Eight blocks per sequence: 5.2 us for one (32000 tokens), 12.3 us
// for 64 (64400 tokens, 33 MB); with four 7.7 and 17, with two 12 and 28 (against 5.8 and 14
// then, with every row of the piece scanned).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>

#include "dwa_internal.h"
#include "sm100_ptx.cuh"

namespace dwa {

namespace {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyMaxCluster = 8;
constexpr int kBatch = 4;

struct VerifyArgs {
  const void *target, *draft;
  const int32_t* tokens;
  const float *accept_u, *sample_u;
  const int32_t* draft_lengths;
  int64_t B;
  int K, V;
  int piece;  // entries per warp, a multiple of 4
  int wide;   // rows may be read four entries at a time
  int32_t *n_accepted, *out_tokens;
};

template <typename T>
__device__ __forceinline__ float prob(const T* p) {
  if constexpr (sizeof(T) == 2)
    return __uint_as_float(static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t*>(p))) << 16);
  else
    return __ldg(p);
}

// Not a positive finite number: nothing.
__device__ __forceinline__ float mass(float x) {
  x = fmaxf(x, 0.f);  // NaN too
  return x < INFINITY ? x : 0.f;
}

// Entries i .. i + 3 of a row, zeros from V on.
template <typename T>
__device__ __forceinline__ void probs4(const T* row, int i, int V, int wide, float (&x)[4]) {
  if (wide && i < V) {
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
    for (int j = 0; j < 4; ++j) x[j] = i + j < V ? prob(row + i + j) : 0.f;
  }
}

// The weights of four entries from p's and q's values there (q's zeros where there is
// none).  `one` is the place, of 0 to 3, at which a certain drafter's q is 1.
__device__ __forceinline__ void weights4(const float (&p)[4], const float (&q)[4], int one,
                                         double (&w)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float x = mass(p[j]), y = mass(q[j]);  // compared in f32: the 64-bit units are few
    const double d = static_cast<double>(x) - static_cast<double>(y);
    w[j] = x > y && j != one ? d : 0.0;
  }
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
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

// The halves of cluster_sync.
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename T>
__global__ void __launch_bounds__(kVerifyThreads, 4)
    verify_drafts_kernel(const VerifyArgs a, const int cluster) {
  __shared__ double sums[2][kVerifyWarps];
  const int rank = static_cast<int>(blockIdx.x % cluster);
  const int64_t b = blockIdx.x / cluster;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int K = a.K, V = a.V;
  const T* target = static_cast<const T*>(a.target) + b * (K + 1) * V;
  const T* draft = a.draft ? static_cast<const T*>(a.draft) + b * K * V : nullptr;

  // How many drafts stand: every warp for itself.  The tests' values are fetched
  // without waiting for the number of drafts.
  int n = a.draft_lengths ? a.draft_lengths[b] : K;
  const double u = a.sample_u[b];
  int kept = K;
  for (int i0 = 0; i0 < K && kept == K; i0 += 32) {
    const int i = i0 + lane;
    bool stands = true;
    if (i < K) {
      const int x = a.tokens[b * K + i];
      stands = false;
      if (x >= 0 && x < V) {
        const double p = mass(prob(target + static_cast<int64_t>(i) * V + x));
        const double q = draft ? mass(prob(draft + static_cast<int64_t>(i) * V + x)) : 1.0;
        stands = static_cast<double>(a.accept_u[b * K + i]) * q < p;
      }
    }
    const uint32_t fallen = __ballot_sync(0xFFFFFFFFu, !stands);
    if (fallen) kept = i0 + __ffs(fallen) - 1;
  }
  n = min(max(n, 0), K);
  kept = min(kept, n);

  const T* p = target + static_cast<int64_t>(kept) * V;
  const T* q = kept < n && draft ? draft + static_cast<int64_t>(kept) * V : nullptr;
  // far below every entry where no drafter was certain
  int one = kept < n && !draft ? a.tokens[b * K + kept] : INT_MIN / 2;
  const int pieces = cluster * kVerifyWarps;
  const int lo = min((rank * kVerifyWarps + warp) * a.piece, V);
  const int hi = min(lo + a.piece, V);
  int token = -1;
  bool mine = false;  // this warp writes the outcome
  for (int pass = 0; pass < 2; ++pass) {
    // Rows of 128 entries, kBatch of them under way together.
    double s = 0.0;
    for (int i0 = lo; i0 < hi; i0 += 128 * kBatch) {
      float x[kBatch][4], y[kBatch][4] = {};
#pragma unroll
      for (int r = 0; r < kBatch; ++r) {
        const int i = i0 + 128 * r + 4 * lane;
        probs4(p, i, hi, a.wide, x[r]);
        if (q != nullptr) probs4(q, i, hi, a.wide, y[r]);
      }
#pragma unroll
      for (int r = 0; r < kBatch; ++r) {
        double w[4];
        weights4(x[r], y[r], one - (i0 + 128 * r + 4 * lane), w);
        s += (w[0] + w[1]) + (w[2] + w[3]);
      }
    }
    s = warp_sum(s);
    if (lane == 0) sums[pass][warp] = s;
    cluster_sync();
    // Lane l has the sums of pieces 2 l and 2 l + 1, and by a scan what lies before them;
    // every block computes the same.
    double mine0 = 0.0, mine1 = 0.0;
    if (2 * lane < pieces) {
      const int c = 2 * lane / kVerifyWarps, k = 2 * lane % kVerifyWarps;
      mine0 = ld_cluster_f64(&sums[pass][k], c);
      mine1 = ld_cluster_f64(&sums[pass][k + 1], c);
    }
    double before = mine0 + mine1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xFFFFFFFFu, before, o);
      if (lane >= o) before += y;
    }
    const double total = __shfl_sync(0xFFFFFFFFu, before, 31);
    if (total > 0.0 || pass == 1) cluster_arrive();  // this warp has read the others' sums
    if (total > 0.0) {
      const double goal = u * total;
      before -= mine0 + mine1;  // within rounding: what this decides is decided once, below
      const double mid = before + mine0;
      // the first piece whose running sum passes the goal, or the last with any weight
      const uint32_t past = __ballot_sync(0xFFFFFFFFu, (mine0 > 0.0 && mid > goal) ||
                                                           (mine1 > 0.0 && mid + mine1 > goal));
      const uint32_t some = __ballot_sync(0xFFFFFFFFu, mine0 > 0.0 || mine1 > 0.0);
      const int src = past ? __ffs(past) - 1 : 31 - __clz(some);
      const bool first = past ? mine0 > 0.0 && mid > goal : !(mine1 > 0.0);
      const int at = __shfl_sync(0xFFFFFFFFu, 2 * lane + (first ? 0 : 1), src);
      double run = __shfl_sync(0xFFFFFFFFu, first ? before : mid, src);
      if (at == rank * kVerifyWarps + warp) {
        mine = true;
        // the row (of 128 entries) that the draw is in; where rounding keeps the running sum at
        // the goal to the end, the last with weight
        int i = -1;
        bool in = false;
        for (int i0 = lo; i0 < hi && !in; i0 += 128 * kBatch) {
          float x[kBatch][4], y[kBatch][4] = {};
          double row[kBatch];
#pragma unroll
          for (int r = 0; r < kBatch; ++r) {
            const int k = i0 + 128 * r + 4 * lane;
            probs4(p, k, hi, a.wide, x[r]);
            if (q != nullptr) probs4(q, k, hi, a.wide, y[r]);
          }
#pragma unroll
          for (int r = 0; r < kBatch; ++r) {
            double w[4];
            weights4(x[r], y[r], one - (i0 + 128 * r + 4 * lane), w);
            row[r] = warp_sum((w[0] + w[1]) + (w[2] + w[3]));
          }
#pragma unroll
          for (int r = 0; r < kBatch; ++r)
            if (!in && row[r] > 0.0) {
              i = i0 + 128 * r + 4 * lane;
              in = run + row[r] > goal;
              if (!in) run += row[r];
            }
        }
        // in it the first entry whose running sum passes the goal, or the last with weight
        float x[4], y[4] = {};
        double w[4];
        probs4(p, i, hi, a.wide, x);
        if (q != nullptr) probs4(q, i, hi, a.wide, y);
        weights4(x, y, one - i, w);
        const double four = (w[0] + w[1]) + (w[2] + w[3]);
        double incl = four;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double z = __shfl_up_sync(0xFFFFFFFFu, incl, o);
          if (lane >= o) incl += z;
        }
        const uint32_t hit = __ballot_sync(0xFFFFFFFFu, in && four > 0.0 && run + incl > goal);
        const uint32_t any = __ballot_sync(0xFFFFFFFFu, four > 0.0);
        int j = w[3] > 0.0 ? 3 : w[2] > 0.0 ? 2 : w[1] > 0.0 ? 1 : 0;  // the last with weight
        if (hit) {
          const double c = run + (incl - four);
#pragma unroll
          for (int k = 2; k >= 0; --k) {
            double head = c + w[0];
            if (k > 0) head += w[1];
            if (k > 1) head += w[2];
            if (w[k] > 0.0 && head > goal) j = k;
          }
        }
        token = __shfl_sync(0xFFFFFFFFu, i + j, hit ? __ffs(hit) - 1 : 31 - __clz(any));
      }
      break;
    }
    if (pass == 1 && rank == 0 && warp == 0) mine = true;  // no mass anywhere: token -1
    // nothing left of p - q: draw from p
    q = nullptr;
    one = INT_MIN / 2;
  }
  if (mine) {
    if (lane == 0) a.n_accepted[b] = kept;
    for (int i = lane; i <= K; i += 32)
      a.out_tokens[b * (K + 1) + i] = i < kept ? a.tokens[b * K + i] : i == kept ? token : -1;
  }
  cluster_wait();  // no block leaves while another reads its sums
}

}  // namespace

cudaError_t launch_verify_drafts(const void* target, const void* draft, int probs_bf16,
                                 const int32_t* tokens, const float* accept_u, const float* sample_u,
                                 const int32_t* draft_lengths, int64_t B, int K, int V,
                                 int32_t* n_accepted, int32_t* out_tokens, cudaStream_t stream) {
  VerifyArgs a{};
  a.target = target; a.draft = draft; a.tokens = tokens;
  a.accept_u = accept_u; a.sample_u = sample_u; a.draft_lengths = draft_lengths;
  a.B = B; a.K = K; a.V = V;
  a.n_accepted = n_accepted; a.out_tokens = out_tokens;
  // one block per 2048 entries, up to the portable cluster size
  int cluster = 1;
  while (cluster < kVerifyMaxCluster && cluster * 2048 < V) cluster *= 2;
  const int pieces = cluster * kVerifyWarps;
  a.piece = (((V + pieces - 1) / pieces) + 3) & ~3;
  const uintptr_t at = reinterpret_cast<uintptr_t>(target) | reinterpret_cast<uintptr_t>(draft);
  a.wide = V % 4 == 0 && at % (probs_bf16 ? 8 : 16) == 0;

  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(B * cluster));
  cfg.blockDim = dim3(kVerifyThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(cluster);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return probs_bf16 ? cudaLaunchKernelEx(&cfg, verify_drafts_kernel<uint16_t>, a, cluster)
                    : cudaLaunchKernelEx(&cfg, verify_drafts_kernel<float>, a, cluster);
}

}  // namespace dwa
