// paged_attention.cu — attention of a few new rows per key/value head over the
// paged cache: decoding steps and drafted tokens (and any other chunk, slowly).
//
// A row is one (new token, query head); the rows of a key/value head are
// token-major, its `group` query heads side by side.  Bound by HBM: each
// cached key and value is read once for up to 8 NT rows.
//
// The products are transposed so that the few rows lie along the 8 columns of
// mma.m16n8k16: S^T = K Q^T takes 16 keys by 8 rows, O^T += V^T P^T takes 16
// channels by 8 rows.  Both big operands go from global memory straight into
// the fragments, without shared memory or a barrier: the order of the
// summation index and of the output channels is free, so every lane loads 16
// neighbouring bytes and whatever channels those are take the places the
// fragment gives them (Q is loaded in the same order; the output channel of
// each accumulator is known).  P^T is turned between the products by movmatrix.
// Each warp keeps the next block's keys in flight while it works on this
// block's values and the other way round.
//
// The context of one (sequence, head) is split over the warps of a cluster of
// blocks, 16 or 32 keys at a time in turn, and joined through shared and
// distributed shared memory in one launch, in a fixed order.
//
// e4m3 codes become bf16 exactly: moving the 7 magnitude bits down by four
// gives a bf16 of 2^-120 times the value (subnormals too), one product with
// 2^120 puts it right.  The keys' scales multiply the scores, the values'
// scales the probabilities.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "dwa_internal.h"
#include "paged_attention.cuh"
#include "sm100_ptx.cuh"

namespace dwa {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxCluster = 8;
constexpr int kFewRows = 32;  // per key/value head; more go to the tcgen05 kernel

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Bytes 1 and 3 of w, e4m3, as a pair of bf16.
__device__ __forceinline__ uint32_t e4m3_bytes13(uint32_t w) {
  const uint32_t small = ((w >> 4) & 0x07F007F0u) | (w & 0x80008000u);
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(small), "r"(0x7B807B80u));  // 2^120
  return r;
}

// 16 bytes that are read once.
__device__ __forceinline__ uint4 ld16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld8(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];"
               : "=r"(v.x), "=r"(v.y)
               : "l"(p));
  return v;
}

// The halves of w (the values of one key at two channels) that are not finite
// become 0 and note the key.
__device__ __forceinline__ uint32_t only_finite(uint32_t w, int key, int* first_lo, int* first_hi) {
  if ((w & 0x7F80u) == 0x7F80u) {
    atomicMin(first_lo, key);
    w &= 0xFFFF0000u;
  }
  if ((w & 0x7F800000u) == 0x7F800000u) {
    atomicMin(first_hi, key);
    w &= 0x0000FFFFu;
  }
  return w;
}

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

// kE4m3: 8-bit cache.  DP: d rounded up to 64 or 128.  NT: column tiles of 8 rows.
template <bool kE4m3, int DP, int NT>
struct Cfg {
  static constexpr int kSub = kE4m3 ? 2 : 1;     // 16-key tiles per block, so that a block is 4 KB
  static constexpr int kKeys = 16 * kSub;
  static constexpr int kSteps = DP / 16;         // k-steps of S, channel tiles of O
  static constexpr int kRows = 8 * NT;
  // 16-byte chunks of a key row held by one lane (of the 4 that share it)
  static constexpr int kChunksK = kE4m3 ? DP / 64 : DP / 32;
  static constexpr int kWordsK = 4 * kChunksK;   // per key
  // words of a value row held by one lane (of the 8 that share it)
  static constexpr int kWordsV = kE4m3 ? DP / 32 : DP / 16;
};

template <bool kE4m3, int DP, int NT>
__global__ void __launch_bounds__(kThreads)
    paged_rows_kernel(const PagedArgs a, const int row_groups, const int cluster) {
  using C = Cfg<kE4m3, DP, NT>;
  // one partial per warp, then (in warp 0's place) one per block
  __shared__ __align__(16) float part_o[kWarps][C::kRows][DP];
  __shared__ float part_m[kWarps][C::kRows], part_l[kWarps][C::kRows];
  __shared__ float block_m[C::kRows], block_l[C::kRows];
  __shared__ int first_bad[DP];  // least key with a value that is not finite, by channel

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  int64_t unit = blockIdx.x / cluster;
  const int split = static_cast<int>(blockIdx.x % cluster);
  const int rg = static_cast<int>(unit % row_groups);
  unit /= row_groups;
  const int hk = static_cast<int>(unit % a.H_kv);
  const int b = static_cast<int>(unit / a.H_kv);

  PagedSeq seq = paged_seq(a, b);
  if (seq.bad && hk == 0 && rg == 0 && split == 0 && threadIdx.x == 0) paged_report(a.status);
  const int64_t all_rows = static_cast<int64_t>(seq.n) * a.group;
  const int64_t r0 = static_cast<int64_t>(rg) * C::kRows;
  if (r0 >= all_rows) return;  // the whole cluster
  if (seq.bad) {
    // every group its own rows, and those row_groups groups further on: a
    // sequence with more rows than max_q has more than there are groups
    const int64_t stride = static_cast<int64_t>(row_groups) * C::kRows;
    for (int64_t base = r0; base < all_rows; base += stride)
      for (int i = split * kThreads + threadIdx.x; i < C::kRows * a.d; i += cluster * kThreads) {
        const int64_t row = base + i / a.d;
        if (row < all_rows)
          a.out[(seq.row0 + row / a.group) * a.out_ld +
                (static_cast<int64_t>(hk) * a.group + row % a.group) * a.d + i % a.d] = 0x7FC0u;
      }
    return;
  }
  const int rows = static_cast<int>(min(all_rows - r0, static_cast<int64_t>(C::kRows)));
  const int vis_min = paged_visible(seq, static_cast<int>(r0 / a.group));
  const int vis_max = paged_visible(seq, static_cast<int>((r0 + rows - 1) / a.group));

  for (int i = threadIdx.x; i < DP; i += kThreads) first_bad[i] = 0x7FFFFFFF;
  __syncthreads();

  // Q^T fragments: lane (g, t) holds row 8 nt + g at the channels its key chunks have
  uint32_t qf[NT][C::kSteps][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = 8 * nt + g;
    const int64_t row = r0 + r;
    const uint16_t* src = a.q + (seq.row0 + row / a.group) * a.q_ld +
                          (static_cast<int64_t>(hk) * a.group + row % a.group) * a.d;
#pragma unroll
    for (int c = 0; c < C::kChunksK; ++c) {
      const int at = (4 * c + t) * (kE4m3 ? 16 : 8);
      uint32_t w[kE4m3 ? 8 : 4];
#pragma unroll
      for (int i = 0; i < (kE4m3 ? 2 : 1); ++i) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (r < rows && at < a.d) x = __ldg(reinterpret_cast<const uint4*>(src + at) + i);
        w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
      }
      if constexpr (kE4m3) {
        // a word of four codes gives its bytes 0 and 2, then 1 and 3
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          qf[nt][4 * c + i][0] = __byte_perm(w[2 * i], w[2 * i + 1], 0x5410);
          qf[nt][4 * c + i][1] = __byte_perm(w[2 * i], w[2 * i + 1], 0x7632);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) qf[nt][2 * c + (i >> 1)][i & 1] = w[i];
      }
    }
  }
  // tokens each of this lane's columns (rows 8 nt + 2 t and + 1) may see
  int vis[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = 8 * nt + 2 * t + j;
      vis[nt][j] = r < rows ? paged_visible(seq, static_cast<int>((r0 + r) / a.group)) : 0;
    }

  float o[NT][C::kSteps][4] = {};
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) { m[nt][0] = m[nt][1] = -INFINITY; l[nt][0] = l[nt][1] = 0.f; }

  const int n_blocks = (vis_max + C::kKeys - 1) / C::kKeys;
  const int step = cluster * kWarps;
  const int page_mask = (1 << a.page_log2) - 1;
  const int32_t* table = a.table + static_cast<int64_t>(b) * a.ld_table;
  const int esize = kE4m3 ? 1 : 2;
  bool bad_page = false;

  uint32_t kw[C::kSub][2][C::kWordsK], vw[C::kSub][4][C::kWordsV];
  float ks[C::kSub][2], vs[C::kSub][2];

  // first vector (row of d) of a 16-key tile, -1 where the tile has no page
  auto tile_vector = [&](int key, int64_t* scale_at) -> int64_t {
    if (key >= vis_max) return -1;
    const int page = __ldg(table + (key >> a.page_log2));
    if (page < 0 || page >= a.n_pages) {
      bad_page = true;
      return -1;
    }
    const int64_t in_page = (static_cast<int64_t>(hk) << a.page_log2) + (key & page_mask);
    *scale_at = page * a.ld_scale_page + in_page;
    return page * a.ld_page + in_page * a.d;
  };
  auto load_k = [&](int block) {
#pragma unroll
    for (int s = 0; s < C::kSub; ++s) {
      int64_t scale_at = 0;
      const int64_t at = tile_vector(block * C::kKeys + 16 * s, &scale_at);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const char* row = static_cast<const char*>(a.k) + (at + static_cast<int64_t>(g + 8 * i) * a.d) * esize;
#pragma unroll
        for (int c = 0; c < C::kChunksK; ++c) {
          const int chunk = 4 * c + t;
          uint4 x = make_uint4(0, 0, 0, 0);
          if (at >= 0 && chunk * 16 < a.d * esize) x = ld16(row + 16 * chunk);
          kw[s][i][4 * c] = x.x; kw[s][i][4 * c + 1] = x.y;
          kw[s][i][4 * c + 2] = x.z; kw[s][i][4 * c + 3] = x.w;
        }
        if constexpr (kE4m3) {
          ks[s][i] = at >= 0 ? __ldg(a.k_scale + scale_at + g + 8 * i) : 0.f;
          vs[s][i] = at >= 0 ? __ldg(a.v_scale + scale_at + g + 8 * i) : 0.f;
        }
      }
    }
  };
  auto load_v = [&](int block) {
#pragma unroll
    for (int s = 0; s < C::kSub; ++s) {
      int64_t scale_at = 0;
      const int64_t at = tile_vector(block * C::kKeys + 16 * s, &scale_at);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 2 * t + (i & 1) + 8 * (i >> 1);
        const char* row = static_cast<const char*>(a.v) + (at + static_cast<int64_t>(key) * a.d) * esize;
        if constexpr (C::kWordsV == 2) {  // 8 codes
          uint2 x = make_uint2(0, 0);
          if (at >= 0 && 8 * g < a.d) x = ld8(row + 8 * g);
          vw[s][i][0] = x.x; vw[s][i][1] = x.y;
        } else {
#pragma unroll
          for (int c = 0; c < C::kWordsV / 4; ++c) {
            const int chunk = 8 * c + g;
            uint4 x = make_uint4(0, 0, 0, 0);
            if (at >= 0 && chunk * 16 < a.d * esize) x = ld16(row + 16 * chunk);
            vw[s][i][4 * c] = x.x; vw[s][i][4 * c + 1] = x.y;
            vw[s][i][4 * c + 2] = x.z; vw[s][i][4 * c + 3] = x.w;
          }
        }
      }
    }
  };

  int block = split * kWarps + warp;
  if (block < n_blocks) {
    load_k(block);
    load_v(block);
  }
  for (; block < n_blocks; block += step) {
    const int key0 = block * C::kKeys;
    const int next = block + step;
    float s[C::kSub][NT][4] = {};
#pragma unroll
    for (int u = 0; u < C::kSub; ++u)
#pragma unroll
      for (int k = 0; k < C::kSteps; ++k) {
        uint32_t f[4];
        if constexpr (kE4m3) {
          f[0] = e4m3_bytes13(kw[u][0][k] << 8);
          f[1] = e4m3_bytes13(kw[u][1][k] << 8);
          f[2] = e4m3_bytes13(kw[u][0][k]);
          f[3] = e4m3_bytes13(kw[u][1][k]);
        } else {
          f[0] = kw[u][0][2 * k]; f[1] = kw[u][1][2 * k];
          f[2] = kw[u][0][2 * k + 1]; f[3] = kw[u][1][2 * k + 1];
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_bf16(s[u][nt], f, qf[nt][k][0], qf[nt][k][1]);
      }
    float sk[C::kSub][2], sv[C::kSub][2];
#pragma unroll
    for (int u = 0; u < C::kSub; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        sk[u][i] = kE4m3 ? ks[u][i] * a.scale_log2 : a.scale_log2;
        sv[u][i] = kE4m3 ? vs[u][i] : 1.f;
      }
    if (next < n_blocks) load_k(next);

    // scores in units of log2, masked; the columns' maxima over the block
    const bool edge = key0 + C::kKeys > vis_min;
    uint32_t pb[C::kSub][NT][2];
    bool moved = false;
    float shrink[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float top = m[nt][j];
#pragma unroll
        for (int u = 0; u < C::kSub; ++u)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float x = s[u][nt][2 * i + j] * sk[u][i];
            if (edge && key0 + 16 * u + 8 * i + g >= vis[nt][j]) x = -INFINITY;
            s[u][nt][2 * i + j] = x;
            top = fmaxf(top, x);
          }
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
        const float was = m[nt][j];
        shrink[nt][j] = 1.f;
        if (top > was) {
          shrink[nt][j] = was == -INFINITY ? 0.f : fast_exp2(was - top);
          m[nt][j] = top;
          moved = true;
        }
        const float base = m[nt][j] == -INFINITY ? 0.f : m[nt][j];
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < C::kSub; ++u)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float p = fast_exp2(s[u][nt][2 * i + j] - base);
            sum += p;
            // a masked key's scale may be anything: its weight is 0, not 0 times that
            s[u][nt][2 * i + j] =
                edge && key0 + 16 * u + 8 * i + g >= vis[nt][j] ? 0.f : p * sv[u][i];
          }
        l[nt][j] = l[nt][j] * shrink[nt][j] + sum;
      }
    // probabilities are rounded to bf16 for the tensor cores (2^-9 each, averaged
    // over the keys); their sum l is kept in f32 from the unrounded ones
#pragma unroll
    for (int u = 0; u < C::kSub; ++u)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          pb[u][nt][i] = transpose8x8(pack_bf16(s[u][nt][2 * i], s[u][nt][2 * i + 1]));
    if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < C::kSteps; ++k)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[nt][k][j] *= shrink[nt][j & 1];
    }
    if constexpr (!kE4m3) {
      if (edge) {  // keys that some row may not see: their values must not reach it as 0 * NaN
#pragma unroll
        for (int u = 0; u < C::kSub; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = key0 + 16 * u + 2 * t + (i & 1) + 8 * (i >> 1);
#pragma unroll
            for (int w = 0; w < C::kWordsV; ++w) {
              const int ch = 8 * (8 * (w >> 2) + g) + 2 * (w & 3);
              if (key >= vis_max) vw[u][i][w] = 0;
              else if (key >= vis_min)
                vw[u][i][w] = only_finite(vw[u][i][w], key, &first_bad[ch], &first_bad[ch + 1]);
            }
          }
      }
    }
#pragma unroll
    for (int u = 0; u < C::kSub; ++u)
#pragma unroll
      for (int k = 0; k < C::kSteps; ++k) {
        uint32_t f[4];
        if constexpr (kE4m3) {
          // tile k: channel 2 k of the chunk in rows 0..7, 2 k + 1 in rows 8..15
          const int w = k >> 1;
          const uint32_t lo = (k & 1) ? 0x6020u : 0x4000u;  // byte 2 (k & 1) of both keys
          const uint32_t hi = (k & 1) ? 0x7030u : 0x5010u;
          f[0] = e4m3_bytes13(__byte_perm(vw[u][0][w], vw[u][1][w], lo));
          f[1] = e4m3_bytes13(__byte_perm(vw[u][0][w], vw[u][1][w], hi));
          f[2] = e4m3_bytes13(__byte_perm(vw[u][2][w], vw[u][3][w], lo));
          f[3] = e4m3_bytes13(__byte_perm(vw[u][2][w], vw[u][3][w], hi));
        } else {
          f[0] = __byte_perm(vw[u][0][k], vw[u][1][k], 0x5410);
          f[1] = __byte_perm(vw[u][0][k], vw[u][1][k], 0x7632);
          f[2] = __byte_perm(vw[u][2][k], vw[u][3][k], 0x5410);
          f[3] = __byte_perm(vw[u][2][k], vw[u][3][k], 0x7632);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_bf16(o[nt][k], f, pb[u][nt][0], pb[u][nt][1]);
      }
    if (next < n_blocks) load_v(next);
  }
  if (__any_sync(0xFFFFFFFFu, bad_page)) {
    if (lane == 0) paged_report(a.status);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) l[nt][0] = l[nt][1] = __uint_as_float(0x7FC00000u);
  }

  // this warp's partial
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float x = l[nt][j];
      x += __shfl_xor_sync(0xFFFFFFFFu, x, 4);
      x += __shfl_xor_sync(0xFFFFFFFFu, x, 8);
      x += __shfl_xor_sync(0xFFFFFFFFu, x, 16);
      const int r = 8 * nt + 2 * t + j;
      if (g == 0) {
        part_m[warp][r] = m[nt][j];
        part_l[warp][r] = x;
      }
      if (r < rows) {
#pragma unroll
        for (int k = 0; k < C::kSteps; ++k) {
          // channels 2 k' and 2 k' + 1 of this lane's chunk
          const int ch = kE4m3 ? (DP / 8) * g + 2 * k : 8 * (8 * (k >> 2) + g) + 2 * (k & 3);
          *reinterpret_cast<float2*>(&part_o[warp][r][ch]) =
              make_float2(o[nt][k][j], o[nt][k][2 + j]);
        }
      }
    }
  __syncthreads();
  // the block's: row by row, warps in order
  for (int i = threadIdx.x; i < rows * (DP / 2); i += kThreads) {
    const int r = i / (DP / 2), ch = 2 * (i % (DP / 2));
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, part_m[w][r]);
    float sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = part_m[w][r] == -INFINITY ? 0.f : fast_exp2(part_m[w][r] - top);
      // a warp without keys has l = 0 (or NaN, after a bad page, which has to stay)
      sum += part_m[w][r] == -INFINITY ? part_l[w][r] : f * part_l[w][r];
      const float2 p = *reinterpret_cast<const float2*>(&part_o[w][r][ch]);
      x += f * p.x;
      y += f * p.y;
    }
    if (ch == 0) {
      block_m[r] = top;
      block_l[r] = sum;
    }
    // only this thread reads or writes these entries
    *reinterpret_cast<float2*>(&part_o[0][r][ch]) = make_float2(x, y);
  }
  cluster_sync();
  for (int i = split * kThreads + threadIdx.x; i < rows * (DP / 2); i += cluster * kThreads) {
    const int r = i / (DP / 2), ch = 2 * (i % (DP / 2));
    if (ch >= a.d) continue;
    float ms[kMaxCluster], ls[kMaxCluster];
    float2 os[kMaxCluster];
    int bad0 = 0x7FFFFFFF, bad1 = 0x7FFFFFFF;
    float top = -INFINITY;
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) {
      ms[c] = -INFINITY;
      if (c < cluster) {
        ms[c] = ld_cluster_f32(&block_m[r], c);
        ls[c] = ld_cluster_f32(&block_l[r], c);
        os[c] = ld_cluster_f32x2(&part_o[0][r][ch], c);
        if (!kE4m3) {
          bad0 = min(bad0, ld_cluster_s32(&first_bad[ch], c));
          bad1 = min(bad1, ld_cluster_s32(&first_bad[ch + 1], c));
        }
        top = fmaxf(top, ms[c]);
      }
    }
    float sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c)
      if (c < cluster) {
        const float f = ms[c] == -INFINITY ? 0.f : fast_exp2(ms[c] - top);
        sum += ms[c] == -INFINITY ? ls[c] : f * ls[c];
        x += f * os[c].x;
        y += f * os[c].y;
      }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t row = r0 + r;
    const int seen = paged_visible(seq, static_cast<int>(row / a.group));
    x = bad0 < seen ? __uint_as_float(0x7FC00000u) : x * inv;
    y = bad1 < seen ? __uint_as_float(0x7FC00000u) : y * inv;
    *reinterpret_cast<uint32_t*>(a.out + (seq.row0 + row / a.group) * a.out_ld +
                                 (static_cast<int64_t>(hk) * a.group + row % a.group) * a.d + ch) =
        pack_bf16(x, y);
  }
  cluster_sync();  // no block leaves while another reads its partial
}

template <bool kE4m3, int DP, int NT>
cudaError_t launch_rows(const PagedArgs& a, int cluster, cudaStream_t stream) {
  const int64_t most_rows = static_cast<int64_t>(a.max_q) * a.group;
  const int row_groups = static_cast<int>((most_rows + 8 * NT - 1) / (8 * NT));
  const int64_t blocks = static_cast<int64_t>(a.B) * a.H_kv * row_groups * cluster;
  if (blocks > 0x7FFFFFFFll) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(cluster);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_rows_kernel<kE4m3, DP, NT>, a, row_groups, cluster);
}

template <bool kE4m3, int DP>
cudaError_t launch_rows_nt(const PagedArgs& a, cudaStream_t stream) {
  const int64_t most_rows = static_cast<int64_t>(a.max_q) * a.group;
  const int nt = most_rows <= 8 ? 1 : 2;
  const int64_t units = static_cast<int64_t>(a.B) * a.H_kv * ((most_rows + 8 * nt - 1) / (8 * nt));
  // split a context until there are some blocks for every SM, while each warp
  // keeps two blocks of keys
  const int64_t keys = static_cast<int64_t>(a.max_pages) << a.page_log2;
  int cluster = 1;
  while (cluster < kMaxCluster && units * cluster < 4ll * device_sm_count() &&
         keys > 2ll * cluster * kWarps * Cfg<kE4m3, DP, 1>::kKeys)
    cluster *= 2;
  return nt == 1 ? launch_rows<kE4m3, DP, 1>(a, cluster, stream)
                 : launch_rows<kE4m3, DP, 2>(a, cluster, stream);
}

}  // namespace

cudaError_t launch_paged_attention(const PagedArgs& a, cudaStream_t stream) {
  if (static_cast<int64_t>(a.max_q) * a.group > kFewRows) return launch_paged_attention_mma(a, stream);
  const bool e4m3 = a.k_scale != nullptr;
  if (a.d <= 64) return e4m3 ? launch_rows_nt<true, 64>(a, stream) : launch_rows_nt<false, 64>(a, stream);
  return e4m3 ? launch_rows_nt<true, 128>(a, stream) : launch_rows_nt<false, 128>(a, stream);
}

}  // namespace dwa
