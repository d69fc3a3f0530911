// paged_attention.cu — attention of a few new rows per key/value head over the
// paged cache: decoding steps and drafted tokens.
//
// A row is one (new token, query head); the rows of a key/value head are
// token-major, its `group` query heads side by side.  Bound by HBM: each
// cached key and value is read once for up to 16 rows.
//
// The products are transposed so that the few rows lie along the 8 columns of
// mma.m16n8k16: S^T = K Q^T takes 16 keys by 8 rows, O^T += V^T P^T takes 16
// channels by 8 rows.  The order of the summation index, of the keys in a tile and
// of the output channels is free, so every lane takes its part of the big operands
// as 16 neighbouring bytes and whatever channels those are get the places the
// fragment has for them (Q is loaded in the same order; the channel of each
// accumulator is known).  P^T is turned between the products by movmatrix.
//
// Each warp works alone on blocks of 16 (bf16) or 32 (e4m3) keys, which its own
// ring of TMA copies brings, up to 8 KB at a time and two in flight, three blocks of four warps
// to an SM.  (Loaded into registers, one block ahead: 137 us instead of 83 for 64 ragged
// sequences of 16 heads of 128, bf16, 0.52 GB: 6.2 TB/s.)
// The context of one (sequence, head) is split over the warps of a cluster of
// blocks, block by block in turn, and joined through shared and distributed shared
// memory in one launch, in a fixed order.
//
// bf16 caches: P is used as the sum of two bf16 parts, so that only the result's
// rounding is left.  e4m3 caches: codes become fp16 exactly, Q is scaled per row by
// a power of two into fp16 (a part below 2^-37 of its largest is lost), the keys' scales multiply the scores,
// and P times the values' scales, relative to a power of two of the row's own, is rounded
// to fp16 (2^-11).  (Relative to one above every value's scale, a row loses its bits to
// values that it may not see, or sees without weight.)
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "dwa_internal.h"
#include "paged_attention.cuh"
#include "sm100_ptx.cuh"

namespace dwa {

namespace {

constexpr int kMaxCluster = 8;

template <bool kF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (kF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// The halves of w (the values of one key at two channels) that are not finite
// become 0 and note the key (of a tree the node, 0 to 15).
template <bool kTree>
__device__ __forceinline__ uint32_t only_finite(uint32_t w, int key, int* first_lo, int* first_hi) {
  auto note = [&](int* at) {
    if constexpr (kTree) atomicOr(at, 1 << key);
    else atomicMin(at, key);
  };
  if ((w & 0x7F80u) == 0x7F80u) {
    note(first_lo);
    w &= 0xFFFF0000u;
  }
  if ((w & 0x7F800000u) == 0x7F800000u) {
    note(first_hi);
    w &= 0x0000FFFFu;
  }
  return w;
}

// kE4m3: 8-bit cache.  DP: d rounded up to 64 or 128.  NT: column tiles of 8 rows.
// W: warps per block.
template <bool kE4m3, int DP, int NT, int W>
struct RowsCfg {
  static constexpr int kWarps = W, kThreads = 32 * W;
  static constexpr int kSub = kE4m3 ? 2 : 1;      // 16-key tiles per block
  static constexpr int kKeys = 16 * kSub;
  static constexpr int kSteps = DP / 16;          // k-steps of S, channel tiles of O
  static constexpr int kRows = 8 * NT;            // kFewRows at most
  static constexpr int kRowBytes = kE4m3 ? DP : 128;              // of a TMA box
  static constexpr int kHalves = kE4m3 ? 1 : DP / 64;             // boxes side by side
  static constexpr int kBoxBytes = 16 * kRowBytes;
  static constexpr int kBoxes = kSub * kHalves;                   // of K; as many of V
  static constexpr int kStageBytes = 2 * kBoxes * kBoxBytes;
  static constexpr int kStages = kE4m3 || DP == 128 ? 2 : 3;
  static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
  static constexpr int kPartBytes = kWarps * kRows * DP * 4;      // takes the ring's place
  static constexpr int kSmem = 1024 + (kRingBytes > kPartBytes ? kRingBytes : kPartBytes);
  static constexpr int kScales = kE4m3 ? 32 : 1;  // keys with a scale per block
};

// Keys of the rows of a 16-key tile: row r of the fragment is key row_key(r & 7) + (r & 8).
// With 128-byte rows swizzled by TMA this order keeps the 16-byte reads of both
// operands free of bank conflicts: neighbouring rows differ in bit 2 (K), every second
// row's keys differ above bit 0 (V).
__device__ __forceinline__ int row_key(int r) { return (0x37156240 >> (4 * r)) & 7; }

// The same for bf16 rows that lie one behind the other, an odd number of 32 bytes each:
// neighbouring rows' keys differ by 2 and every second row's are all different, modulo 4.
// (Rows of codes, an odd number of 16 bytes, do in their own order.)
__device__ __forceinline__ int linear_key(int r) { return r & 1 ? ((r >> 1) + 2) % 4 + 4 : r >> 1; }

__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ void copy_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// This thread's arrival on `bar`, once its cp.async copies so far have landed.
__device__ __forceinline__ void arrive_when_copied(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// kLinear: the rows of a block lie one behind the other, as in the page.  kTree: the new tokens
// (16 at most) see what the tree's masks say.
template <bool kE4m3, int DP, int NT, int W, bool kLinear, bool kTree>
__global__ void __launch_bounds__(32 * W, W == 8 ? 1 : NT == 1 ? 3 : 2)
    paged_rows_kernel(const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const PagedArgs a,
                      const int cluster, const int wide, const int rank) {
  using C = RowsCfg<kE4m3, DP, NT, W>;
  constexpr int kWarps = W, kThreads = 32 * W;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full_bar[kWarps][C::kStages];
  __shared__ float scales[kWarps][C::kStages][2][C::kScales];  // keys', values'
  __shared__ float part_m[kWarps][C::kRows], part_l[kWarps][C::kRows];
  __shared__ float block_m[C::kRows], block_l[C::kRows];
  // least key with a value that is not finite, by channel; trees: the nodes with one, as bits
  __shared__ int first_bad[DP];
  constexpr int kNoBad = kTree ? 0 : 0x7FFFFFFF;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  // one partial per warp, then (in warp 0's place) one per block
  float* const part_o = reinterpret_cast<float*>(smem_raw + (base - smem_u32(smem_raw)));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t unit = blockIdx.x / cluster;  // the grid has 32 bits
  const int split = static_cast<int>(blockIdx.x % cluster);
  const int hk = static_cast<int>(unit % a.H_kv);
  // the longest sequences first, where blocks share SMs or wait for one
  __shared__ int costs[kMostRanked], start_of[kMostRanked + 1], found;
  int b = static_cast<int>(unit / a.H_kv);
  PagedSeq seq;
  if (rank && a.B > 1 && a.B <= kMostRanked) {  // what is read for it is not read again
    for (int i = threadIdx.x; i <= a.B; i += kThreads) start_of[i] = q_start_at(a, i);
    b = ranked(a.B, b, costs, &found, [&](int i) { return __ldg(a.lengths + i); });
    seq = paged_seq(a, b, start_of[b], start_of[b + 1], costs[b]);
  } else {
    seq = paged_seq(a, b);
  }
  if (seq.bad && hk == 0 && split == 0 && threadIdx.x == 0) paged_report(a.status);
  const int64_t all_rows = static_cast<int64_t>(seq.n) * a.group;
  if (all_rows == 0) return;  // the whole cluster
  if (seq.bad) {  // it may have more rows than max_q
    for (int64_t i = split * kThreads + threadIdx.x; i < all_rows * a.d; i += cluster * kThreads) {
      const int64_t row = i / a.d;
      a.out[(seq.row0 + row / a.group) * a.out_ld +
            (static_cast<int64_t>(hk) * a.group + row % a.group) * a.d + i % a.d] = 0x7FC0u;
    }
    return;
  }
  const int rows = static_cast<int>(all_rows);  // max_q bounds them to kRows
  const int prefix = tree_prefix(seq);
  const int vis_min = kTree ? max(prefix, 0) : paged_visible(seq, 0);
  const int vis_max = kTree ? seq.length : paged_visible(seq, seq.n - 1);
  // Whether a row sees a key at the edge, of what paged_visible (or the tree's mask) says of it.
  auto sees = [&](int key, int vis) -> bool {
    if constexpr (kTree)
      return key < vis_min || (key < vis_max && ((static_cast<uint32_t>(vis) >> (key - prefix)) & 1u));
    else
      return key < vis;
  };
  auto row_sees = [&](uint32_t token) -> int {
    if constexpr (kTree) return static_cast<int>(__ldg(a.tree + (seq.row0 + token) * a.tree_words));
    else return paged_visible(seq, token);
  };

  // ------------------------------------------------ Q^T fragments, on their way
  // lane (g, t) holds row 8 nt + g at the channels its key chunks have
  constexpr int kChunk = kE4m3 ? 16 : 8;            // channels per 16 bytes
  constexpr int kChunksK = DP / (4 * kChunk);       // of a key row, per lane
  uint32_t qf[NT][C::kSteps][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = 8 * nt + g;
    const uint32_t row = r, token = row_token(row, a.group);
    const uint16_t* src = a.q + (seq.row0 + token) * a.q_ld +
                          (static_cast<int64_t>(hk) * a.group + row - token * a.group) * a.d;
#pragma unroll
    for (int c = 0; c < kChunksK; ++c)
#pragma unroll
      for (int i = 0; i < kChunk / 8; ++i) {
        const int at = (4 * c + t) * kChunk + 8 * i;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (r < rows && at < a.d) x = __ldg(reinterpret_cast<const uint4*>(src + at));
        const int k = (c * kChunk + 8 * i) / 4;
        qf[nt][k][0] = x.x; qf[nt][k][1] = x.y;
        qf[nt][k + 1][0] = x.z; qf[nt][k + 1][1] = x.w;
      }
  }

  // ------------------------------------------------ this warp's ring
  const uint32_t ring = base + warp * C::kStages * C::kStageBytes;
  const uint32_t bar0 = smem_u32(&full_bar[warp][0]);
  if (lane == 0) {
    for (int i = 0; i < C::kStages; ++i) mbar_init(bar0 + 8 * i, kE4m3 ? 33 : 1);  // with every lane's scales
    fence_mbar_init();
  }
  for (int i = threadIdx.x; i < DP; i += kThreads) first_bad[i] = kNoBad;
  __syncthreads();

  const int n_blocks = (vis_max + C::kKeys - 1) / C::kKeys;
  const int step = cluster * kWarps;
  const int page_mask = (1 << a.page_log2) - 1;
  const int32_t* table = a.table + static_cast<int64_t>(b) * a.ld_table;
  bool bad_page = false;
  // The first lane brings a block: a box of 16 keys by 128 bytes for each half of the
  // channels (or 32 keys, or both halves, as the map has them), K then V.  What a copy costs
  // is its issue, so they are few and their operands the same in all lanes.  An e4m3 block's lane brings one key's scales by cp.async:
  // loads into registers were waited for at the end of the step.
  int held0 = 0, held1 = 0, brought = 0;
  auto hold = [&](int block) {  // the pages of this warp's next 32 blocks, a block to a lane
    const int64_t key = (block + static_cast<int64_t>(lane) * step) * C::kKeys;
    held0 = key < vis_max ? __ldg(table + (key >> a.page_log2)) : 0;
    held1 = C::kSub == 2 && key + 16 < vis_max ? __ldg(table + ((key + 16) >> a.page_log2)) : 0;
  };
  auto checked = [&](int page) -> int {  // page 0 in a bad one's place; the rows become NaN
    if (page >= 0 && page < a.n_pages) return page;
    bad_page = true;
    return 0;
  };
  const int pitch = kLinear ? a.d * (kE4m3 ? 1 : 2) : C::kRowBytes;  // of keys in a tile
  auto bring = [&](int block, int stage) {
    if (brought % 32 == 0) hold(block);
    int page0 = __shfl_sync(0xFFFFFFFFu, held0, brought % 32);
    int page1 = C::kSub == 2 ? __shfl_sync(0xFFFFFFFFu, held1, brought % 32) : 0;
    ++brought;
    const int key = block * C::kKeys;
    const uint32_t bar = bar0 + 8 * stage, dst = ring + stage * C::kStageBytes;
    const bool two = C::kSub == 2 && key + 16 < vis_max;  // the block's second tile exists
    page0 = checked(page0);
    if (two) page1 = checked(page1);
    if (lane == 0) {
      mbar_arrive_expect_tx(bar, (C::kSub == 2 && (two || wide) ? 2u : 1u) * 2 *
                                     (kLinear ? 16 * pitch : C::kHalves * C::kBoxBytes));
      const int y = key & page_mask;
      if constexpr (kLinear) {
        const uint32_t tile = 16 * pitch, bytes = C::kSub == 2 && wide ? 2 * tile : tile;
        auto rows_of = [&](const void* cache, int page, int at) {
          return static_cast<const uint8_t*>(cache) +
                 (page * a.ld_page + ((static_cast<int64_t>(hk) << a.page_log2) + at) * a.d) * (kE4m3 ? 1 : 2);
        };
        bulk_load(dst, rows_of(a.k, page0, y), bytes, bar);
        bulk_load(dst + C::kBoxes * C::kBoxBytes, rows_of(a.v, page0, y), bytes, bar);
        if (two && !wide) {
          const int y1 = (key + 16) & page_mask;
          bulk_load(dst + tile, rows_of(a.k, page1, y1), tile, bar);
          bulk_load(dst + C::kBoxes * C::kBoxBytes + tile, rows_of(a.v, page1, y1), tile, bar);
        }
      } else if (C::kSub == 2) {
        tma_load_page(dst, &map_k, bar, 0, y, 0, hk, page0);
        tma_load_page(dst + 2 * C::kBoxBytes, &map_v, bar, 0, y, 0, hk, page0);
        if (two && !wide) {
          const int y1 = (key + 16) & page_mask;
          tma_load_page(dst + C::kBoxBytes, &map_k, bar, 0, y1, 0, hk, page1);
          tma_load_page(dst + 3 * C::kBoxBytes, &map_v, bar, 0, y1, 0, hk, page1);
        }
      } else {
        tma_load_page(dst, &map_k, bar, 0, y, 0, hk, page0);
        tma_load_page(dst + C::kHalves * C::kBoxBytes, &map_v, bar, 0, y, 0, hk, page0);
        if (C::kHalves == 2 && !wide) {
          tma_load_page(dst + C::kBoxBytes, &map_k, bar, 64, y, 0, hk, page0);
          tma_load_page(dst + 3 * C::kBoxBytes, &map_v, bar, 64, y, 0, hk, page0);
        }
      }
    }
    if constexpr (kE4m3) {
      if (key + lane < vis_max) {
        const int64_t at = (lane < 16 ? page0 : page1) * a.ld_scale_page +
                           (static_cast<int64_t>(hk) << a.page_log2) + ((key + lane) & page_mask);
        copy_async4(smem_u32(&scales[warp][stage][0][lane]), a.k_scale + at);
        copy_async4(smem_u32(&scales[warp][stage][1][lane]), a.v_scale + at);
      }
      arrive_when_copied(bar);
    }
  };
  int block = split * kWarps + warp;
#pragma unroll
  for (int i = 0; i < C::kStages; ++i)
    if (block + i * step < n_blocks) bring(block + i * step, i);

  // ------------------------------------------------ Q's scale, visible counts
  // columns of this lane: rows 8 nt + 2 t and + 1
  float factor[NT][2];  // of the columns' scores, to log2 units
  int vis[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float f = a.scale_log2;
    if constexpr (kE4m3) {
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < C::kSteps; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          top = max(top, max((qf[nt][k][i] << 16) & 0x7FFF0000u, qf[nt][k][i] & 0x7FFF0000u));
      top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
      top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
      float up;
      f = f16_row_scale(top, a.scale_log2, &up);
#pragma unroll
      for (int k = 0; k < C::kSteps; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          qf[nt][k][i] = pack_f16(__uint_as_float(qf[nt][k][i] << 16) * up,
                                  __uint_as_float(qf[nt][k][i] & 0xFFFF0000u) * up);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      factor[nt][j] = kE4m3 ? __shfl_sync(0xFFFFFFFFu, f, 4 * (2 * t + j)) : f;
      const int rc = 8 * nt + 2 * t + j;
      vis[nt][j] = rc < rows ? row_sees(row_token(rc, a.group)) : 0;
    }
  }

  float o[NT][C::kSteps][4] = {};
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) { m[nt][0] = m[nt][1] = -INFINITY; l[nt][0] = l[nt][1] = 0.f; }
  // e4m3: a column's o is in units of 2^(m + v_exp) / kPScale.  One v_exp, found in the first
  // block, serves all columns while the values' scales stay between v_low and v_high (the
  // loop's first form).  From the first block on where they do not, each column has its own, and
  // v_room says how far m has risen since a weight set it: so much lower it still holds every
  // weight so far (the second form: 12 rows over 1024 keys of 24 sequences, 16 heads of 80, 57
  // us instead of 45; 64 sequences of 2048, 16 heads of 128, 101 instead of 97).
  int v_exp[NT][2], v_all = 0;
  float v_room[NT][2];
  float v_mul = 0.f, v_low = 0.f, v_high = 0.f;

  // this lane's keys of a tile: rows g (and g + 8) of K, rows 2 t, 2 t + 1 (and + 8) of V
  constexpr bool kSwizzled = C::kRowBytes == 128 && !kLinear;
  auto key_of = [](int r) { return kSwizzled ? row_key(r) : kLinear && !kE4m3 ? linear_key(r) : r; };
  const int key_g = key_of(g);
  const int key_t[2] = {key_of(2 * t), key_of(2 * t + 1)};
  const int tile_bytes = 16 * pitch;
  auto chunk_at = [&](int key, int chunk) -> uint32_t {  // of a box
    return key * pitch + ((kSwizzled ? chunk ^ (key & 7) : chunk) << 4);
  };

  int stage = 0, parity = 0;
  // Whether the rest is for the second form.
  auto go = [&](auto apart_) -> bool {
    constexpr bool kApart = decltype(apart_)::value;
    for (; block < n_blocks; block += step) {
      const int key0 = block * C::kKeys;
      if (!__all_sync(0xFFFFFFFFu, mbar_wait(bar0 + 8 * stage, parity, a.status, nullptr))) {
        // given up, by the whole warp: NaN, once the copies in flight have had as long again
        bad_page = true;
        for (int i = 0; i < C::kStages; ++i) {
          if (block + i * step < n_blocks) mbar_wait(bar0 + 8 * stage, parity, a.status, nullptr);
          if (++stage == C::kStages) { stage = 0; parity ^= 1; }
        }
        return false;
      }
      const uint32_t kb = ring + stage * C::kStageBytes, vb = kb + C::kBoxes * C::kBoxBytes;
      // two sums per score: half the chain of dependent products
      float s[C::kSub][NT][4] = {}, s2[C::kSub][NT][4] = {};
#pragma unroll
      for (int u = 0; u < C::kSub; ++u) {
        if constexpr (kE4m3) {
#pragma unroll
          for (int c = 0; c < kChunksK; ++c) {
            uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
            if (!kLinear || 16 * (4 * c + t) < a.d) {  // behind a linear row comes the next
              lo = lds16(kb + u * tile_bytes + chunk_at(key_g, 4 * c + t));
              hi = lds16(kb + u * tile_bytes + chunk_at(key_g + 8, 4 * c + t));
            }
            const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t f[4] = {e4m3x2_f16x2(wl[i], 0), e4m3x2_f16x2(wh[i], 0),
                                     e4m3x2_f16x2(wl[i], 1), e4m3x2_f16x2(wh[i], 1)};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma16816<true>(i & 1 ? s2[u][nt] : s[u][nt], f, qf[nt][4 * c + i][0],
                               qf[nt][4 * c + i][1]);
            }
          }
        } else {
#pragma unroll
          for (int c = 0; c < kChunksK; ++c) {
            const uint32_t box = kLinear ? kb : kb + (c >> 1) * C::kBoxBytes;
            const int chunk = kLinear ? 4 * c + t : 4 * (c & 1) + t;
            uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
            if (!kLinear || 8 * chunk < a.d) {
              lo = lds16(box + chunk_at(key_g, chunk));
              hi = lds16(box + chunk_at(key_g + 8, chunk));
            }
            const uint32_t f0[4] = {lo.x, hi.x, lo.y, hi.y}, f1[4] = {lo.z, hi.z, lo.w, hi.w};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma16816<false>(s[u][nt], f0, qf[nt][2 * c][0], qf[nt][2 * c][1]);
              mma16816<false>(s2[u][nt], f1, qf[nt][2 * c + 1][0], qf[nt][2 * c + 1][1]);
            }
          }
        }
      }
      const bool edge = key0 + C::kKeys > vis_min;
      float sk[C::kSub][2], sv[C::kSub][2];
      if constexpr (kE4m3) {
        float top = 0.f, low = INFINITY;  // of the values' scales that are numbers, and not 0
#pragma unroll
        for (int u = 0; u < C::kSub; ++u)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            sk[u][i] = scales[warp][stage][0][16 * u + 8 * i + key_g];
            sv[u][i] = scales[warp][stage][1][16 * u + 8 * i + key_g];
            if (edge && key0 + 16 * u + 8 * i + key_g >= vis_max) sv[u][i] = 0.f;
            const float x = fabsf(sv[u][i]);
            top = fmaxf(top, x);
            low = fminf(low, x == 0.f ? INFINITY : x);
          }
        if (!kApart && __any_sync(0xFFFFFFFFu, top > v_high || low < v_low)) {
          if (v_mul == 0.f) {  // the first block
            float most = top < INFINITY ? top : 0.f;
            most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 4));
            most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 8));
            most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 16));
            v_all = max(exponent_above(most) + 11, kLeastExp);
            v_mul = exp_scale(v_all);
            v_low = kLowWeight / v_mul;
            v_high = kMostWeight / v_mul;
          }
          // (every row's key of its m has had a weight of kLowWeight or more so far: no room)
          if (__any_sync(0xFFFFFFFFu, top > v_high || low < v_low)) return true;
        }
      }

      // scores in units of log2, masked; the columns' maxima over the block
      bool moved = false;
      float shrink[NT][2], rise[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float top = m[nt][j];
#pragma unroll
          for (int u = 0; u < C::kSub; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float x = (s[u][nt][2 * i + j] + s2[u][nt][2 * i + j]) *
                        (kE4m3 ? sk[u][i] * factor[nt][j] : factor[nt][j]);
              if (edge && !sees(key0 + 16 * u + 8 * i + key_g, vis[nt][j])) x = -INFINITY;
              s[u][nt][2 * i + j] = x;
              top = fmaxf(top, x);
            }
          top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
          const float was = m[nt][j];
          shrink[nt][j] = 1.f;
          rise[nt][j] = 0.f;
          if (top > was) {
            shrink[nt][j] = was == -INFINITY ? 0.f : fast_exp2(was - top);
            m[nt][j] = top;
            moved = true;
            rise[nt][j] = top - was;
          }
          const float ref = m[nt][j] == -INFINITY ? 0.f : m[nt][j];
          float sum = 0.f;
#pragma unroll
          for (int u = 0; u < C::kSub; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float p = fast_exp2(s[u][nt][2 * i + j] - ref);
              sum += p;
              if constexpr (kE4m3) {
                if (!kApart) p *= sv[u][i] * v_mul;
                // a masked key's scale may be anything: its weight is 0, not 0 times that
                if (edge && !sees(key0 + 16 * u + 8 * i + key_g, vis[nt][j])) p = 0.f;
              }
              s[u][nt][2 * i + j] = p;
            }
          l[nt][j] = l[nt][j] * shrink[nt][j] + sum;
        }
      if constexpr (kApart) {
#pragma unroll
        for (int u = 0; u < C::kSub; ++u)
#pragma unroll
          for (int i = 0; i < 2; ++i) sv[u][i] = fmaf(sv[u][i], 0.f, sv[u][i]);  // an infinity becomes NaN
        auto weight = [&](int u, int nt, int i, int j) -> float {
          const float x = s[u][nt][2 * i + j] * exp_scale(v_exp[nt][j]) * sv[u][i];
          return edge && !sees(key0 + 16 * u + 8 * i + key_g, vis[nt][j]) ? 0.f : x;
        };
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            v_room[nt][j] = rise[nt][j] == INFINITY ? kAllRoom : v_room[nt][j] + rise[nt][j];
            for (int tries = 0; tries < 4; ++tries) {  // of an infinite weight only that it is too large is known
              float top = 0.f;
#pragma unroll
              for (int u = 0; u < C::kSub; ++u)
                top = fmaxf(top, fmaxf(fabsf(weight(u, nt, 0, j)), fabsf(weight(u, nt, 1, j))));
              top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 4));
              top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 8));
              top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16));
              int up = 0;
              if (top > kMostWeight) {
                up = exponent_above(top);
                v_room[nt][j] = 0.f;
              } else if (top < kLowWeight && top > 0.f) {
                up = -min(min(static_cast<int>(v_room[nt][j]), v_exp[nt][j] - kLeastExp), -exponent_above(top));
                v_room[nt][j] += static_cast<float>(up);
              }
              v_exp[nt][j] += up;
              const float f0 = pow2(-(up / 2)), f1 = pow2(-(up - up / 2));
#pragma unroll
              for (int k = 0; k < C::kSteps; ++k) {
                o[nt][k][j] = o[nt][k][j] * f0 * f1;
                o[nt][k][2 + j] = o[nt][k][2 + j] * f0 * f1;
              }
              if (!__any_sync(0xFFFFFFFFu, top == INFINITY)) break;
            }
            if (v_room[nt][j] > 0.5f * kAllRoom) v_room[nt][j] = 0.f;
#pragma unroll
            for (int u = 0; u < C::kSub; ++u)
#pragma unroll
              for (int i = 0; i < 2; ++i) s[u][nt][2 * i + j] = weight(u, nt, i, j);
          }
      }
      uint32_t pb[C::kSub][NT][2], pl[C::kSub][NT][2];
#pragma unroll
      for (int u = 0; u < C::kSub; ++u)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float p0 = s[u][nt][2 * i], p1 = s[u][nt][2 * i + 1];
            if constexpr (kE4m3) {
              pb[u][nt][i] = transpose8x8(pack_f16(p0, p1));
            } else {
              const uint32_t big = pack_bf16(p0, p1);
              pb[u][nt][i] = transpose8x8(big);
              pl[u][nt][i] = transpose8x8(pack_bf16(p0 - __uint_as_float(big << 16),
                                                    p1 - __uint_as_float(big & 0xFFFF0000u)));
            }
          }
      if (__any_sync(0xFFFFFFFFu, moved)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float f0 = shrink[nt][0], f1 = shrink[nt][1];
#pragma unroll
          for (int k = 0; k < C::kSteps; ++k) {
            o[nt][k][0] *= f0; o[nt][k][1] *= f1;
            o[nt][k][2] *= f0; o[nt][k][3] *= f1;
          }
        }
      }
      // 16 bytes (8 for e4m3 at 64 channels) of four keys' values at a time
      constexpr int kPieces = kE4m3 ? 1 : DP / 64;
      constexpr int kWords = kE4m3 && DP == 64 ? 2 : 4;
#pragma unroll
      for (int u = 0; u < C::kSub; ++u)
#pragma unroll
        for (int c = 0; c < kPieces; ++c) {
          uint32_t w[4][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = key_t[i & 1] + 8 * (i >> 1);
            if constexpr (kWords == 2) {
              const uint2 x = lds8(vb + u * tile_bytes + key * pitch + 8 * g);
              w[i][0] = x.x; w[i][1] = x.y;
            } else {
              const uint4 x = lds16(vb + (kE4m3 ? u * tile_bytes : kLinear ? c * 128 : c * C::kBoxBytes) +
                                    chunk_at(key, g));
              w[i][0] = x.x; w[i][1] = x.y; w[i][2] = x.z; w[i][3] = x.w;
            }
            if (edge) {  // keys that some row may not see: their values must not reach it as 0 * NaN
              const int at = key0 + 16 * u + key;
#pragma unroll
              for (int k = 0; k < kWords; ++k) {
                const int ch = 8 * (8 * c + g) + 2 * k;
                if (at >= vis_max) w[i][k] = 0;
                else if (!kE4m3 && at >= vis_min)
                  w[i][k] = only_finite<kTree>(w[i][k], kTree ? at - prefix : at, &first_bad[ch], &first_bad[ch + 1]);
              }
            }
          }
#pragma unroll
          for (int k = 0; k < kWords; ++k) {
            if constexpr (kE4m3) {
              // both keys' codes of a channel side by side, then four codes to fp16
              const uint32_t a01 = __byte_perm(w[0][k], w[1][k], 0x5140);
              const uint32_t b01 = __byte_perm(w[2][k], w[3][k], 0x5140);
              const uint32_t a23 = __byte_perm(w[0][k], w[1][k], 0x7362);
              const uint32_t b23 = __byte_perm(w[2][k], w[3][k], 0x7362);
              const uint32_t f0[4] = {e4m3x2_f16x2(a01, 0), e4m3x2_f16x2(a01, 1),
                                      e4m3x2_f16x2(b01, 0), e4m3x2_f16x2(b01, 1)};
              const uint32_t f1[4] = {e4m3x2_f16x2(a23, 0), e4m3x2_f16x2(a23, 1),
                                      e4m3x2_f16x2(b23, 0), e4m3x2_f16x2(b23, 1)};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma16816<true>(o[nt][2 * k], f0, pb[u][nt][0], pb[u][nt][1]);
                mma16816<true>(o[nt][2 * k + 1], f1, pb[u][nt][0], pb[u][nt][1]);
              }
            } else {
              const uint32_t f[4] = {
                  __byte_perm(w[0][k], w[1][k], 0x5410), __byte_perm(w[0][k], w[1][k], 0x7632),
                  __byte_perm(w[2][k], w[3][k], 0x5410), __byte_perm(w[2][k], w[3][k], 0x7632)};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma16816<false>(o[nt][4 * c + k], f, pb[u][nt][0], pb[u][nt][1]);
                mma16816<false>(o[nt][4 * c + k], f, pl[u][nt][0], pl[u][nt][1]);
              }
            }
          }
        }
      __syncwarp();  // every lane has read the stage
      const int ahead = block + C::kStages * step;
      if (ahead < n_blocks) bring(ahead, stage);
      if (++stage == C::kStages) { stage = 0; parity ^= 1; }
    }
    return false;
  };
  const bool more = go(std::false_type{});
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    v_exp[nt][0] = v_exp[nt][1] = v_all;
    v_room[nt][0] = v_room[nt][1] = 0.f;
  }
  if (kE4m3 && more) go(std::bool_constant<kE4m3>{});
  if (__any_sync(0xFFFFFFFFu, bad_page)) {
    if (lane == 0) paged_report(a.status);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) l[nt][0] = l[nt][1] = __uint_as_float(0x7FC00000u);
  }
  __syncthreads();  // the rings' place is the partials' now

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
      const float v_back = kE4m3 ? 1.f / exp_scale(v_exp[nt][j]) : 1.f;
      if (g == 0) {
        part_m[warp][r] = m[nt][j];
        part_l[warp][r] = x;
      }
      if (r < rows) {
#pragma unroll
        for (int k = 0; k < C::kSteps; ++k) {
          // channels 2 k' and 2 k' + 1 of this lane's chunk
          const int ch = kE4m3 ? (DP / 8) * g + 2 * k : 8 * (8 * (k >> 2) + g) + 2 * (k & 3);
          *reinterpret_cast<float2*>(&part_o[(warp * C::kRows + r) * DP + ch]) =
              make_float2(o[nt][k][j] * v_back, o[nt][k][2 + j] * v_back);
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
      const float2 p = *reinterpret_cast<const float2*>(&part_o[(w * C::kRows + r) * DP + ch]);
      x += f * p.x;
      y += f * p.y;
    }
    if (ch == 0) {
      block_m[r] = top;
      block_l[r] = sum;
    }
    // only this thread reads or writes these entries
    *reinterpret_cast<float2*>(&part_o[r * DP + ch]) = make_float2(x, y);
  }
  if (cluster > 1) cluster_sync();
  else __syncthreads();
  for (int i = split * kThreads + threadIdx.x; i < rows * (DP / 2); i += cluster * kThreads) {
    const int r = i / (DP / 2), ch = 2 * (i % (DP / 2));
    if (ch >= a.d) continue;
    float ms[kMaxCluster], ls[kMaxCluster];
    float2 os[kMaxCluster];
    int bad0 = kNoBad, bad1 = kNoBad;
    float top = -INFINITY;
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) {
      ms[c] = -INFINITY;
      if (c < cluster) {
        ms[c] = ld_cluster_f32(&block_m[r], c);
        ls[c] = ld_cluster_f32(&block_l[r], c);
        os[c] = ld_cluster_f32x2(&part_o[r * DP + ch], c);
        if (!kE4m3) {
          const int x = ld_cluster_s32(&first_bad[ch], c), y = ld_cluster_s32(&first_bad[ch + 1], c);
          bad0 = kTree ? bad0 | x : min(bad0, x);
          bad1 = kTree ? bad1 | y : min(bad1, y);
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
    const uint32_t row = r, token = row_token(row, a.group);
    const int seen = row_sees(token);
    x = (kTree ? (bad0 & seen) != 0 : bad0 < seen) ? __uint_as_float(0x7FC00000u) : x * inv;
    y = (kTree ? (bad1 & seen) != 0 : bad1 < seen) ? __uint_as_float(0x7FC00000u) : y * inv;
    *reinterpret_cast<uint32_t*>(a.out + (seq.row0 + token) * a.out_ld +
                                 (static_cast<int64_t>(hk) * a.group + row - token * a.group) * a.d + ch) =
        pack_bf16(x, y);
  }
  if (cluster > 1) cluster_sync();  // no block leaves while another reads its partial
}

template <bool kE4m3, int DP, int NT, int W, bool kLinear, bool kTree>
cudaError_t launch_rows(const PagedArgs& a, int64_t units, int cluster, cudaStream_t stream) {
  using C = RowsCfg<kE4m3, DP, NT, W>;
  CUtensorMap mk{}, mv{};
  // one box where a page holds a whole e4m3 block, or both halves of full bf16 rows
  const bool wide = kE4m3 ? a.page_log2 >= 5 : a.d == 128;
  const int box_rows = kE4m3 && wide ? 32 : 16, box_halves = !kE4m3 && wide ? 2 : 1;
  if (!kLinear && (!make_page_map(&mk, a.k, a, C::kRowBytes, box_rows, box_halves) ||
                   !make_page_map(&mv, a.v, a, C::kRowBytes, box_rows, box_halves)))
    return cudaErrorInvalidValue;
  if (units * cluster > 0x7FFFFFFFll) return cudaErrorInvalidConfiguration;
  constexpr auto kKernel = paged_rows_kernel<kE4m3, DP, NT, W, kLinear, kTree>;
  if (cudaError_t e = allow_smem_once<kKernel>(C::kSmem); e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(units * cluster));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(cluster);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kKernel, mk, mv, a, cluster, wide ? 1 : 0,
                            units * cluster > device_sm_count() ? 1 : 0);
}

// How a call is cut up: the longest context is split over 2^n blocks of 4 warps
// until there are 3 blocks for every SM (as many reside) or a warp is left with fewer
// than 8 steps, whose pipeline then hardly fills; below 2 blocks per SM it is split
// down to 2 steps all the same.  (32 sequences up to 16384 tokens, 8 heads, e4m3: one
// block each 212 us, 2 126, 4 132, 8 156; 64 up to 2048, 16 heads, bf16: 83, 97, 128.)
// What still leaves half the SMs without a block gets 8 warps per block (one sequence of
// 30000, 8 heads, 8 blocks each: 78 us with 4 warps, 46 with 8), not more: a block of 8
// fills an SM, and clusters of them do not fit side by side.  Two blocks of 4 warps become one
// of 8 where every SM has at most one then: no cluster to join, no order to find (16 sequences
// up to 256, 6 heads of 64: 5.8 us, 4.9 so; 32 of 512, 4 heads of 128, e4m3: 9.1, 7.9).
// (Step: 32 keys of an e4m3 cache, 16 of a bf16 one.)
//
// Where d is an odd number of 16 channels (16, 48, 80, 112) rows can be read out of
// shared memory without a swizzle as well as with it, so a block of them comes as it lies
// in the page, in one bulk copy; a tiled copy goes row by row, two requests to a row that
// crosses 128 bytes (64 sequences up to 2048, 16 heads of 80: e4m3 60 us, 46 so; bf16 63.7
// and 62.2.  24 up to 1024 with drafts, e4m3: 18.7 and 15.8).
template <bool kE4m3, int DP, int NT, bool kLinear, bool kTree>
cudaError_t launch_rows_cut(const PagedArgs& a, int64_t units, cudaStream_t stream) {
  const int64_t sms = device_sm_count();
  const int64_t steps = (static_cast<int64_t>(a.max_pages) << a.page_log2) / (kE4m3 ? 32 : 16);
  int cluster = 1;
  while (cluster < kMaxCluster) {
    const int64_t blocks = units * cluster, per_warp = steps / (4 * 2 * cluster);
    if (!(blocks < 2 * sms ? per_warp >= 2 : blocks < 3 * sms && per_warp >= 8)) break;
    cluster *= 2;
  }
  if (cluster == 2 && units <= sms && 2 * units > sms / 2)
    return launch_rows<kE4m3, DP, NT, 8, kLinear, kTree>(a, units, 1, stream);
  return units * cluster <= sms / 2 && steps >= 8 * cluster
             ? launch_rows<kE4m3, DP, NT, 8, kLinear, kTree>(a, units, cluster, stream)
             : launch_rows<kE4m3, DP, NT, 4, kLinear, kTree>(a, units, cluster, stream);
}

template <bool kE4m3, int DP, bool kTree>
cudaError_t launch_rows_nt(const PagedArgs& a, cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(a.max_q) * a.group;
  const int64_t heads = static_cast<int64_t>(a.B) * a.H_kv;
  if (a.d % 32 != 0)
    return rows <= 8 ? launch_rows_cut<kE4m3, DP, 1, true, kTree>(a, heads, stream)
                     : launch_rows_cut<kE4m3, DP, 2, true, kTree>(a, heads, stream);
  return rows <= 8 ? launch_rows_cut<kE4m3, DP, 1, false, kTree>(a, heads, stream)
                   : launch_rows_cut<kE4m3, DP, 2, false, kTree>(a, heads, stream);
}

template <bool kTree>
cudaError_t launch_few_rows(const PagedArgs& a, cudaStream_t stream) {
  const bool e4m3 = a.k_scale != nullptr;
  if (a.d <= 64) return e4m3 ? launch_rows_nt<true, 64, kTree>(a, stream) : launch_rows_nt<false, 64, kTree>(a, stream);
  return e4m3 ? launch_rows_nt<true, 128, kTree>(a, stream) : launch_rows_nt<false, 128, kTree>(a, stream);
}

}  // namespace

cudaError_t launch_paged_attention(const PagedArgs& a, cudaStream_t stream) {
  if (static_cast<int64_t>(a.max_q) * a.group > kFewRows) return launch_paged_attention_mma(a, stream);
  return launch_few_rows<false>(a, stream);
}

cudaError_t launch_paged_tree_attention(const PagedArgs& a, void* workspace, cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(a.max_q) * a.group;
  return rows <= kFewRows   ? launch_few_rows<true>(a, stream)
         : tree_is_short(a) ? launch_tree_attention_short(a, stream)
         : tree_has_room(a) ? launch_tree_attention(a, workspace, stream)
                            : launch_paged_attention_mma(a, stream);
}

}  // namespace dwa
