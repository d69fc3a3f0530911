// tree_attention_short.cu — attention of a tree's nodes over the paged cache on tcgen05 where contexts are
// short for as many sequences as there are: what tree_attention.cu computes, by blocks that have a
// unit each.
//
// A row is one (node, query head of the group), node-major.  A unit is up to 32 rows of one key/value
// head; it goes over the sequence's keys 128 at a time, its products transposed:
//
//   S^T = K Q^T       128 keys by 32 rows      tcgen05, K and Q in shared memory, S in TMEM
//   P   = exp2(S - a) a thread per key and 16 rows
//   O^T += V^T P      128 channels by 32 rows  tcgen05, V and P in shared memory, O in TMEM
//
// What a row's weights are relative to, a, moves only when a score passes the limit (2^20 for bf16, for e4m3
// what keeps a weight times its value's scale below 2^15), which every step asks by a vote.  Scores of 2^20 and more, and
// values' scales 2^90 apart, take the careful steps of tree_tiles.cuh.
//
// Rounding: bf16 caches none beside f32 sums (P is the sum of two bf16 parts).  e4m3: codes are
// exact; Q is, per row, a power of two times the sum of two e4m3 numbers, exactly down to 2^-9 of the
// row's largest value and to 2^-18 of that below; P times the value's scale is rounded to fp16, 11 bits.
//
// Bound by latency: a block's set-up, its first loads and its way out take as long as four to six steps, and a
// step is a chain of product, vote, exponentials, product.  So two blocks share an SM, each with half of
// its shared memory and registers, and none has more to find out than its own sequence: no shares, no
// parts to join.  16 sequences of 32 nodes, 16 heads of 128 channels, over 128 and 1024 tokens: bf16 11 and
// 31 us, e4m3 12 and 25; a block to an SM that shares out the steps 17 and 40, 18 and 38.  24 ragged ones of 5 to 40
// nodes over 50 to 1500 tokens, 16 heads of 80, e4m3: 45 us, 66 in tiles of 128 rows.  Long contexts
// turn this round: the longest unit has a block to itself (see tree_is_short).
//
// Eight warps: softmax, sixteen columns to each four; e4m3: they turn the values' codes into fp16 too.  One warp:
// tcgen05.mma.  Two: TMA, straight from the pages, keys by one, values by the other.  One sets the barriers up.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "dwa_internal.h"
#include "f32x2.cuh"
#include "paged_attention.cuh"
#include "sm100_ptx.cuh"
#include "tree_tiles.cuh"

namespace dwa {

namespace {

constexpr int kSmemLimit = 113 * 1024;  // two blocks to an SM

// kE4m3: 8-bit cache.  DP: d rounded up to 64 or 128.  N: rows of a unit.
template <bool kE4m3, int DP, int N>
struct ShortCfg {
  static constexpr int kThreads = 384, kSoftmax = 256, kSharers = 2;  // warpgroups, each a sixteen of columns
  static_assert(N == 16 * kSharers);
  static constexpr int kHalves = DP / 64;
  static constexpr int kQPart = N * 128;                       // 64 bf16 channels, or 128 codes
  static constexpr int kQBytes = (kE4m3 ? 2 : kHalves) * kQPart;
  static constexpr int kPCols = (kE4m3 ? 1 : 2) * N;           // bf16: both parts of P side by side, in one product
  static constexpr int kPBytes = kBlock;
  static constexpr int kKBytes = (kE4m3 ? 1 : kHalves) * kBlock;
  // Values arrive as they go into their product, or as codes, which become one tile of fp16.
  static constexpr int kVBytes = kE4m3 ? kTile * DP : kHalves * kBlock;
  static constexpr int kWideBytes = kE4m3 ? kHalves * kBlock : 0;
  // Scores run two tiles ahead of weights, so that tiles of keys go early.
  static constexpr int kKStages = DP == 128 ? 1 : 2, kVStages = DP == 64 ? 3 : kE4m3 ? 2 : 1;
  // e4m3: scales of the keys and values of a tile come with its keys, and stay until its weights are made.
  static constexpr int kScaleBytes = kE4m3 ? 2 * kTile * 4 : 0, kScaleSlots = DP == 128 ? 4 : 8;
  static_assert(kKStages + 2 < kScaleSlots);
  static constexpr int kKAt = kQBytes, kVAt = kKAt + kKStages * kKBytes, kWideAt = kVAt + kVStages * kVBytes;
  // (A tile of 64 channels is read as if there were 128: what is behind it makes rows that nobody reads.)
  static constexpr int kPAt = kWideAt + kWideBytes, kScalesAt = kPAt + kPBytes;
  static constexpr int kSmem = 1024 + kScalesAt + kScaleSlots * kScaleBytes;
  static constexpr int kStatic = 2048;  // at most
  static_assert(kSmem + kStatic <= kSmemLimit);
  static constexpr int kTmemCols = 128;
  static_assert(2 * N + kPCols <= kTmemCols, "two S, one O");
};

// ---------------------------------------------------------------- work
// A block's unit: 32 rows at most of one key/value head of a sequence.
struct Unit {
  int hk, rb;        // key/value head, block of rows
  int steps;         // tiles of 128 keys
  PagedSeq seq;
  int64_t table;     // where its pages are
};

// Tiles of a sequence.  (One for rows that see no key, or get NaN.)
__device__ __forceinline__ int tree_steps(const PagedSeq& s) {
  return s.n == 0 ? 0 : s.bad ? 1 : max((s.length + kTile - 1) / kTile, 1);
}
// The longest sequences start first; a head's blocks of rows side by side, as they read the same pages.
__device__ __forceinline__ Unit find_unit(const PagedArgs& a, uint32_t block, uint32_t row_units, int* scratch) {
  const uint32_t head = block / row_units;
  int b = static_cast<int>(head / a.H_kv);
  Unit u;
  u.rb = static_cast<int>(block - head * row_units);
  u.hk = static_cast<int>(head - static_cast<uint32_t>(b) * a.H_kv);
  if (a.B > 1 && a.B <= kMostRanked)
    b = ranked(a.B, b, scratch, scratch + kMostRanked, [&](int i) { return tree_steps(paged_seq(a, i)); });
  u.seq = paged_seq(a, b);
  u.steps = tree_steps(u.seq);
  u.table = static_cast<int64_t>(b) * a.ld_table;
  return u;
}

// ---------------------------------------------------------------- the kernel
template <bool kE4m3, int N>
struct ShortShared {
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
  uint64_t scales_full[kE4m3 ? 8 : 1];
  uint64_t q_ready, s_ready[2], s_free[2], p_ready, p_free;
  uint32_t tmem;
  int abort;
  int bad_page, any_bad;
  alignas(16) float neg_a[N];   // minus what a column's weights are relative to
  alignas(16) float f[kE4m3 ? N : 4];     // its scores' factor, to log2 units
  int most[N];                  // across keys, ordered
  int row[N];                   // of q
  uint32_t tops[2][4];          // e4m3: scales' exponents
  float d[kE4m3 ? N : 4];       // e4m3: O's units are 2^d beside the references'
  float shrink_l[N], shrink_o[N];
  int careful[2];               // of each warpgroup
};

template <bool kE4m3, int DP, int N>
__global__ void __launch_bounds__(ShortCfg<kE4m3, DP, N>::kThreads, 2)
    short_tree_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                          const __grid_constant__ PagedArgs a, const uint32_t row_units) {
  using C = ShortCfg<kE4m3, DP, N>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ ShortShared<kE4m3, N> sh;
  static_assert(sizeof(ShortShared<kE4m3, N>) <= C::kStatic, "as much as is left for it");
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kMma = C::kSoftmax / 32, kTma = kMma + 1;  // warps; two for TMA

  // ------------------------------------------------ set-up
  auto bar = [&](const uint64_t& x) { return smem_u32(&x); };
  if (warp == kTma + 2 && lane == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(bar(sh.k_full[i]), 1);
      mbar_init(bar(sh.k_empty[i]), 1);
      mbar_init(bar(sh.v_full[i]), 1);
      mbar_init(bar(sh.v_empty[i]), kE4m3 ? C::kSoftmax / 32 : 1);
    }
    sh.bad_page = sh.any_bad = 0;
    for (int i = 0; i < (kE4m3 ? 8 : 1); ++i) mbar_init(bar(sh.scales_full[i]), 1);
    mbar_init(bar(sh.q_ready), C::kSoftmax / 32);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(sh.s_ready[i]), 1);
      mbar_init(bar(sh.s_free[i]), C::kSoftmax / 32);
    }
    mbar_init(bar(sh.p_ready), C::kSoftmax / 32);
    mbar_init(bar(sh.p_free), 1);
    sh.abort = 0;
    fence_mbar_init();
  }
  // ------------------------------------------------ the block's work
  const Unit p = find_unit(a, blockIdx.x, row_units, reinterpret_cast<int*>(smem));
  if (p.seq.bad && p.hk == 0 && p.rb == 0 && threadIdx.x == 0) paged_report(a.status);
  const int64_t all_rows = static_cast<int64_t>(p.seq.n) * a.group;
  if (static_cast<int64_t>(p.rb) * N >= all_rows) return;
  const int rows = static_cast<int>(min(all_rows - static_cast<int64_t>(p.rb) * N, static_cast<int64_t>(N)));
  const int cols = (rows + 15) & ~15;
  const int n = p.seq.length == 0 ? 0 : p.steps;  // 0: nothing to read
  if (p.seq.bad) {  // all its rows, which may be more than max_q says
    const int64_t stride = static_cast<int64_t>(row_units) * N;
    for (int64_t r = static_cast<int64_t>(p.rb) * N; r < all_rows; r += stride)
      for (int i = threadIdx.x; i < N * a.d; i += C::kThreads) {
        const int64_t row = r + i / a.d;
        if (row < all_rows)
          a.out[(p.seq.row0 + row / a.group) * a.out_ld +
                (static_cast<int64_t>(p.hk) * a.group + row % a.group) * a.d + i % a.d] = 0x7FC0u;
      }
    return;
  }

  if (warp == kMma) {
    tmem_alloc(smem_u32(&sh.tmem), C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm_s = sh.tmem, tm_o = sh.tmem + 2 * N;  // S: + N (it & 1)
  int* const status = a.status;
  volatile int* const abort_flag = &sh.abort;
  auto wait = [&](const uint64_t& x, int phase) -> bool {
    return warp_wait(bar(x), phase & 1, status, abort_flag);
  };
  auto wait2 = [&](const uint64_t& x, int phase_x, const uint64_t& y, int phase_y) -> bool {
    return warp_wait2(bar(x), phase_x & 1, bar(y), phase_y & 1, status, abort_flag);
  };
  auto warp_arrive = [&](const uint64_t& x) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(x));
  };
  const uint32_t s_k = base + C::kKAt, s_v = base + C::kVAt, s_p = base + C::kPAt;
  if (warp >= kMma) {
    if (warp > kMma && warp < kTma + 2) {
      // ---------------------------------------------- TMA: a warp for keys, one for values
      const bool values = warp == kTma + 1;
      const int stages = values ? C::kVStages : C::kKStages, stage_bytes = values ? C::kVBytes : C::kKBytes;
      const uint32_t tiles = values ? s_v : s_k;
      const uint32_t full0 = values ? bar(sh.v_full[0]) : bar(sh.k_full[0]);
      const uint32_t empty0 = values ? bar(sh.v_empty[0]) : bar(sh.k_empty[0]);
      const CUtensorMap* map = values ? &map_v : &map_k;
      const int row_bytes = values && kE4m3 ? DP : 128;
      const int page_size = 1 << a.page_log2, of_tile = kTile >> a.page_log2;  // pages of a tile: 1 to 8
      int stage = 0, use = 0, slot = 0;
      bool ok = true;
      const int32_t* table = a.table + p.table;
      const int hk = p.hk;
      const int pages = (p.seq.length + page_size - 1) >> a.page_log2;
      int held = 0;  // the pages of the next 4 to 32 tiles, a page to a lane
      for (int j = 0; j < n; ++j) {
        const int at = (j * of_tile) & 31;
        if (at == 0) {
          const int i = j * of_tile + lane;
          held = i < pages ? __ldg(table + i) : 0;
          if (held < 0 || held >= a.n_pages) {
            if (i < n * of_tile) sh.bad_page = 1;  // read page 0 in its place; the rows become NaN
            held = 0;
          }
        }
        const int here = min(of_tile, pages - j * of_tile);
        const uint32_t full = full0 + 8 * stage;
        if (use > 0 && !(ok = warp_wait(empty0 + 8 * stage, (use - 1) & 1, status, abort_flag))) break;
        // Both tiles' scales come with the keys.  (Their slot has been read: see kScaleSlots.)
        const bool scales = kE4m3 && !values;
        const uint32_t slot_full = bar(sh.scales_full[kE4m3 ? slot : 0]);
        if (lane == 0) {
          mbar_arrive_expect_tx(full, static_cast<uint32_t>(here * page_size * row_bytes) * (kE4m3 ? 1 : C::kHalves));
          if (scales) mbar_arrive_expect_tx(slot_full, static_cast<uint32_t>(here * page_size) * 8);
        }
        __syncwarp();
        uint32_t dst = tiles + stage * stage_bytes;
        for (int q = 0; q < here; ++q, dst += page_size * row_bytes) {
          const int page = __shfl_sync(0xFFFFFFFFu, held, at + q);
          if (lane == 0) {
#pragma unroll
            for (int h = 0; h < (kE4m3 ? 1 : C::kHalves); ++h)
              tma_load_page(dst + h * kBlock, map, full, 64 * h, 0, 0, hk, page);
            if (scales) {
              const int64_t from = page * a.ld_scale_page + (static_cast<int64_t>(hk) << a.page_log2);
              const uint32_t to = base + C::kScalesAt + slot * C::kScaleBytes + q * page_size * 4;
              bulk_load(to, a.k_scale + from, page_size * 4, slot_full);
              bulk_load(to + kTile * 4, a.v_scale + from, page_size * 4, slot_full);
            }
          }
        }
        slot = (slot + 1) % C::kScaleSlots;
        if (++stage == stages) {
          stage = 0;
          ++use;
        }
      }
      // after an abort nobody else waits for the copies in flight
      if (*abort_flag) {
        for (int i = 0; i < stages && (use > 0 || stage > 0); ++i) {
          if (--stage < 0) {
            stage = stages - 1;
            --use;
          }
          mbar_wait(full0 + 8 * stage, use & 1, status, nullptr);
          if (kE4m3 && !values) {  // the same tile's scales
            slot = (slot + C::kScaleSlots - 1) % C::kScaleSlots;
            mbar_wait(bar(sh.scales_full[kE4m3 ? slot : 0]), ((use * stages + stage) / C::kScaleSlots) & 1, status, nullptr);
          }
        }
      }
    } else if (warp == kMma) {
      // ---------------------------------------------- tcgen05.mma
      constexpr uint32_t kM = kTile / 16 << 24;
      constexpr uint32_t kF16 = kE4m3 ? 0u : (1u << 7) | (1u << 10);  // fp16 or bf16
      const int k_steps = kE4m3 ? (a.d + 31) / 32 : a.d / 16;
      const uint32_t one = elect_one();
      // Only a descriptor's start address changes: its low word by constants, so that the one issuing
      // lane spends a few instructions per product.
      const uint32_t k_hi = static_cast<uint32_t>(sw128_kmajor_desc(0) >> 32), k_lo = static_cast<uint32_t>(sw128_kmajor_desc(0));
      const uint32_t v_hi = static_cast<uint32_t>(by_key_desc(0) >> 32), v_lo = static_cast<uint32_t>(by_key_desc(0));
      auto desc = [](uint32_t lo, uint32_t hi) -> uint64_t {
        uint64_t r;
        asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
        return r;
      };
      auto addr = [](uint32_t x) -> uint32_t { return (x >> 4) & 0x3FFFu; };
      const bool full_d = a.d == DP;
      bool ok = n > 0;
      const uint32_t idesc_s = (1u << 4) | kF16 | (static_cast<uint32_t>(cols) / 8 << 17) | kM;
      const uint32_t idesc_o = (1u << 4) | kF16 | (1u << 15) | (1u << 16) | (static_cast<uint32_t>(C::kPCols - N + cols) / 8 << 17) | kM;
      ok = ok && wait(sh.q_ready, 0);
      auto scores = [&](int i) -> bool {  // S = K_i Q^T
        const int ks = i % C::kKStages;
        const bool again = i >= 2;  // S has been used before
        if (!wait2(sh.k_full[ks], i / C::kKStages, again ? sh.s_free[i & 1] : sh.k_full[ks],
                   again ? (i >> 1) - 1 : i / C::kKStages))
          return false;
        tc_fence_after();
        const uint32_t d = tm_s + N * (i & 1);
        const uint32_t kt = k_lo + addr(s_k + ks * C::kKBytes), qt = k_lo + addr(base);
        auto step = [&](int s) {
          if constexpr (kE4m3) {
            mma_ss<true>(d, desc(kt + 2 * s, k_hi), desc(qt + 2 * s, k_hi), idesc_s, s > 0, one);
            mma_ss<true>(d, desc(kt + 2 * s, k_hi), desc(qt + C::kQPart / 16 + 2 * s, k_hi), idesc_s, 1, one);
          } else {
            mma_ss<false>(d, desc(kt + ((s >> 2) * kBlock + (s & 3) * 32) / 16, k_hi),
                          desc(qt + ((s >> 2) * C::kQPart + (s & 3) * 32) / 16, k_hi), idesc_s, s > 0, one);
          }
        };
        if (full_d) {
#pragma unroll
          for (int s = 0; s < DP / (kE4m3 ? 32 : 16); ++s) step(s);
        } else {
#pragma unroll 1
          for (int s = 0; s < k_steps; ++s) step(s);
        }
        commit(bar(sh.s_ready[i & 1]), one);
        commit(bar(sh.k_empty[ks]), one);
        return true;
      };
      // Scores two tiles ahead: a warpgroup finds its next ones when it has written its weights.
      if (ok) ok = scores(0);
      if (ok && n > 1) ok = scores(1);
      for (int it = 0; it < n && ok; ++it) {
        // the tile after next goes where this one's scores have been read
        if (it + 2 < n && !(ok = scores(it + 2))) break;
        // (values have been waited for, and made ready, by those who wrote the weights)
        if (!(ok = wait(sh.p_ready, it))) break;
        tc_fence_after();
        const uint32_t vt = v_lo + addr(kE4m3 ? base + C::kWideAt : s_v + it % C::kVStages * C::kVBytes), pt = v_lo + addr(s_p);
#pragma unroll
        for (int s = 0; s < kTile / 16; ++s)
          mma_ss<false>(tm_o, desc(vt + 128 * s, v_hi), desc(pt + 128 * s, v_hi), idesc_o, it > 0 || s > 0, one);
        commit(bar(sh.p_free), one);
        if (!kE4m3) commit(bar(sh.v_empty[it % C::kVStages]), one);
      }
    }
    __syncwarp();
  } else {
    const int wg = warp >> 2, quad = warp & 3, t = threadIdx.x & 127;
    const int group_bar = 1 + wg, c0 = 16 * wg;  // this warpgroup's columns
    const uint32_t lanes = static_cast<uint32_t>(32 * quad) << 16;
    auto all_sync = [&]() { asm volatile("barrier.cta.sync 3, 256;" ::: "memory"); };
    // columns' numbers, while nothing reads P
    float* const sums = reinterpret_cast<float*>(smem + C::kPAt);  // [quad][N]: of weights
    float* const weights = sums + 4 * N;
    int64_t* const places = reinterpret_cast<int64_t*>(weights + N);
    float* const halves = reinterpret_cast<float*>(places + N);    // e4m3: roots of O's units, which have more than f32's exponents
    // Where weights have to stay: bf16 below 2^20, so that their sums with values of 2^100 are f32; e4m3 below
    // 2^15 with their values' scales, and by themselves below 2^105, so that their sums are f32.  When a moves it
    // leaves this much room.
    // (kLeast: where a value's scale is 2^90 and more beside 1 / g.)
    constexpr float kMost = kE4m3 ? 105.f : 20.f, kLeast = -75.f, kRoom = kE4m3 ? 5.f : 20.f;
    bool alive = true;
    auto hold = [&](const uint64_t& x, int phase) {  // after an abort nothing is waited for any more
      if (alive) alive = wait(x, phase);
    };
    const bool mine = c0 < cols;  // this warpgroup has columns
    const int prefix = p.seq.length - p.seq.n, vis_min = max(prefix, 0), vis_max = p.seq.length;
    // ---------------------------------------------- the rows of Q
    {
      constexpr int kPerRow = C::kSoftmax / N;  // threads
      const int c = threadIdx.x / kPerRow, piece0 = threadIdx.x % kPerRow;
      const uint32_t row = static_cast<uint32_t>(p.rb) * N + c;
      const bool live = c < rows;
      const uint32_t token = live ? row_token(row, a.group) : 0, head = live ? row - token * a.group : 0;
      const uint16_t* src = a.q + (p.seq.row0 + token) * a.q_ld + (static_cast<int64_t>(p.hk) * a.group + head) * a.d;
      constexpr int kPieces = (DP / 8 + kPerRow - 1) / kPerRow;  // of 16 bytes
      uint4 x[kPieces];
#pragma unroll
      for (int k = 0; k < kPieces; ++k) {
        const int piece = piece0 + k * kPerRow;
        x[k] = make_uint4(0, 0, 0, 0);
        if (live && 8 * piece < a.d) x[k] = __ldg(reinterpret_cast<const uint4*>(src) + piece);
      }
      if (threadIdx.x < 2) sh.careful[threadIdx.x] = 0;
      if (piece0 == 0) {
        sh.row[c] = static_cast<int>(p.seq.row0 + token);
        sh.neg_a[c] = live ? kUnset : 0.f;
        sh.most[c] = ordered(-INFINITY);
        if constexpr (kE4m3) sh.d[c] = 0.f;
      }
      if constexpr (kE4m3) {
        uint32_t tops = 0;
#pragma unroll
        for (int k = 0; k < kPieces; ++k)
          tops = __vmaxu2(__vmaxu2(tops, __vmaxu2(x[k].x & 0x7FFF7FFFu, x[k].y & 0x7FFF7FFFu)),
                          __vmaxu2(x[k].z & 0x7FFF7FFFu, x[k].w & 0x7FFF7FFFu));
        uint32_t top = max(tops << 16, tops & 0xFFFF0000u);
#pragma unroll
        for (int o = 1; o < kPerRow; o <<= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        // times the power of two that puts the largest magnitude in [2^7, 2^8); a row that is not
        // finite gets NaN from its factor
        const bool finite = top < 0x7F800000u;
        const int e = top == 0 || !finite ? 7 : static_cast<int>(top >> 23) - 127;
        const int m = min(7 - e, 126);
        const float up = pow2(m);
        if (piece0 == 0)
          sh.f[c] = finite ? fmaxf(a.scale_log2 * pow2(-m), 0x1p-126f) : __uint_as_float(0x7FC00000u);
#pragma unroll
        for (int k = 0; k < 16 / kPerRow; ++k) {  // of all 128 channels: those from d on are zeros
          const int piece = piece0 + k * kPerRow;
          uint32_t hi[2] = {0, 0}, lo[2] = {0, 0};
          if (k < kPieces && finite) {
            const uint4& v = x[k < kPieces ? k : 0];
            const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e2 = 0; e2 < 4; ++e2) {
              const float y0 = __uint_as_float(u[e2] << 16) * up, y1 = __uint_as_float(u[e2] & 0xFFFF0000u) * up;
              uint16_t h, l;
              asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(h) : "f"(y1), "f"(y0));
              const uint32_t back = e4m3x2_f16x2(h, 0);
              float b0, b1;
              asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
                  : "=f"(b0), "=f"(b1) : "r"(back));
              asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(l) : "f"(y1 - b1), "f"(y0 - b0));
              hi[e2 >> 1] |= static_cast<uint32_t>(h) << (16 * (e2 & 1));
              lo[e2 >> 1] |= static_cast<uint32_t>(l) << (16 * (e2 & 1));
            }
          }
          uint8_t* dst = smem + c * 128 + (((piece >> 1) ^ (c & 7)) << 4) + 8 * (piece & 1);
          *reinterpret_cast<uint2*>(dst) = make_uint2(hi[0], hi[1]);
          *reinterpret_cast<uint2*>(dst + C::kQPart) = make_uint2(lo[0], lo[1]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
          const int piece = piece0 + k * kPerRow;
          if (piece < DP / 8)
            *reinterpret_cast<uint4*>(smem + (piece >> 3) * C::kQPart + c * 128 + (((piece & 7) ^ (c & 7)) << 4)) = x[k];
        }
      }
    }
    fence_proxy_async_smem();
    if (n > 0) warp_arrive(sh.q_ready);

    uint64_t l[8];  // sums of weights, in pairs of columns
#pragma unroll
    for (int e = 0; e < 8; ++e) l[e] = 0;
    float g = 1.f;  // e4m3: values' scales go times g = 2^-d
    // Columns whose rows do not see this thread's key of a tile (which may leave -inf to those that do).
    auto hidden_in = [&](int it) -> uint32_t {
      const int key_w = it * kTile + t - lane, left = vis_max - key_w;  // the warp's first key, keys from there on
      if ((it + 1) * kTile <= vis_min) return 0u;
      // which of the warp's 32 keys the columns' rows see: lane l has column l's bits
      const uint32_t valid = left >= 32 ? 0xFFFFFFFFu : left > 0 ? (1u << left) - 1u : 0u;
      uint32_t win = 0u, hidden = 0u;
      if (lane < 16 && valid) win = tree_bits(a, sh.row[c0 + lane], key_w - prefix) & valid;
#pragma unroll
      for (int e = 0; e < 16; ++e) hidden |= (~(__shfl_sync(0xFFFFFFFFu, win, e) >> lane) & 1u) << e;
      return hidden;
    };
    // A tile's values, made ready for their product, which the weights have been for.
    auto give_values = [&](int it) {
      const int vs = it % C::kVStages;
      uint8_t* const stage = smem + C::kVAt + vs * C::kVBytes;
      const int left = vis_max - it * kTile;
      hold(sh.v_full[vs], it / C::kVStages);
      if constexpr (kE4m3) {
        // Codes to fp16.  A warp has eight rows at a time, four lanes a row: codes 16 c .. and 64 +
        // 16 c .. of it (c = lane & 3).  Neighbouring groups of four take rows r and r ^ 5, so that neither
        // the reads nor the writes meet in a bank.
        constexpr int kPer = DP / 64, kWarps = C::kSoftmax / 32, kRounds = kTile / 8 / kWarps;
        const int c = lane & 3, pair_row = (lane >> 3) & 3, row8 = (lane & 4) ? pair_row ^ 5 : pair_row;
        uint4 u[kRounds][kPer];
#pragma unroll
        for (int k = 0; k < kRounds; ++k)
#pragma unroll
          for (int q = 0; q < kPer; ++q) {
            const int r = 8 * (warp + kWarps * k) + row8;
            u[k][q] = *reinterpret_cast<const uint4*>(stage + r * DP + (((c + 4 * q) ^ (DP == 128 ? row8 : 0)) << 4));
            if (r >= left) u[k][q] = make_uint4(0, 0, 0, 0);  // not this sequence's
          }
        warp_arrive(sh.v_empty[vs]);
#pragma unroll
        for (int k = 0; k < kRounds; ++k)
#pragma unroll
          for (int q = 0; q < kPer; ++q) {
            const uint4& v = u[k][q];
            uint8_t* row = smem + C::kWideAt + q * kBlock + (8 * (warp + kWarps * k) + row8) * 128;
            *reinterpret_cast<uint4*>(row + (((2 * c) ^ row8) << 4)) =
                make_uint4(e4m3x2_f16x2(v.x, 0), e4m3x2_f16x2(v.x, 1), e4m3x2_f16x2(v.y, 0), e4m3x2_f16x2(v.y, 1));
            *reinterpret_cast<uint4*>(row + (((2 * c + 1) ^ row8) << 4)) =
                make_uint4(e4m3x2_f16x2(v.z, 0), e4m3x2_f16x2(v.z, 1), e4m3x2_f16x2(v.w, 0), e4m3x2_f16x2(v.w, 1));
          }
      } else if ((it + 1) * kTile > vis_min) {  // values that not every row sees: 0 * NaN would reach rows that must not see it
        const int pc = lane & 7;
#pragma unroll 1
        for (int h = 0; h < C::kHalves; ++h)
#pragma unroll 2
          for (int r = 4 * warp + (lane >> 3); r < kTile; r += C::kSoftmax / 8) {
            uint4* const at = reinterpret_cast<uint4*>(stage + h * kBlock + r * 128 + pc * 16);
            if (r >= left) {
              *at = make_uint4(0, 0, 0, 0);
            } else if (it * kTile + r >= vis_min) {
              auto finite = [](uint32_t u) -> uint32_t {
                if ((u & 0x7F80u) == 0x7F80u) u &= 0xFFFF0000u;
                if ((u & 0x7F800000u) == 0x7F800000u) u &= 0x0000FFFFu;
                return u;
              };
              const uint4 v = *at, y = make_uint4(finite(v.x), finite(v.y), finite(v.z), finite(v.w));
              if (v.x != y.x || v.y != y.y || v.z != y.z || v.w != y.w) {
                *at = y;
                sh.any_bad = 1;
              }
            }
          }
      }
      fence_proxy_async_smem();
      tc_fence_before();
      warp_arrive(sh.p_ready);
    };
    all_sync();  // the columns' numbers are there
    int it = 0;
    for (; it < n; ++it) {
      const uint32_t ts = tm_s + N * (it & 1) + lanes + c0;
      const int key = it * kTile + t;
      const bool edge = (it + 1) * kTile > vis_min;
      const uint32_t hidden = hidden_in(it);
      hold(sh.s_ready[it & 1], it >> 1);
      tc_fence_after();
      float sk = 1.f, sv = 1.f, limit = kMost;
      if constexpr (kE4m3) {
        hold(sh.scales_full[it % C::kScaleSlots], it / C::kScaleSlots);
        const float* scales = reinterpret_cast<const float*>(smem + C::kScalesAt + (it % C::kScaleSlots) * C::kScaleBytes);
        const bool valid = key < vis_max;
        sk = valid ? scales[t] : 0.f;
        sv = valid ? scales[kTile + t] : 0.f;
        if (it == 0) {
          // g: one over a power of two near the first tile's largest scale.  (Not above 2^60: where
          // that tile holds nothing but zeros, whose scale is 2^-126, numbers may follow.)
          const uint32_t bits = fabsf(sv) < INFINITY ? __float_as_uint(fabsf(sv)) : 0u;
          const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, bits);
          if (lane == 0) sh.tops[wg][quad] = top;
          group_sync(group_bar);
          const uint32_t most = max(max(sh.tops[wg][0], sh.tops[wg][1]), max(sh.tops[wg][2], sh.tops[wg][3]));
          const int e = most == 0 ? 0 : static_cast<int>(most >> 23) - 127;
          const int shift = min(max(e, -60), 120);
          g = pow2(-shift);
          if (t < 16) sh.d[c0 + t] = static_cast<float>(shift);
        }
        sv = fmaf(sv, 0.f, sv) * g;  // an infinity becomes NaN
        limit = 15.f - fast_log2(fabsf(sv));
        if (!(limit > kLeast && limit < kMost)) limit = -INFINITY;  // beyond what one g allows: any score asks
      }
      // Scores relative to a, in log2 units.
      const uint64_t sk2 = pair(sk, sk), scale2 = pair(a.scale_log2, a.scale_log2);
      float x[16], top = -INFINITY;
      auto fetch = [&]() {
        uint32_t s[16];
        tmem_ld_x16(ts, s);
        tmem_wait_x16(s);
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const ulonglong2 ref = *reinterpret_cast<const ulonglong2*>(&sh.neg_a[c0 + e]);
          uint64_t s01 = pair(__uint_as_float(s[e]), __uint_as_float(s[e + 1]));
          uint64_t s23 = pair(__uint_as_float(s[e + 2]), __uint_as_float(s[e + 3]));
          if constexpr (kE4m3) {
            const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(&sh.f[c0 + e]);
            s01 = fma2(mul2(s01, f.x), sk2, ref.x);
            s23 = fma2(mul2(s23, f.y), sk2, ref.y);
          } else {
            s01 = fma2(s01, scale2, ref.x);
            s23 = fma2(s23, scale2, ref.y);
          }
          unpair(s01, x[e], x[e + 1]);
          unpair(s23, x[e + 2], x[e + 3]);
        }
        if (edge) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if ((hidden >> e) & 1u) x[e] = -INFINITY;
        }
      };
      if (mine) {
        fetch();
#pragma unroll
        for (int e = 0; e < 16; e += 2) top = max3(top, x[e], x[e + 1]);
      }
      if (group_any<128>(group_bar, top > limit)) {
        // ------------------------------------------ a moves: the columns' maxima across keys
        uint32_t s[16];
        tmem_ld_x16(ts, s);
        tmem_wait_x16(s);
        float most = -INFINITY;  // lane e: column e's
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float z = __uint_as_float(s[e]) * (kE4m3 ? sh.f[c0 + e] : a.scale_log2) * sk - limit;
          if ((hidden >> e) & 1u) z = -INFINITY;
          const float largest = warp_max(z);
          if ((lane & 15) == e) most = largest;
        }
        if (lane < 16 && most == most) atomicMax(&sh.most[c0 + lane], ordered(most));
        if (most > -INFINITY && fabsf(most) >= kBig) sh.careful[wg] = 1;
        group_sync(group_bar);
        __syncwarp();
        if (*static_cast<volatile int*>(&sh.careful[wg]) != 0) break;  // the same for all threads
        if (it > 0) {
          hold(sh.p_free, it - 1);
          tc_fence_after();
          float shrink[16];
          bool moved = false;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float was = -sh.neg_a[c0 + e], now = from_ordered(sh.most[c0 + e]);
            shrink[e] = now > was ? fast_exp2(was - (now + kRoom)) : 1.f;
            moved |= now > was;
          }
          if (moved) {  // the same for all threads
#pragma unroll
            for (int e = 0; e < 8; ++e) l[e] = mul2(l[e], pair(shrink[2 * e], shrink[2 * e + 1]));
#pragma unroll 1
            for (int h = 0; h < C::kPCols; h += N) {
              uint32_t o[16];
              tmem_ld_x16(tm_o + lanes + h + c0, o);
              tmem_wait_x16(o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * shrink[e]);
              tmem_st_x16(tm_o + lanes + h + c0, o);
              asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            }
          }
        }
        group_sync(group_bar);
        if (t < 16) {
          const float now = from_ordered(sh.most[c0 + t]);
          if (now > -sh.neg_a[c0 + t]) sh.neg_a[c0 + t] = -(now + kRoom);
          sh.most[c0 + t] = ordered(-INFINITY);
        }
        group_sync(group_bar);
        __syncwarp();
        fetch();
      }
      tc_fence_before();
      warp_arrive(sh.s_free[it & 1]);
      // ------------------------------------------ weights
      if (it > 0) hold(sh.p_free, it - 1);
      if (mine) {
        uint8_t* const prow = smem + C::kPAt + t * 128;
        auto put = [&](int c, const uint32_t (&v)[8]) {  // at columns c .. c + 15
          const int piece = c >> 3;
          *reinterpret_cast<uint4*>(prow + ((piece ^ (t & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
          *reinterpret_cast<uint4*>(prow + (((piece + 1) ^ (t & 7)) << 4)) = make_uint4(v[4], v[5], v[6], v[7]);
        };
        const uint64_t sv2 = pair(sv, sv), minus = pair(-1.f, -1.f);
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          uint64_t w = pair(fast_exp2(x[2 * e]), fast_exp2(x[2 * e + 1]));
          l[e] = add2(l[e], w);
          float p0, p1;
          if constexpr (kE4m3) {
            w = mul2(w, sv2);
            unpair(w, p0, p1);
            if (edge) {  // a hidden key's scale may be anything
              if ((hidden >> (2 * e)) & 1u) p0 = 0.f;
              if ((hidden >> (2 * e + 1)) & 1u) p1 = 0.f;
            }
            hi[e] = pack_f16(p0, p1);
          } else {
            unpair(w, p0, p1);
            hi[e] = pack_bf16(p0, p1);
            unpair(fma2(pair(__uint_as_float(hi[e] << 16), __uint_as_float(hi[e] & 0xFFFF0000u)), minus, w), p0, p1);
            lo[e] = pack_bf16(p0, p1);
          }
        }
        put(c0, hi);
        if constexpr (!kE4m3) put(N + c0, lo);
      }
      give_values(it);
    }
    // ---------------------------------------------- careful steps (see tree_tiles.cuh), from tile `it` on
    if (it < n) {
      if (t < 16) sh.most[c0 + t] = ordered(-INFINITY);
      group_sync(group_bar);
      for (; it < n; ++it) {
        const int key = it * kTile + t;
        const uint32_t hidden = hidden_in(it);
        hold(sh.s_ready[it & 1], it >> 1);
        float sk = 1.f, sv = 1.f;
        if constexpr (kE4m3) {
          hold(sh.scales_full[it % C::kScaleSlots], it / C::kScaleSlots);
          const float* scales = reinterpret_cast<const float*>(smem + C::kScalesAt + (it % C::kScaleSlots) * C::kScaleBytes);
          sk = key < vis_max ? scales[t] : 0.f;
          sv = key < vis_max ? scales[kTile + t] : 0.f;
        }
        if (it > 0) hold(sh.p_free, it - 1);
        tc_fence_after();
        careful_step<kE4m3, N>(CarefulColumns{sh.neg_a + c0, sh.d + (kE4m3 ? c0 : 0), sh.most + c0, sh.shrink_l + c0,
                                              sh.shrink_o + c0, sh.f + (kE4m3 ? c0 : 0)},
                               group_bar, tm_s + N * (it & 1) + lanes + c0, tm_o + lanes + c0, it > 0, hidden,
                               a.scale_log2, sk, sv, smem + C::kPAt + t * 128, c0, l);
        tc_fence_before();
        warp_arrive(sh.s_free[it & 1]);
        give_values(it);
      }
    }
    // ---------------------------------------------- out
    if (n > 0) hold(sh.p_free, n - 1);  // the last product
    tc_fence_after();
    tc_fence_before();
    all_sync();  // nothing reads P any more, and O is whole
    tc_fence_after();
    if (mine) {
      float v[16];
#pragma unroll
      for (int e = 0; e < 8; ++e) unpair(l[e], v[2 * e], v[2 * e + 1]);
      const float sum = sum16(v);
      if (!(lane & 1)) sums[quad * N + c0 + (lane >> 1)] = sum;
    }
    const bool bad_page = n > 0 && sh.bad_page, some_bad = !kE4m3 && n > 0 && sh.any_bad;
    if (threadIdx.x == 0 && bad_page) paged_report(a.status);
    all_sync();
    const int ch = 32 * quad + lane;
    if (threadIdx.x < cols) {  // a thread settles a column
      const int c = threadIdx.x;
      const float* x = sums + c;
      float total = (x[0] + x[N]) + (x[2 * N] + x[3 * N]);
      if (bad_page || !alive) total = __uint_as_float(0x7FC00000u);
      const int64_t row = static_cast<int64_t>(p.rb) * N + c, token = sh.row[c] - p.seq.row0;
      places[c] = static_cast<int64_t>(sh.row[c]) * a.out_ld + (static_cast<int64_t>(p.hk) * a.group + row - token * a.group) * a.d;
      weights[c] = total == 0.f ? 0.f : 1.f / total;
      if constexpr (kE4m3) halves[c] = fast_exp2(0.5f * sh.d[c]);
    }
    all_sync();
    if (mine) {
      float y[16] = {};
      if (n > 0) {
        constexpr int kParts = C::kPCols / N;
        uint32_t o[kParts][16];
#pragma unroll
        for (int h = 0; h < kParts; ++h) tmem_ld_x16(tm_o + lanes + N * h + c0, o[h]);
#pragma unroll
        for (int h = 0; h < kParts; ++h) tmem_wait_x16(o[h]);
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const float4 f = *reinterpret_cast<const float4*>(&weights[c0 + e]);
          const float w4[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float v = __uint_as_float(o[0][e + k]);
            if constexpr (kParts > 1) v += __uint_as_float(o[kParts - 1][e + k]);
            y[e + k] = v * w4[k];
          }
        }
      }
      if (some_bad) {
#pragma unroll 1
        for (int e = 0; e < 16; ++e) {
          const bool bad = c0 + e < rows && ch < a.d &&
                           tree_sees_bad<kE4m3>(a, p.seq, a.table + p.table, p.hk, sh.row[c0 + e], ch);
#pragma unroll
          for (int k = 0; k < 16; ++k)
            if (bad && k == e) y[k] = __uint_as_float(0x7FC00000u);
        }
      }
      if (ch < a.d) {
        uint16_t* const to = a.out + ch;
#pragma unroll
        for (int e = 0; e < 16; ++e)  // a sum of 0 has made y 0, or left it NaN
          if (c0 + e < rows) {
            if constexpr (kE4m3) y[e] = y[e] * halves[c0 + e] * halves[c0 + e];
            to[places[c0 + e]] = __bfloat16_as_ushort(__float2bfloat16_rn(y[e]));
          }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == kMma) {
    tc_fence_after();
    tmem_dealloc(sh.tmem, C::kTmemCols);
  }
}

template <bool kE4m3, int DP>
cudaError_t launch_short(const PagedArgs& a, cudaStream_t stream) {
  using C = ShortCfg<kE4m3, DP, kTreeRows>;
  CUtensorMap mk, mv;
  const int box_rows = 1 << a.page_log2;
  if (!make_page_map(&mk, a.k, a, 128, box_rows, 1) ||
      !make_page_map(&mv, a.v, a, kE4m3 ? DP : 128, box_rows, 1))
    return cudaErrorInvalidValue;
  constexpr auto kKernel = short_tree_kernel<kE4m3, DP, kTreeRows>;
  if (cudaError_t e = allow_smem_once<kKernel>(C::kSmem); e != cudaSuccess) return e;
  const int64_t row_units = (static_cast<int64_t>(a.max_q) * a.group + kTreeRows - 1) / kTreeRows;
  const int64_t grid = static_cast<int64_t>(a.B) * a.H_kv * row_units;
  if (grid > 0x7FFFFFFFll) return cudaErrorInvalidConfiguration;
  kKernel<<<static_cast<unsigned>(grid), C::kThreads, C::kSmem, stream>>>(mk, mv, a, static_cast<uint32_t>(row_units));
  return cudaGetLastError();
}

}  // namespace

// Whether a call of more than kFewRows rows comes here: where there are more units than SMs, and contexts, by
// the table's width, are short for that, so that a block with a unit of its own is through about when the
// others are; and where a unit is one step.  Measured with 128 channels, us, contexts all as long and ragged
// ones, here and else:
//   32 rows, bf16:   128 units over 128 8.8 and 9.0 (else 9.4, 9.5), over 1024 17.3 and 16.7 (14.9, 14.4)
//                    256 units over 1024 30.6 and 20.3 (39.6, 29.0), over 4096 86.8 and 67.9 (94.2, 63.9)
//                    1024 units over 512 67.0 and 51.7 (72.3, 73.2), over 2048 183 and 101 (180, 109)
//   64 rows, bf16:   256 heads over 512 29.6 and 23.5 (29.4, 24.9), over 1024 46.6 and 30.1 (41.5, 30.7: with 8 bits
//                    of the probabilities instead of 16), over 2048 73.8 and 46.7 (63.6, 42.9)
//   64 rows, e4m3:   256 heads over 2048 77.1 and 45.8 (78.2, 50.1), over 4096 136.2 and 71.8 (133.8, 77.2)
// More rows than 64 read the same keys too often: 128 rows of 128 heads over 128 tokens 20.3 (12.0).
bool tree_is_short(const PagedArgs& a) {
  const int64_t rows = static_cast<int64_t>(a.max_q) * a.group;
  const int64_t steps = ((static_cast<int64_t>(a.max_pages) << a.page_log2) + kTile - 1) / kTile;
  const int64_t units = static_cast<int64_t>(a.B) * a.H_kv;
  if (rows <= kTreeRows) return steps <= 1 || (units > device_sm_count() && 8 * steps < units);
  return rows <= 2 * kTreeRows && steps <= (a.k_scale != nullptr ? 16 : 8) && 4 * steps <= units && !tree_has_room(a);
}

cudaError_t launch_tree_attention_short(const PagedArgs& a, cudaStream_t stream) {
  const bool e4m3 = a.k_scale != nullptr;
  if (a.d <= 64) return e4m3 ? launch_short<true, 64>(a, stream) : launch_short<false, 64>(a, stream);
  return e4m3 ? launch_short<true, 128>(a, stream) : launch_short<false, 128>(a, stream);
}

}  // namespace dwa
