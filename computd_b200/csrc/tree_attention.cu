// tree_attention.cu — attention of a tree's nodes over the paged cache on tcgen05, for
// more rows per key/value head than paged_attention.cu takes.
//
// A row is one (node, query head of the group), node-major.  A unit is up to 32 rows of one key/value
// head; it goes over the sequence's keys 128 at a time, its products transposed:
//
//   S^T = K Q^T       128 keys by 32 rows     tcgen05, K and Q in shared memory, S in TMEM
//   P   = exp2(S - a) a thread per key and 16 rows
//   O^T += V^T P      128 channels by 32 rows tcgen05, V and P in shared memory, O in TMEM
//
// so that neither the tensor pipe nor the exponentials work on rows that are not there: a tile
// of 128 rows would be 75 to 87 % empty.  A key's scales (e4m3) are one number of its thread's.
//
// What a row's weights are relative to, a, is not its maximum but anything that keeps them in
// range; it moves when a score passes the limit, which every step asks by a vote, and only
// then are maxima taken across keys.  The limit is 2^20 for bf16 (whose range is f32's) and for e4m3
// what keeps a weight times its value's scale below 2^15 in fp16.  Scores of 2^20 and more, and values' scales 2^90 apart,
// take the careful steps of tree_tiles.cuh.
//
// Rounding: bf16 caches none beside f32 sums (P is the sum of two bf16 parts).  e4m3: codes are
// exact; Q is, per row, a power of two times the sum of two e4m3 numbers, exactly down to 2^-9 of the
// row's largest value and to 2^-18 of that below (so that keys go into their product as they lie in the
// cache, at twice the rate of fp16 and without a conversion); P times the value's scale is
// rounded to fp16, 11 bits.
//
// Bound by HBM where contexts are long and all as long: 16 sequences of 32 nodes over 4096 tokens, 16 heads of
// 128 channels, bf16, 94 us, 5.7 TB/s; else by the length of a step's chain (loads from TMEM, vote, exponentials,
// stores, product) and by what a unit costs beside its steps: 20 to 32 nodes over 300 to 4096 tokens 56 us, 4.8 TB/s
// (floor 41); one sequence over 4096 20 us, e4m3 21.  (More rows are no work for this layout: a thread reads
// its columns' references, 4 bytes each, from shared memory, which with 64 or 128 columns takes as long as all
// else.)
// Work is cut by steps, not by units: each block takes an equal share of all steps, whatever sequence they
// belong to, and writes a unit that it has only a part of to a workspace, from which a second
// kernel joins the parts in a fixed order.
//
// Sixteen warps: softmax, a warpgroup to sixteen columns of every other tile (with eight warps a step's
// chain was twice as long); e4m3: they turn the values' codes into fp16 too, bf16: they look over
// the values of the tree's nodes, since 0 * NaN would reach rows that must not see it.  One warp: tcgen05.mma.  Two:
// TMA, straight from the pages.  One: the block's next parts.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "dwa_internal.h"
#include "f32x2.cuh"
#include "paged_attention.cuh"
#include "sm100_ptx.cuh"
#include "tree_tiles.cuh"

namespace dwa {

namespace {

constexpr int kLeastShare = 6;    // of a block, in steps
// What a unit costs beside its steps: Q, first references and the way out.  Work is shared out in
// steps and these, so that short sequences' units do not pile up in a few blocks (24 ragged ones of 50 to 1500 tokens,
// 16 heads of 80: 112 us without).
constexpr int kUnitCost = 4;
constexpr int kSmemLimit = 227 * 1024;

template <bool kE4m3, int DP, int N>
struct TreeCfg {
  static constexpr int kThreads = 640, kSoftmax = 512, kSoftmaxRegs = 104, kOtherRegs = 64;
  // Four warpgroups: two for each of alternate tiles of keys (a side), each with sixteen columns.
  static constexpr int kSharers = 2;
  static_assert(N == 16 * kSharers);
  static constexpr int kHalves = DP / 64;
  static constexpr int kQPart = N * 128;                       // 64 bf16 channels, or 128 codes
  static constexpr int kQBytes = (kE4m3 ? 2 : kHalves) * kQPart;
  static constexpr int kPCols = (kE4m3 ? 1 : 2) * N;           // bf16: both parts of P side by side, in one product
  static constexpr int kPBytes = kBlock;                       // of a buffer, and a side has one
  static constexpr int kPBufs = 2;
  static constexpr int kKBytes = (kE4m3 ? 1 : kHalves) * kBlock;
  // Codes of values arrive where their fp16 values go (128 channels: the second block), or behind it.
  static constexpr int kRawAt = kBlock;
  static constexpr int kVBytes = kHalves * kBlock + (kE4m3 && DP == 64 ? kTile * 64 : 0);
  static constexpr int kStatic = 3 * 1024;  // at most
  // e4m3: scales of the keys and values of eight tiles: keys are up to kKStages + 2 tiles ahead of the softmax
  static constexpr int kScaleBytes = kE4m3 ? 2 * kTile * 4 : 0, kScaleSlots = 8;
  static constexpr int kLeft = kSmemLimit - 1024 - kStatic - kQBytes - kPBufs * kPBytes - kScaleSlots * kScaleBytes;
  static constexpr bool fits(int k, int v) { return k * kKBytes + v * kVBytes <= kLeft; }
  // Scores run two tiles ahead, so that a tile of values is held longer than one of keys.
  static constexpr int kVStages = fits(2, 4) ? 4 : fits(2, 3) ? 3 : 2;
  static constexpr int kKStages = fits(4, kVStages) ? 4 : fits(3, kVStages) ? 3 : 2;
  static_assert(fits(kKStages, kVStages) && kKStages + 2 < kScaleSlots, "tiles fit");
  static constexpr int kKAt = kQBytes, kVAt = kKAt + kKStages * kKBytes, kPAt = kVAt + kVStages * kVBytes;
  static constexpr int kScalesAt = kPAt + kPBufs * kPBytes;
  static constexpr int kSmem = 1024 + kScalesAt + kScaleSlots * kScaleBytes;
  // TMEM: two S, then O of each P buffer
  static constexpr int kColsUsed = 2 * N + kPBufs * kPCols;
  static constexpr int kTmemCols = kColsUsed > 256 ? 512 : kColsUsed > 128 ? 256 : 128;
};

// ---------------------------------------------------------------- work
struct Part {
  int hk, rb;          // key/value head, block of rows
  int tile0, n, steps; // its tiles of 128 keys (n = 0: nothing to read) of the unit's `steps`
  int64_t row0;        // the sequence, as PagedSeq has it, and its pages
  int seq_n, length;
  int64_t table;
  bool bad, whole, last;  // last: there is no such part, the block is done
};

struct Plan {       // of a block
  int64_t g, end;   // cost, counted over all units: of each kUnitCost, then its steps
  int b;            // the sequence of cost g, and the cost before it
  int64_t base;
  int64_t total, share;
};

// Tiles and blocks of rows of a sequence.  (One step for rows that see no key, or get NaN.)
__device__ __forceinline__ int64_t tree_steps(const PagedSeq& s) {
  return s.n == 0 ? 0 : s.bad ? 1 : max((s.length + kTile - 1) / kTile, 1);
}
template <int N>
__device__ __forceinline__ int64_t tree_blocks(const PagedArgs& a, const PagedSeq& s) {
  return (static_cast<int64_t>(s.n) * a.group + N - 1) / N;
}

// Block c's share of `blocks` blocks', found by the block together; `scratch` is shared memory.
constexpr int kPlanScratch = 32 + 3;  // 64-bit words
template <int N, int kThreads>
__device__ __forceinline__ Plan make_plan(const PagedArgs& a, int c, int blocks, int64_t* scratch) {
  int64_t* const warp_sums = scratch;
  unsigned long long& all = reinterpret_cast<unsigned long long&>(scratch[32]);
  int64_t &found_base = scratch[33], &found_b = scratch[34];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto steps_of = [&](int b) -> int64_t {
    if (b >= a.B) return 0;
    const PagedSeq s = paged_seq(a, b);
    return s.n == 0 ? 0 : (kUnitCost + tree_steps(s)) * tree_blocks<N>(a, s) * a.H_kv;
  };
  if (threadIdx.x == 0) {
    all = 0;
    found_b = a.B;
    found_base = 0;
  }
  __syncthreads();
  int64_t mine = 0;
  const int64_t first = steps_of(threadIdx.x);
  mine = first;
  for (int b = threadIdx.x + kThreads; b < a.B; b += kThreads) mine += steps_of(b);
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xFFFFFFFFu, mine, o);
  if (lane == 0 && mine) atomicAdd(&all, static_cast<unsigned long long>(mine));
  __syncthreads();
  Plan p;
  p.total = static_cast<int64_t>(all);
  p.share = max((p.total + blocks - 1) / blocks, static_cast<int64_t>(kLeastShare));
  p.g = min(c * p.share, p.total);
  p.end = min(p.g + p.share, p.total);
  int64_t before = 0;
  for (int b0 = 0; b0 < a.B; b0 += kThreads) {  // the sequence that has step g
    const int b = b0 + threadIdx.x;
    const int64_t w = b0 == 0 ? first : steps_of(b);
    int64_t incl = w;
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xFFFFFFFFu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    int64_t base = before, sum = 0;
    for (int i = 0; i < kThreads / 32; ++i) {
      if (i < warp) base += warp_sums[i];
      sum += warp_sums[i];
    }
    base += incl - w;
    if (b < a.B && p.g >= base && p.g < base + w) {
      found_b = b;
      found_base = base;
    }
    before += sum;
    __syncthreads();
    if (p.g < before) break;
  }
  p.b = static_cast<int>(found_b);
  p.base = found_base;
  return p;
}

__device__ __forceinline__ void set_seq(Part& p, const PagedArgs& a, int b, const PagedSeq& s) {
  p.row0 = s.row0;
  p.seq_n = s.n;
  p.length = s.length;
  p.bad = s.bad;
  p.table = static_cast<int64_t>(b) * a.ld_table;
}
// The next part of the block's share, if there is one; *of_unit: where in its unit's cost the share, or
// the unit, begins.
template <int N>
__device__ __forceinline__ bool next_part(const PagedArgs& a, Plan& w, Part& p, int64_t* of_unit) {
  while (w.g < w.end) {
    PagedSeq seq;
    int64_t steps, blocks;
    while (true) {
      seq = paged_seq(a, w.b);
      steps = tree_steps(seq);
      blocks = tree_blocks<N>(a, seq);
      const int64_t all = seq.n == 0 ? 0 : (kUnitCost + steps) * blocks * a.H_kv;
      if (w.g - w.base < all) break;
      w.base += all;
      ++w.b;
    }
    const int64_t local = w.g - w.base, cost = kUnitCost + steps;
    int64_t unit;
    if (local >> 32) unit = local / cost;
    else unit = static_cast<uint32_t>(local) / static_cast<uint32_t>(cost);  // cost: below 2^24
    const int64_t from = local - unit * cost, to = min(cost, from + (w.end - w.g));
    w.g += to - from;
    const int64_t tile0 = max(from - kUnitCost, int64_t{0}), tile1 = max(to - kUnitCost, int64_t{0});
    if (tile1 == tile0) continue;  // the next block begins it
    set_seq(p, a, w.b, seq);
    p.hk = (unit | blocks) >> 32 ? static_cast<int>(unit / blocks)
                                 : static_cast<int>(static_cast<uint32_t>(unit) / static_cast<uint32_t>(blocks));
    p.rb = static_cast<int>(unit - p.hk * blocks);
    p.tile0 = static_cast<int>(tile0);
    p.steps = static_cast<int>(steps);
    p.n = seq.bad || seq.length == 0 ? 0 : static_cast<int>(tile1 - tile0);
    p.whole = tile1 - tile0 == steps;
    p.last = false;
    *of_unit = from;
    return true;
  }
  return false;
}

template <int kRegs>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// ---------------------------------------------------------------- the kernel
template <bool kE4m3, int N>
struct TreeShared {
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4], part_full[4], part_empty[4];
  uint64_t scales_full[kE4m3 ? 8 : 1];
  uint64_t q_ready, s_ready[2], s_free[2], p_ready[2], p_free[2];
  uint32_t tmem;
  int abort;
  Part parts[4];                // under way, by their number
  int bad_page[8], any_bad[8];
  alignas(16) float neg_a[2 * N];  // minus what a column's weights are relative to (of each side)
  alignas(16) float f[kE4m3 ? N : 4];     // its scores' factor, to log2 units
  int most[2 * N];  // across keys, ordered
  int row[N];                   // of q
  uint32_t tops[4][4];          // e4m3: scales' exponents
  float d[kE4m3 ? 2 * N : 4];   // e4m3: O's units are 2^d beside the references', of each side
  float shrink_l[2 * N], shrink_o[2 * N];
  int careful[4];               // of each warpgroup
};

struct TreeArgs {
  PagedArgs p;
  float* parts;   // null: every block has whole units
  int row_units;  // blocks of rows of a sequence, at most (without parts)
};

// A part's place in the workspace: a, l and the exponent of O's unit beside 2^a by rows, then O.
template <int DP, int N>
__device__ __forceinline__ float* part_at(float* parts, int block, bool begins) {
  return parts + (static_cast<int64_t>(block) * 2 + (begins ? 1 : 0)) * (N * (DP + 3));
}

template <bool kE4m3, int DP, int N>
__global__ void __launch_bounds__(TreeCfg<kE4m3, DP, N>::kThreads, 1)
    tree_attention_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                          const __grid_constant__ TreeArgs ta) {
  using C = TreeCfg<kE4m3, DP, N>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ TreeShared<kE4m3, N> sh;
  static_assert(sizeof(TreeShared<kE4m3, N>) <= C::kStatic, "as much as is left for it");
  const PagedArgs& a = ta.p;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kMma = C::kSoftmax / 32, kTma = kMma + 1, kPlanner = kMma + 3;  // warps; two for TMA

  // ------------------------------------------------ the block's work
  Plan plan{};
  if (ta.parts != nullptr) {
    plan = make_plan<N, C::kThreads>(a, blockIdx.x, gridDim.x, reinterpret_cast<int64_t*>(smem));
    if (blockIdx.x == 0)
      for (int b = threadIdx.x; b < a.B; b += C::kThreads)
        if (paged_seq(a, b).bad) paged_report(a.status);
    if (plan.g >= plan.end) return;
  }

  // ------------------------------------------------ set-up
  auto bar = [&](const uint64_t& x) { return smem_u32(&x); };
  if (warp == kPlanner && lane == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(bar(sh.k_full[i]), 1);
      mbar_init(bar(sh.k_empty[i]), 1);
      mbar_init(bar(sh.v_full[i]), 1);
      mbar_init(bar(sh.part_full[i]), 1);
      mbar_init(bar(sh.part_empty[i]), kPlanner);  // a warp each
      mbar_init(bar(sh.v_empty[i]), 1);
    }
    for (int i = 0; i < 8; ++i) sh.bad_page[i] = sh.any_bad[i] = 0;
    for (int i = 0; i < (kE4m3 ? 8 : 1); ++i) mbar_init(bar(sh.scales_full[i]), 1);
    mbar_init(bar(sh.q_ready), C::kSoftmax / 32);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(sh.s_ready[i]), 1);
      mbar_init(bar(sh.s_free[i]), 4 * C::kSharers);
      mbar_init(bar(sh.p_ready[i]), 4 * C::kSharers);
      mbar_init(bar(sh.p_free[i]), 1);
    }
    sh.abort = 0;
    fence_mbar_init();
  }
  if (warp == kMma) {
    tmem_alloc(smem_u32(&sh.tmem), C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm_s = sh.tmem, tm_o = sh.tmem + 2 * N;  // S: + N (it & 1); O: + kPCols (P's buffer)
  // the buffer of P and O that tile `it` goes through, and which use of it that is
  auto p_buf = [](int it) -> int { return it & 1; };
  auto p_use = [](int it) -> int { return it >> 1; };
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
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // join_parts_kernel, where there is room
  const uint32_t s_k = base + C::kKAt, s_v = base + C::kVAt, s_p = base + C::kPAt;
  auto rows_of = [&](int seq_n, int rb) -> int {  // of the unit
    return static_cast<int>(min(static_cast<int64_t>(seq_n) * a.group - static_cast<int64_t>(rb) * N,
                                static_cast<int64_t>(N)));
  };

  if (warp >= kMma) {
    regs_dec<C::kOtherRegs>();
    if (warp == kPlanner) {
      // ---------------------------------------------- the parts, a few ahead
      Plan w = plan;
      for (int part = 0;; ++part) {
        Part p{};
        if (ta.parts != nullptr) {
          int64_t at;
          p.last = !next_part<N>(a, w, p, &at);
        } else {  // one unit: (sequence, head, block of rows)
          const uint32_t unit = blockIdx.x, of_seq = unit / static_cast<uint32_t>(ta.row_units);
          const int b = static_cast<int>(of_seq / static_cast<uint32_t>(a.H_kv));
          const PagedSeq seq = paged_seq(a, b);
          set_seq(p, a, b, seq);
          p.rb = static_cast<int>(unit - of_seq * ta.row_units);
          p.hk = static_cast<int>(of_seq - static_cast<uint32_t>(b) * a.H_kv);
          p.steps = static_cast<int>(tree_steps(seq));
          p.n = seq.bad || seq.length == 0 ? 0 : p.steps;
          p.whole = true;
          p.last = part > 0 || !(p.rb < tree_blocks<N>(a, seq) || (seq.bad && p.rb == 0));
        }
        if (part >= 4 && !wait(sh.part_empty[part & 3], (part >> 2) - 1)) break;
        if (lane == 0) {
          sh.parts[part & 3] = p;
          mbar_arrive(bar(sh.part_full[part & 3]));
        }
        __syncwarp();
        if (p.last) break;
      }
    } else if (warp != kMma) {
      // ---------------------------------------------- TMA: a warp for keys, one for values
      const bool values = warp == kTma + 1;
      const int stages = values ? C::kVStages : C::kKStages, stage_bytes = values ? C::kVBytes : C::kKBytes;
      const uint32_t tiles = values ? s_v + (kE4m3 ? C::kRawAt : 0) : s_k;
      const uint32_t full0 = values ? bar(sh.v_full[0]) : bar(sh.k_full[0]);
      const uint32_t empty0 = values ? bar(sh.v_empty[0]) : bar(sh.k_empty[0]);
      const CUtensorMap* map = values ? &map_v : &map_k;
      const int row_bytes = values && kE4m3 ? DP : 128;
      const int page_size = 1 << a.page_log2, of_tile = kTile >> a.page_log2;  // pages of a tile: 1 to 8
      int stage = 0, use = 0, slot = 0;
      bool ok = true;
      for (int part = 0; ok && (ok = wait(sh.part_full[part & 3], part >> 2)); ++part) {
        const Part& p = sh.parts[part & 3];
        if (p.last) break;
        const int32_t* table = a.table + p.table;
        const int n = p.n, hk = p.hk, page0 = p.tile0 * of_tile;
        const int pages = (p.length + page_size - 1) >> a.page_log2;
        warp_arrive(sh.part_empty[part & 3]);
        int held = 0;  // the pages of the next 4 to 32 tiles, a page to a lane
        for (int j = 0; j < n; ++j) {
          const int at = (j * of_tile) & 31;
          if (at == 0) {
            const int i = page0 + j * of_tile + lane;
            held = i < pages ? __ldg(table + i) : 0;
            if (held < 0 || held >= a.n_pages) {
              if (i < page0 + n * of_tile) sh.bad_page[part & 7] = 1;  // read page 0 in its place; the rows become NaN
              held = 0;
            }
          }
          const int here = min(of_tile, pages - page0 - j * of_tile);
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
    } else {
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
      int it = 0, parts = 0;
      bool ok = true;
      for (int part = 0; ok && (ok = wait(sh.part_full[part & 3], part >> 2)); ++part) {
        const Part& p = sh.parts[part & 3];
        if (p.last) break;
        const int n = p.n;
        const uint32_t cols = static_cast<uint32_t>((rows_of(p.seq_n, p.rb) + 15) & ~15);
        warp_arrive(sh.part_empty[part & 3]);
        if (n == 0) continue;
        const uint32_t idesc_s = (1u << 4) | kF16 | (cols / 8 << 17) | kM;
        const uint32_t idesc_o = (1u << 4) | kF16 | (1u << 15) | (1u << 16) | ((C::kPCols - N + cols) / 8 << 17) | kM;
        ok = wait(sh.q_ready, parts++);
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
        const int first = it;
        if (ok) ok = scores(it);
        if (ok && n > 1) ok = scores(it + 1);
        for (int j = 0; j < n && ok; ++j, ++it) {
          // the tile after next goes where this one's scores have been read
          if (j + 2 < n && !(ok = scores(first + j + 2))) break;
          const int vs = it % C::kVStages, buf = p_buf(it);
          // (values have been waited for, and made ready, by those who wrote the weights)
          if (!(ok = wait(sh.p_ready[buf], p_use(it)))) break;
          tc_fence_after();
          const uint32_t vt = v_lo + addr(s_v + vs * C::kVBytes), pt = v_lo + addr(s_p + C::kPBytes * buf);
#pragma unroll
          for (int s = 0; s < kTile / 16; ++s)
            mma_ss<false>(tm_o + C::kPCols * buf, desc(vt + 128 * s, v_hi), desc(pt + 128 * s, v_hi), idesc_o,
                          j >= C::kPBufs || s > 0, one);
          commit(bar(sh.p_free[buf]), one);
          commit(bar(sh.v_empty[vs]), one);
        }
      }
    }
    __syncwarp();
  } else {
    regs_inc<C::kSoftmaxRegs>();
    const int wg = warp >> 2, quad = warp & 3, t = threadIdx.x & 127;
    const int group_bar = 1 + wg, side = wg >> 1, c0 = 16 * (wg % C::kSharers);  // c0: this warpgroup's columns
    const uint32_t lanes = static_cast<uint32_t>(32 * quad) << 16;
    auto all_sync = [&]() { asm volatile("barrier.cta.sync 5, 512;" ::: "memory"); };
    float* const neg_a = sh.neg_a + side * N;
    int* const mosts = sh.most + side * N;
    // columns' numbers, while nothing reads P
    float* const sums = reinterpret_cast<float*>(smem + C::kPAt);  // [side][quad][N]: of weights
    float* const weights = sums + 1024;                            // [side][N]: of the accumulators
    int64_t* const places = reinterpret_cast<int64_t*>(weights + 2 * N);
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
    int it0 = 0;
    for (int part = 0;; ++part) {
      hold(sh.part_full[part & 3], part >> 2);
      // together, and only behind the last part's reads of the columns' numbers; all stop, or none
      if (group_any<C::kSoftmax>(5, !alive)) break;
      const Part& p = sh.parts[part & 3];
      if (p.last) break;
      const int64_t all_rows = static_cast<int64_t>(p.seq_n) * a.group;
      if (p.bad) {
        if (ta.parts == nullptr && p.hk == 0 && p.rb == 0 && threadIdx.x == 0) paged_report(a.status);
        // rows N rb .., and without parts, where max_q does not bound them, every row_units-th block
        const int64_t by = ta.parts == nullptr ? static_cast<int64_t>(ta.row_units) * N : all_rows;
        for (int64_t r0 = static_cast<int64_t>(p.rb) * N; r0 < all_rows; r0 += by)
          for (int64_t i = threadIdx.x; i < min(static_cast<int64_t>(N), all_rows - r0) * a.d; i += C::kSoftmax) {
            const int64_t row = r0 + i / a.d;
            a.out[(p.row0 + row / a.group) * a.out_ld +
                  (static_cast<int64_t>(p.hk) * a.group + row % a.group) * a.d + i % a.d] = 0x7FC0u;
          }
        warp_arrive(sh.part_empty[part & 3]);
        continue;
      }
      const int n = p.n, tile0 = p.tile0, rows = rows_of(p.seq_n, p.rb), cols = (rows + 15) & ~15;
      const int prefix = p.length - p.seq_n, vis_min = max(prefix, 0), vis_max = p.length;
      // ---------------------------------------------- the rows of Q
      {
        constexpr int kPerRow = C::kSoftmax / N;  // threads
        const int c = threadIdx.x / kPerRow, piece0 = threadIdx.x % kPerRow;
        const uint32_t row = static_cast<uint32_t>(p.rb) * N + c;
        const bool live = c < rows;
        const uint32_t token = live ? row_token(row, a.group) : 0, head = live ? row - token * a.group : 0;
        const uint16_t* src = a.q + (p.row0 + token) * a.q_ld + (static_cast<int64_t>(p.hk) * a.group + head) * a.d;
        constexpr int kPieces = (DP / 8 + kPerRow - 1) / kPerRow;  // of 16 bytes
        uint4 x[kPieces];
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
          const int piece = piece0 + k * kPerRow;
          x[k] = make_uint4(0, 0, 0, 0);
          if (live && 8 * piece < a.d) x[k] = __ldg(reinterpret_cast<const uint4*>(src) + piece);
        }
        if (threadIdx.x < 4) sh.careful[threadIdx.x] = 0;
        if (piece0 == 0) {
          sh.row[c] = static_cast<int>(p.row0 + token);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            sh.neg_a[k * N + c] = live ? kUnset : 0.f;
            sh.most[k * N + c] = ordered(-INFINITY);
            if constexpr (kE4m3) sh.d[k * N + c] = 0.f;
          }
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

      const bool mine = c0 < cols;
      uint64_t l[8];  // sums of weights, in pairs of columns
#pragma unroll
      for (int e = 0; e < 8; ++e) l[e] = 0;
      // The tiles of this side: j0, j0 + kPBufs, ...
      const int j0 = (side - it0) & 1;
      float g = 1.f;               // e4m3: values' scales go times g = 2^-d
      bool careful = false;        // as tree_tiles.cuh has it
      all_sync();  // the columns' numbers are there
      for (int j = j0; j < n; j += C::kPBufs) {
        const int it = it0 + j, buf = p_buf(it);
        const uint32_t ts = tm_s + N * (it & 1) + lanes;
        const int key = (tile0 + j) * kTile + t;
        const bool edge = (tile0 + j + 1) * kTile > vis_min;
        // Which of this warp's 32 keys the columns' rows see: lane l has column l's bits.
        uint32_t win = 0u;
        if (edge) {
          const int key_w = key - lane, left = vis_max - key_w;  // the warp's first key, keys from there on
          const uint32_t valid = left >= 32 ? 0xFFFFFFFFu : left > 0 ? (1u << left) - 1u : 0u;
          if (lane < 16 && valid) win = tree_bits(a, sh.row[c0 + lane], key_w - prefix) & valid;
        }
        uint32_t hidden = 0;  // columns whose rows do not see this thread's key (which may leave -inf to those that do)
        if (edge) {
#pragma unroll
          for (int e = 0; e < 16; ++e) hidden |= (~(__shfl_sync(0xFFFFFFFFu, win, e) >> lane) & 1u) << e;
        }
        hold(sh.s_ready[it & 1], it >> 1);
        tc_fence_after();
        float sk = 1.f, sv = 1.f, limit = kMost;
        if constexpr (kE4m3) {
          hold(sh.scales_full[it % C::kScaleSlots], it / C::kScaleSlots);
          const float* scales = reinterpret_cast<const float*>(smem + C::kScalesAt + (it % C::kScaleSlots) * C::kScaleBytes);
          const bool valid = key < vis_max;
          sk = valid ? scales[t] : 0.f;
          sv = valid ? scales[kTile + t] : 0.f;
          if (j == j0) {
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
            if (t < 16) sh.d[side * N + c0 + t] = static_cast<float>(shift);
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
          tmem_ld_x16(ts + c0, s);
          tmem_wait_x16(s);
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const ulonglong2 ref = *reinterpret_cast<const ulonglong2*>(&neg_a[c0 + e]);
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
        if (mine && !careful) {
          fetch();
#pragma unroll
          for (int e = 0; e < 16; e += 2) top = max3(top, x[e], x[e + 1]);
        }
        if (!careful && group_any<128>(group_bar, top > limit)) {
          // ------------------------------------------ a moves: the columns' maxima across keys
          uint32_t s[16];
          tmem_ld_x16(ts + c0, s);
          tmem_wait_x16(s);
          float most = -INFINITY;  // lane e: column e's
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float z = __uint_as_float(s[e]) * (kE4m3 ? sh.f[c0 + e] : a.scale_log2) * sk - limit;
            if ((hidden >> e) & 1u) z = -INFINITY;
            const float largest = warp_max(z);
            if ((lane & 15) == e) most = largest;
          }
          if (lane < 16 && most == most) atomicMax(&mosts[c0 + lane], ordered(most));
          if (most > -INFINITY && fabsf(most) >= kBig) sh.careful[wg] = 1;
          group_sync(group_bar);
          __syncwarp();
          careful = *static_cast<volatile int*>(&sh.careful[wg]) != 0;
          if (j >= C::kPBufs && !careful) {
            hold(sh.p_free[buf], p_use(it) - 1);
            tc_fence_after();
            float shrink[16];
            bool moved = false;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float was = -neg_a[c0 + e], now = from_ordered(mosts[c0 + e]);
              shrink[e] = now > was ? fast_exp2(was - (now + kRoom)) : 1.f;
              moved |= now > was;
            }
            if (moved) {  // the same for all threads
#pragma unroll
              for (int e = 0; e < 8; ++e) l[e] = mul2(l[e], pair(shrink[2 * e], shrink[2 * e + 1]));
#pragma unroll 1
              for (int h = 0; h < C::kPCols; h += N) {
                uint32_t o[16];
                const uint32_t to = tm_o + C::kPCols * buf + lanes + h + c0;
                tmem_ld_x16(to, o);
                tmem_wait_x16(o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * shrink[e]);
                tmem_st_x16(to, o);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
              }
            }
          }
          group_sync(group_bar);
          if (t < 16) {
            const float now = from_ordered(mosts[c0 + t]);
            if (!careful && now > -neg_a[c0 + t]) neg_a[c0 + t] = -(now + kRoom);
            mosts[c0 + t] = ordered(-INFINITY);
          }
          group_sync(group_bar);
          __syncwarp();
          if (!careful) fetch();
        }
        if (careful) {
          if (p_use(it) > 0) hold(sh.p_free[buf], p_use(it) - 1);
          tc_fence_after();
          const int at = side * N + c0;
          const float scale_v = kE4m3 && key < vis_max
                                    ? reinterpret_cast<const float*>(smem + C::kScalesAt + (it % C::kScaleSlots) * C::kScaleBytes)[kTile + t]
                                    : 0.f;
          careful_step<kE4m3, N>(CarefulColumns{sh.neg_a + at, sh.d + (kE4m3 ? at : 0), sh.most + at, sh.shrink_l + at,
                                                sh.shrink_o + at, sh.f + (kE4m3 ? c0 : 0)},
                                 group_bar, ts + c0, tm_o + C::kPCols * buf + lanes + c0, j >= C::kPBufs, hidden,
                                 a.scale_log2, sk, scale_v, smem + C::kPAt + C::kPBytes * buf + t * 128, c0, l);
        }
        tc_fence_before();
        warp_arrive(sh.s_free[it & 1]);
        // ------------------------------------------ weights
        if (p_use(it) > 0) hold(sh.p_free[buf], p_use(it) - 1);
        if (mine && !careful) {
          uint8_t* const prow = smem + C::kPAt + C::kPBytes * buf + t * 128;
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
        // ------------------------------------------ this side's values of the tile
        {
          const int vs = it % C::kVStages;
          uint8_t* const stage = smem + C::kVAt + vs * C::kVBytes;
          const int left = vis_max - (tile0 + j) * kTile;
          if constexpr (kE4m3) {
            // Codes to fp16.  A warp has eight rows at a time, four lanes a row: codes 16 c .. and 64 +
            // 16 c .. of it (c = lane & 3).  Neighbouring groups of four take rows r and r ^ 5, so that neither
            // the reads nor the writes meet in a bank.
            hold(sh.v_full[vs], it / C::kVStages);
            constexpr int kPer = DP / 64, kWarps = 4 * C::kSharers, kRounds = kTile / 8 / kWarps;
            const int c = lane & 3, pair_row = (lane >> 3) & 3, row8 = (lane & 4) ? pair_row ^ 5 : pair_row;
            uint4 u[kRounds][kPer];
#pragma unroll
            for (int k = 0; k < kRounds; ++k)
#pragma unroll
              for (int q = 0; q < kPer; ++q) {
                const int r = 8 * (warp % kWarps + kWarps * k) + row8;
                u[k][q] = *reinterpret_cast<const uint4*>(stage + C::kRawAt + r * DP +
                                                          (((c + 4 * q) ^ (DP == 128 ? row8 : 0)) << 4));
                if (r >= left) u[k][q] = make_uint4(0, 0, 0, 0);  // not this sequence's
              }
            __syncwarp();  // the rows' codes are read: their place may be written
#pragma unroll
            for (int k = 0; k < kRounds; ++k)
#pragma unroll
              for (int q = 0; q < kPer; ++q) {
                const uint4& v = u[k][q];
                uint8_t* row = stage + q * kBlock + (8 * (warp % kWarps + kWarps * k) + row8) * 128;
                *reinterpret_cast<uint4*>(row + (((2 * c) ^ row8) << 4)) =
                    make_uint4(e4m3x2_f16x2(v.x, 0), e4m3x2_f16x2(v.x, 1), e4m3x2_f16x2(v.y, 0), e4m3x2_f16x2(v.y, 1));
                *reinterpret_cast<uint4*>(row + (((2 * c + 1) ^ row8) << 4)) =
                    make_uint4(e4m3x2_f16x2(v.z, 0), e4m3x2_f16x2(v.z, 1), e4m3x2_f16x2(v.w, 0), e4m3x2_f16x2(v.w, 1));
              }
          } else {
            hold(sh.v_full[vs], it / C::kVStages);
            if (edge) {  // values that not every row sees: 0 * NaN would reach rows that must not see it
              const int pc = lane & 7, r_of = 4 * (warp % (4 * C::kSharers)) + (lane >> 3);
#pragma unroll 1
              for (int h = 0; h < C::kHalves; ++h)
#pragma unroll 2
                for (int r = r_of; r < kTile; r += 16 * C::kSharers) {
                  uint4* const at = reinterpret_cast<uint4*>(stage + h * kBlock + r * 128 + pc * 16);
                  const int of = (tile0 + j) * kTile + r;
                  if (r >= left) {
                    *at = make_uint4(0, 0, 0, 0);
                  } else if (of >= vis_min) {
                    auto finite = [](uint32_t u) -> uint32_t {
                      if ((u & 0x7F80u) == 0x7F80u) u &= 0xFFFF0000u;
                      if ((u & 0x7F800000u) == 0x7F800000u) u &= 0x0000FFFFu;
                      return u;
                    };
                    const uint4 x = *at, y = make_uint4(finite(x.x), finite(x.y), finite(x.z), finite(x.w));
                    if (x.x != y.x || x.y != y.y || x.z != y.z || x.w != y.w) {
                      *at = y;
                      sh.any_bad[part & 7] = 1;
                    }
                  }
                }
            }
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        warp_arrive(sh.p_ready[buf]);
      }
      // ---------------------------------------------- out
      const int first_of = it0;
      it0 += n;
      // the last tile of this side, if it had any, is in O
      if (n > j0) {
        const int last = first_of + j0 + (n - 1 - j0) / C::kPBufs * C::kPBufs;
        hold(sh.p_free[p_buf(last)], p_use(last));
      }
      tc_fence_after();
      tc_fence_before();
      all_sync();  // nothing reads P any more, and O is whole
      tc_fence_after();
      if (mine) {
        float v[16];
#pragma unroll
        for (int e = 0; e < 8; ++e) unpair(l[e], v[2 * e], v[2 * e + 1]);
        const float sum = sum16(v);
        if (!(lane & 1)) sums[(4 * side + quad) * N + c0 + (lane >> 1)] = sum;
      }
      const bool bad_page = n > 0 && sh.bad_page[part & 7], some_bad = !kE4m3 && n > 0 && sh.any_bad[part & 7];
      if (threadIdx.x == 0 && bad_page) paged_report(a.status);
      all_sync();
      float* const part_to = p.whole ? nullptr : part_at<DP, N>(ta.parts, blockIdx.x, tile0 == 0);
      const int ch = 32 * quad + lane;
      // is there anything in the O of P's buffers?
      const bool have0 = n > ((0 - first_of) & 1), have1 = n > ((1 - first_of) & 1);
      if (threadIdx.x < cols) {  // a thread settles a column: the weights of both accumulators, the sum and the place
        const int c = threadIdx.x;
        auto sum_of = [&](int of) {
          const float* x = sums + 4 * of * N + c;
          return (x[0] + x[N]) + (x[2 * N] + x[3 * N]);
        };
        const float a0 = -sh.neg_a[c], a1 = -sh.neg_a[N + c], top = fmaxf(a0, a1);
        float f0 = fast_exp2(a0 - top), f1 = fast_exp2(a1 - top);  // nothing seen: sums and O are 0, or NaN to stay
        float total = f0 * sum_of(0) + f1 * sum_of(1), unit = 0.f;  // 2^unit: O's unit beside that of 2^top
        if constexpr (kE4m3) {
          const float d0 = fmaxf((a0 - top) + sh.d[c], kLeastUnit), d1 = fmaxf((a1 - top) + sh.d[N + c], kLeastUnit);
          unit = fmaxf(d0, d1);
          f0 = fast_exp2(d0 - unit);
          f1 = fast_exp2(d1 - unit);
        }
        if (bad_page || !alive) total = __uint_as_float(0x7FC00000u);
        float inv = total == 0.f ? 0.f : 1.f / total;
        int64_t place = 3 * N + c * DP;
        if (part_to != nullptr) {
          part_to[c] = top;
          part_to[N + c] = total;
          part_to[2 * N + c] = unit;
          inv = 1.f;
        } else {
          const int64_t row = static_cast<int64_t>(p.rb) * N + c, token = sh.row[c] - p.row0;
          place = static_cast<int64_t>(sh.row[c]) * a.out_ld + (static_cast<int64_t>(p.hk) * a.group + row - token * a.group) * a.d;
        }
        places[c] = place;
        if constexpr (kE4m3) halves[c] = fast_exp2(0.5f * unit);
        weights[c] = f0 * inv;
        weights[N + c] = f1 * inv;
      }
      all_sync();
      if (side == 0 && mine) {
        float y[16] = {};
#pragma unroll
        for (int b = 0; b < C::kPBufs; ++b)
          if (b ? have1 : have0) {
            constexpr int kParts = C::kPCols / N;
            uint32_t o[kParts][16];
#pragma unroll
            for (int h = 0; h < kParts; ++h) tmem_ld_x16(tm_o + lanes + C::kPCols * b + N * h + c0, o[h]);
#pragma unroll
            for (int h = 0; h < kParts; ++h) tmem_wait_x16(o[h]);
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              const float4 f = *reinterpret_cast<const float4*>(&weights[N * b + c0 + e]);
              const float w4[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                float v = __uint_as_float(o[0][e + k]);
                if constexpr (kParts > 1) v += __uint_as_float(o[kParts - 1][e + k]);
                y[e + k] = fmaf(v, w4[k], y[e + k]);
              }
            }
          }
        if (some_bad) {
          PagedSeq seq;
          seq.row0 = p.row0;
          seq.n = p.seq_n;
          seq.length = vis_max;
          seq.bad = false;
#pragma unroll 1
          for (int e = 0; e < 16; ++e) {
            const bool bad = c0 + e < rows && ch < a.d &&
                             tree_sees_bad<kE4m3>(a, seq, a.table + p.table, p.hk, sh.row[c0 + e], ch);
#pragma unroll
            for (int k = 0; k < 16; ++k)
              if (bad && k == e) y[k] = __uint_as_float(0x7FC00000u);
          }
        }
        if (part_to != nullptr) {
          if (ch < DP) {
            float* const to = part_to + 3 * N + c0 * DP + ch;
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (c0 + e < rows) to[e * DP] = y[e];
          }
        } else if (ch < a.d) {
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
      if (threadIdx.x == 0) sh.bad_page[part & 7] = sh.any_bad[part & 7] = 0;
      warp_arrive(sh.part_empty[part & 3]);
    }
  }
  __syncthreads();
  if (warp == kMma) {
    tc_fence_after();
    tmem_dealloc(sh.tmem, C::kTmemCols);
  }
}

// Joins the parts of the units that more than one block has: block (c, y) rows kJoinRows y .. of
// the unit that the boundary between blocks c and c + 1 is the first to cut, a warp to a row.
constexpr int kJoinRows = 8, kJoinThreads = 32 * kJoinRows;
template <int DP, int N>
__global__ void __launch_bounds__(kJoinThreads) join_parts_kernel(const __grid_constant__ TreeArgs ta, const int blocks) {
  const PagedArgs& a = ta.p;
  const int c = static_cast<int>(blockIdx.x) + 1;
  __shared__ int64_t scratch[kPlanScratch];
  Plan w = make_plan<N, kJoinThreads>(a, c, blocks, scratch);
  Part p;
  // The first part that block c begins, if the boundary cuts its unit and is the first to do so.
  int64_t at = 0;
  const bool some = next_part<N>(a, w, p, &at) && p.tile0 > 0 && at - w.share <= kUnitCost && !p.bad;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the parts are there
  if (!some) return;
  const int others = static_cast<int>((kUnitCost + p.steps - at + w.share - 1) / w.share);  // blocks c, c + 1, ...
  const int rows = static_cast<int>(min(static_cast<int64_t>(p.seq_n) * a.group - static_cast<int64_t>(p.rb) * N,
                                        static_cast<int64_t>(N)));
  const int r = blockIdx.y * kJoinRows + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (r >= rows) return;
  auto part = [&](int i) -> const float* {
    return i == 0 ? part_at<DP, N>(ta.parts, c - 1, true) : part_at<DP, N>(ta.parts, c + i - 1, false);
  };
  // Sums and outputs each relative to the largest of theirs so far: 2^top, and 2^(top + unit).
  constexpr int kPer = DP / 32;  // channels of a lane
  float top = -kUnset, unit = kLeastUnit, sum = 0.f, y[kPer] = {};
#pragma unroll 4
  for (int i = 0; i <= others; ++i) {
    const float* x = part(i);
    const float ref = x[r], l = x[N + r];
    float o[kPer];
    if constexpr (kPer == 4) {
      const float4 v = *reinterpret_cast<const float4*>(x + 3 * N + r * DP + 4 * lane);
      o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w;
    } else {
      const float2 v = *reinterpret_cast<const float2*>(x + 3 * N + r * DP + 2 * lane);
      o[0] = v.x; o[1] = v.y;
    }
    // a part whose keys the row does not see has the least reference and l = 0 (or NaN, which has to stay)
    if (ref > top) {
      sum *= fast_exp2(top - ref);
      unit = fmaxf(unit + (top - ref), kLeastUnit);
      top = ref;
    }
    const float own = fmaxf((ref - top) + x[2 * N + r], kLeastUnit);
    float back = 1.f;
    if (own > unit) {
      back = fast_exp2(unit - own);
      unit = own;
    }
    const float f = fast_exp2(own - unit);
    sum = fmaf(fast_exp2(ref - top), l, sum);
#pragma unroll
    for (int k = 0; k < kPer; ++k) y[k] = fmaf(f, o[k], back * y[k]);
  }
  const uint32_t row = static_cast<uint32_t>(p.rb) * N + r, token = row_token(row, a.group);
  const float inv = sum == 0.f ? 0.f : 1.f / sum, half = fast_exp2(0.5f * unit);
#pragma unroll
  for (int k = 0; k < kPer; ++k) y[k] = sum == 0.f && y[k] == y[k] ? 0.f : y[k] * inv * half * half;
  if (kPer * lane < a.d) {
    uint16_t* const to = a.out + (p.row0 + token) * a.out_ld +
                         (static_cast<int64_t>(p.hk) * a.group + row - token * a.group) * a.d + kPer * lane;
    if constexpr (kPer == 4)
      *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
    else
      *reinterpret_cast<uint32_t*>(to) = pack_bf16(y[0], y[1]);
  }
}

// Whether blocks take shares of all steps, were every sequence as long as its table allows.  Where every
// unit can have a block: from the length on where halves of units and their join cost less than the longest
// unit, which is the later the more blocks have one.  (bf16, 16 heads of 128 channels, contexts all as long and
// ragged, us whole and shared: 2 sequences of 1536 17.5, 17.2 and 18.3, 18.0, of 4096 33.5, 32.6 and 22.3, 21.5;
// 8 of 2048 28.5, 21.1 and 35.6, 24.7, of 4096 47.1, 37.3 and 54.9, 38.1, of 6000 64.1, 50.4 and 72.3, 47.7.)
// Else where a block gets more than a few steps.
bool shares_steps(const PagedArgs& a, int n, int64_t* units) {
  const int64_t row_units = (static_cast<int64_t>(a.max_q) * a.group + n - 1) / n, sms = device_sm_count();
  *units = static_cast<int64_t>(a.B) * a.H_kv * row_units;
  const int64_t steps = ((static_cast<int64_t>(a.max_pages) << a.page_log2) + kTile - 1) / kTile;
  if (*units <= sms) return steps * sms > 8 * sms + 28 * *units;
  return *units * steps > 6 * sms;
}

// Lets the kernel have its shared memory, and checks that the launch brings the registers that the
// warps share out among themselves; once per device.
template <bool kE4m3, int DP, int N>
cudaError_t configure_tree() {
  using C = TreeCfg<kE4m3, DP, N>;
  static std::atomic<bool> done[64] = {};
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
  if (dev < 64 && done[dev].load(std::memory_order_acquire)) return cudaSuccess;
  cudaFuncAttributes attr;
  if (cudaError_t e = cudaFuncGetAttributes(&attr, tree_attention_kernel<kE4m3, DP, N>); e != cudaSuccess) return e;
  if (attr.numRegs / 8 * 8 * C::kThreads < C::kSoftmax * C::kSoftmaxRegs + (C::kThreads - C::kSoftmax) * C::kOtherRegs)
    return cudaErrorInvalidConfiguration;
  cudaError_t e = cudaFuncSetAttribute(tree_attention_kernel<kE4m3, DP, N>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  if (e == cudaSuccess && dev < 64) done[dev].store(true, std::memory_order_release);
  return e;
}

template <bool kE4m3, int DP, int N>
cudaError_t launch_tree(const PagedArgs& a, float* workspace, cudaStream_t stream) {
  using C = TreeCfg<kE4m3, DP, N>;
  CUtensorMap mk, mv;
  const int box_rows = 1 << a.page_log2;
  if (!make_page_map(&mk, a.k, a, 128, box_rows, 1) ||
      !make_page_map(&mv, a.v, a, kE4m3 ? DP : 128, box_rows, 1))
    return cudaErrorInvalidValue;
  constexpr auto kKernel = tree_attention_kernel<kE4m3, DP, N>;
  if (cudaError_t e = configure_tree<kE4m3, DP, N>(); e != cudaSuccess) return e;
  TreeArgs t{};
  t.p = a;
  int64_t units;
  const bool shared = shares_steps(a, N, &units);
  t.parts = shared ? workspace : nullptr;
  t.row_units = static_cast<int>((static_cast<int64_t>(a.max_q) * a.group + N - 1) / N);
  const int64_t grid = shared ? device_sm_count() : units;
  if (grid > 0x7FFFFFFFll) return cudaErrorInvalidConfiguration;
  kKernel<<<static_cast<unsigned>(grid), C::kThreads, C::kSmem, stream>>>(mk, mv, t);
  if (cudaError_t e = cudaGetLastError(); e != cudaSuccess || !shared) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid - 1), N / kJoinRows);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, join_parts_kernel<DP, N>, t, static_cast<int>(grid));
}

}  // namespace

// Whether a call comes here: up to kTreeRows rows, and twice as many where every block of rows can have an SM and is
// a few steps.  (64 rows of 64 heads over 1024 tokens 14.9 us, in tree_attention_short.cu 17.0, in tiles of 128 rows 21.2.)
bool tree_has_room(const PagedArgs& a) {
  const int64_t rows = static_cast<int64_t>(a.max_q) * a.group;
  const int64_t steps = ((static_cast<int64_t>(a.max_pages) << a.page_log2) + kTile - 1) / kTile;
  return rows <= kTreeRows || (rows <= 2 * kTreeRows && steps > 1 && steps <= 8 &&
                               2 * static_cast<int64_t>(a.B) * a.H_kv <= device_sm_count());
}

size_t tree_attention_workspace(const PagedArgs& a) {
  const int64_t most_rows = static_cast<int64_t>(a.max_q) * a.group;
  int64_t units;
  if (most_rows <= kFewRows || most_rows > kTreeRows || tree_is_short(a) || !shares_steps(a, kTreeRows, &units)) return 0;
  return static_cast<size_t>(device_sm_count()) * 2 * kTreeRows * ((a.d <= 64 ? 64 : 128) + 3) * sizeof(float);
}

cudaError_t launch_tree_attention(const PagedArgs& a, void* workspace, cudaStream_t stream) {
  float* ws = static_cast<float*>(workspace);
  const bool e4m3 = a.k_scale != nullptr;
  if (a.d <= 64)
    return e4m3 ? launch_tree<true, 64, kTreeRows>(a, ws, stream) : launch_tree<false, 64, kTreeRows>(a, ws, stream);
  return e4m3 ? launch_tree<true, 128, kTreeRows>(a, ws, stream) : launch_tree<false, 128, kTreeRows>(a, ws, stream);
}

}  // namespace dwa
