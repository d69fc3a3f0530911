// paged_attention_mma.cu — attention of a chunk of new tokens over the paged
// cache on tcgen05: prompts in pieces, long drafts, anything with many rows per
// key/value head.
//
// A block takes 256 rows of one key/value head (a row is one (new token, query
// head), token-major) as two tiles of 128, and goes once over the keys they may
// see (or its share of them), 128 at a time:
//
//   S   = Q_i K^T          tcgen05, Q and K in shared memory, S in TMEM
//   P_i = exp2(S - m)      one thread per row: running maximum, sum, P_i to TMEM
//   O_i += P_i V           tcgen05, P_i from TMEM, V in shared memory, O_i in TMEM
//
// TMEM is full: one S of 128 columns that the tiles use in turn, two P of 64, two O
// of 128.  A row's thread takes its 128 scores into registers at once, so that S is
// free for the other tile's product while it works, and the next S is there when it
// is done: the threads never wait for a product, only the tensor pipe for P.  (With
// an S per tile that P overwrote, each step was a chain of product, exponentials,
// product: 2.9 us per 2 x 128 rows x 128 keys of 128 channels instead of 2.2.)
//
// Per step the products take 2048 cycles of the tensor pipe (8192 FLOP a cycle) and the
// exponentials 32768 / 16 = 2048 of the special-function units.  What bounds it is each
// row's own chain: S out of TMEM 200 cycles, the maximum 450, 128 exponentials with their
// sums and packing 1600 (1024 at the units' rate; a warp alone with these registers takes
// 1400), P into TMEM and the next S 300 to 500.  Measured 3000 cycles a step, e4m3 3900,
// where the conversion shares the issue slots: 4736 rows over 16384 keys, 32 heads of 128,
// 1.0 to 1.12 ms (bf16, 0.97 to 1.08 PFLOP/s, the power limit's clock deciding) and 1.17 to
// 1.3 ms.  Not faster: a polynomial for a quarter of the exponentials (1065 us, 1031 without
// then), S before the other tile's product (3300 cycles), a warp each for S and O, eight
// converting warps.  What can be is done in pairs (f32x2) and triples (max).  m only moves
// when a row's maximum grew by more than 2^kSlack (the result does not depend on m; P
// stays below 2^kSlack), so O is hardly ever rescaled, and then by the row's own thread.
//
// P goes to its product in 16 bits: over a bf16 cache, whose values are bf16 and want P to be
// too, with 8 bits (2 x 2048 rows over 4096 to 8192 keys: relative error 0.0023 against 64 bits,
// 0.0017 with f32 probabilities, which is the result's own rounding).  A second part of P would
// have no place: TMEM and shared memory are full, and its product would take the
// tensor pipe half as long again.
//
// A block costs 9 to 11 thousand cycles before its first scores (launch, the sequence's numbers,
// Q's 64 KB from all SMs at once) and 4 after its last, a split one 8 to 12.
//
// Warps 0-3 and 4-7: the rows of tile 0 and 1.  Warp 8: issues every tcgen05.mma.
// Warp 9: TMA, straight from the pages into the swizzled operand tiles.  bf16
// caches: warps 10-11 look over the values of tiles that end behind what every row
// sees, since 0 * NaN would reach rows that must not see it.  e4m3 caches: warps
// 12-15 turn codes into fp16 operand tiles (code times scale, over a power of two near
// the first tile's scales, rounded to 2^-11), and Q is scaled per row by a power of two into
// fp16, exactly.  (With the keys' scales multiplied into the scores instead, every
// row's thread read 128 of them per step: 1499 us instead of 1333 for 4736 rows over
// 16384 keys, 32 heads.)  One power of two for all tokens would take the bits of those whose
// scales are far smaller, for the sake of one that a row may not even see.  So from the step on
// where scales leave a range of 2^12, operands keep their scales' mantissas only, and the row's
// thread multiplies scores and weights by the powers of two after all, in units of its own: 2048
// rows over 8192 keys, 32 heads, 280 us, and 525 to 580 where that starts at once.  (The check
// and the second form's code cost the first 2 to 4 %.)
//
// Where there are few units of 256 rows, a cluster of blocks shares the keys of one
// and joins its parts through distributed shared memory, in a fixed order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <mutex>
#include <type_traits>

#include "dwa_internal.h"
#include "f32x2.cuh"
#include "paged_attention.cuh"
#include "sm100_ptx.cuh"

namespace dwa {

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

bool make_page_map(CUtensorMap* map, const void* ptr, const PagedArgs& a, int row_bytes, int box_rows,
                   int box_halves) {
  auto encode = tensor_map_encoder();
  if (!encode) return false;
  const bool e4m3 = a.k_scale != nullptr;
  const uint64_t es = e4m3 ? 1 : 2;
  const uint64_t page = 1ull << a.page_log2;
  const cuuint64_t halves = static_cast<cuuint64_t>(box_halves);
  cuuint64_t dims[5] = {static_cast<cuuint64_t>(a.d) / halves, page, halves,
                        static_cast<cuuint64_t>(a.H_kv), static_cast<cuuint64_t>(a.n_pages)};
  cuuint64_t strides[4] = {a.d * es, a.d * es / halves, page * a.d * es, a.ld_page * es};
  cuuint32_t box[5] = {static_cast<cuuint32_t>(row_bytes / es), static_cast<cuuint32_t>(box_rows),
                       static_cast<cuuint32_t>(box_halves), 1, 1};
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return encode(map, e4m3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
                const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                row_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace {

constexpr int kTile = 128;     // rows per tile, keys per step
constexpr int kMaxChannels = 128;
constexpr int kMaxSplit = 8;
constexpr float kSlack = 4.f;  // log2 of how far P may grow before m follows
// e4m3 caches: P in fp16 times 2^11 (with kSlack still below 65504), keys and values
// times f, 8 over a power of two above the first tile's scales.  f may lie between 2^-5, where
// the least code, 2^-9, still makes fp16's least normal number, and 2^7 (448 f below 65504).
constexpr float kPBits = 11.f, kCodeScale = 8.f;
constexpr int kScalesBelow = 8, kScalesAbove = 4;  // the scales' range around that power, in log2

template <bool kE4m3, int DP>
struct MmaCfg {
  static constexpr int kThreads = kE4m3 ? 512 : 384;
  static constexpr int kSoftmaxRegs = kE4m3 ? 176 : 208;
  static constexpr int kOtherRegs = kE4m3 ? 80 : 88;
  static constexpr int kHalves = DP / 64;               // 128-byte wide column blocks
  static constexpr int kBlockBytes = kTile * 128;       // one of them: 16 KB
  static constexpr int kTileBytes = kHalves * kBlockBytes;
  static constexpr int kStages = 5;                     // operand tiles (K and V in turn)
  // Codes arrive in the stage that their fp16 values will take: at 128 channels in the
  // second column block, where row r's codes lie in row r's place; at 64 behind it.
  static constexpr int kRawAt = DP == 128 ? kBlockBytes : kTileBytes;
  static constexpr int kStageBytes = kTileBytes + (kE4m3 && DP == 64 ? kTile * DP : 0);
  static constexpr int kSmem = 1024 + 2 * kTileBytes + kStages * kStageBytes;
  // at the end a split block's parts take Q's and the operands' place
  static constexpr int kPartMl = 2 * kTile * DP * 4;    // behind O
  static constexpr int kPartUnit = kPartMl + 2 * kTile * 8;  // e4m3
  static constexpr int kPartBytes = kPartUnit + (kE4m3 ? 2 * kTile * 4 : 0);
  static_assert(kPartBytes <= 2 * kTileBytes + kStages * kStageBytes, "parts fit");
};

template <bool kE4m3>
struct MmaShared {
  uint64_t full[5], ready[5], empty[5];
  uint64_t q_ready, s_ready[2], s_free, p_ready[2], p_free[2];
  uint32_t tmem;
  int abort;
  int bad_page;
  int any_bad;
  int first_bad[kE4m3 ? 1 : kMaxChannels];  // least key with a value that is not finite (e4m3: whole vectors)
  // e4m3 only: the powers of two that keys and values are divided by; the steps from which
  // each key or value is divided by its own scale's instead, the lesser of the two, and those
  // (as bf16) of three steps
  float k_ref, v_ref;
  int k_from, v_from, apart_from;
  alignas(16) uint16_t k_pow[3][kE4m3 ? kTile : 8], v_pow[3][kE4m3 ? kTile : 8];
  // between the converting warps: the first tile's largest and least scales (keys', values'),
  // and which scales of two steps are out of range (keys' 1, values' 2)
  uint64_t scales_ready, refs_ready;
  uint32_t tops[2][4], lows[2][4], far[2][4];
};

// ---------------------------------------------------------------- tcgen05 pieces
// One lane of a converged warp.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
// The issuing warp stays converged, so that addresses and descriptors live in uniform
// registers; `one` is its elected lane.
// D[tmem] (+)= A[smem] B[smem]^T
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t add, uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(one)
      : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       uint32_t add, uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(add), "r"(one)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar, uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
      "r"(one)
      : "memory");
}
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}
// Multiplies 16 columns of this warp's lanes by `f` in place.
__device__ __forceinline__ void tmem_scale_x16(uint32_t taddr, float f) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * f);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// The powers of two of an even key and the next.
__device__ __forceinline__ void powers_at(const uint16_t* powers, int key, float& x, float& y) {
  const uint32_t w = reinterpret_cast<const uint32_t*>(powers)[key >> 1];
  x = __uint_as_float(w << 16);
  y = __uint_as_float(w & 0xFFFF0000u);
}

// A K-step of 16 keys of a value tile: channels along the rows of 128 bytes (MN-major,
// 128-byte swizzle), 8 keys per 1024-byte atom, the next 64 channels one column block on.
__device__ __forceinline__ uint64_t value_desc(uint32_t addr, uint32_t block_bytes) {
  uint64_t desc = 0;
  desc |= static_cast<uint64_t>((addr >> 4) & 0x3FFFu);
  desc |= static_cast<uint64_t>((block_bytes >> 4) & 0x3FFFu) << 16;  // LBO: 64 channels on
  desc |= static_cast<uint64_t>(1024u >> 4) << 32;                    // SBO: 8 keys on
  desc |= static_cast<uint64_t>(1u) << 46;
  desc |= static_cast<uint64_t>(2u) << 61;
  return desc;
}

__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

// Bounded waits of a whole converged warp, for one barrier or two.  All lanes ask the
// same and go by votes, so that they cannot part: the warp that issues the products
// keeps their descriptors in registers that all its lanes share.  Mostly the phase is
// over already, and a test is cheaper than a wait with a time limit.
__device__ __forceinline__ bool warp_wait2(uint32_t x, uint32_t parity_x, uint32_t y,
                                           uint32_t parity_y, int* status, volatile int* abort_flag) {
  constexpr uint32_t kAll = 0xFFFFFFFFu;
  if (__all_sync(kAll, mbar_test(x, parity_x) & mbar_test(y, parity_y))) return true;
  const uint64_t t0 = globaltimer_ns();
  while (true) {
    const bool x_done = __all_sync(kAll, mbar_try_wait(x, parity_x));
    const bool y_done = __all_sync(kAll, mbar_try_wait(y, parity_y));
    if (x_done && y_done) return true;
    if (__any_sync(kAll, *abort_flag != 0)) return false;
    if (__any_sync(kAll, globaltimer_ns() - t0 > kWaitLimitNs)) {
      if (status) atomicCAS(status, 0, kStatusTimeout);
      *abort_flag = 1;
      __syncwarp();
      return false;
    }
  }
}
__device__ __forceinline__ bool warp_wait1(uint32_t x, uint32_t parity, int* status,
                                           volatile int* abort_flag) {
  constexpr uint32_t kAll = 0xFFFFFFFFu;
  if (__all_sync(kAll, mbar_test(x, parity))) return true;
  const uint64_t t0 = globaltimer_ns();
  while (true) {
    if (__all_sync(kAll, mbar_try_wait(x, parity))) return true;
    if (__any_sync(kAll, *abort_flag != 0)) return false;
    if (__any_sync(kAll, globaltimer_ns() - t0 > kWaitLimitNs)) {
      if (status) atomicCAS(status, 0, kStatusTimeout);
      *abort_flag = 1;
      __syncwarp();
      return false;
    }
  }
}

// The start-address field; in a cluster an address has the block's rank above it.
__device__ __forceinline__ uint32_t desc_addr(uint32_t addr) { return (addr >> 4) & 0x3FFFu; }
__device__ __forceinline__ uint64_t desc64(uint32_t lo, uint32_t hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
  return r;
}

// Rows at equal distances as (new token, query head of the group), divided once.
struct RowWalk {
  uint32_t token, head;
  const uint32_t group, tokens, heads;  // of a step
  __device__ __forceinline__ RowWalk(uint32_t row, int group_, uint32_t by)
      : token(row_token(row, group_)), head(row - token * group_), group(group_),
        tokens(row_token(by, group_)), heads(by - tokens * group_) {}
  __device__ __forceinline__ void next() {
    token += tokens;
    head += heads;
    if (head >= group) {
      head -= group;
      ++token;
    }
  }
};
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
template <int kRegs>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}


template <bool kE4m3, int DP, bool kTree>
__global__ void __launch_bounds__(MmaCfg<kE4m3, DP>::kThreads, 1)
    paged_mma_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                     const __grid_constant__ PagedArgs a, const int row_units, const int cluster) {
  using C = MmaCfg<kE4m3, DP>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ MmaShared<kE4m3> sh;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t s_stage = base + 2 * C::kTileBytes;  // [Q tile 0][Q tile 1][stages]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ------------------------------------------------ the block's work
  const int split = static_cast<int>(blockIdx.x % cluster);
  const uint32_t unit = blockIdx.x / cluster;  // the grid has 32 bits
  // the units with the most keys first; where they are too many to rank, late rows first
  int* const costs = reinterpret_cast<int*>(smem);  // operands come later
  const int hk = static_cast<int>(unit % a.H_kv);
  int pair_of = static_cast<int>(unit / a.H_kv);  // (row unit, sequence)
  const int pairs = a.B * row_units;
  if (pairs > 1 && pairs <= kMostRanked)
    pair_of = ranked(pairs, pair_of, costs, costs + kMostRanked, [&](int i) {
      const PagedSeq s = paged_seq(a, i % a.B);
      const int64_t first = static_cast<int64_t>(row_units - 1 - i / a.B) * 2 * kTile;
      const int64_t end = min(first + 2 * kTile, static_cast<int64_t>(s.n) * a.group);
      return first >= end ? -1
             : kTree      ? s.length
                          : paged_visible(s, row_token(static_cast<uint32_t>(end - 1), a.group));
    });
  const int ru = row_units - 1 - pair_of / a.B, b = pair_of % a.B;
  const PagedSeq seq = paged_seq(a, b);
  if (seq.bad && hk == 0 && ru == 0 && split == 0 && threadIdx.x == 0) paged_report(a.status);
  const int64_t all_rows = static_cast<int64_t>(seq.n) * a.group;
  const int64_t r0 = static_cast<int64_t>(ru) * 2 * kTile;
  if (r0 >= all_rows) return;  // the whole cluster
  if (seq.bad) {
    const int64_t stride = static_cast<int64_t>(row_units) * 2 * kTile;
    for (int64_t r = r0; r < all_rows; r += stride)
      for (int i = split * C::kThreads + threadIdx.x; i < 2 * kTile * a.d; i += cluster * C::kThreads) {
        const int64_t row = r + i / a.d;
        if (row < all_rows)
          a.out[(seq.row0 + row / a.group) * a.out_ld +
                (static_cast<int64_t>(hk) * a.group + row % a.group) * a.d + i % a.d] = 0x7FC0u;
      }
    return;
  }
  const int64_t left = all_rows - r0;
  const int rows0 = static_cast<int>(min(left, static_cast<int64_t>(kTile)));
  const int rows1 = static_cast<int>(max(min(left - kTile, static_cast<int64_t>(kTile)), int64_t{0}));
  const uint32_t row_0 = static_cast<uint32_t>(r0);  // below 2^31: max_q bounds it
  const int prefix = tree_prefix(seq);
  auto visible = [&](uint32_t row) -> int {  // keys before the one behind the last that the row sees
    return kTree ? seq.length : paged_visible(seq, row_token(row, a.group));
  };
  const int vis_min = kTree ? max(prefix, 0) : visible(row_0);
  const int vis0 = visible(row_0 + rows0 - 1);
  const int vis1 = rows1 > 0 ? visible(row_0 + kTile + rows1 - 1) : 0;
  const int vis_max = max(vis0, vis1);
  // this block's share of the key tiles, and how far each row tile goes into it
  const int tiles_all = (vis_max + kTile - 1) / kTile;
  const int share = (tiles_all + cluster - 1) / cluster;
  const int first_tile = min(split * share, tiles_all);
  const int n_steps = min(share, tiles_all - first_tile);
  const int steps0 = min(max((vis0 + kTile - 1) / kTile - first_tile, 0), n_steps);
  const int steps1 = min(max((vis1 + kTile - 1) / kTile - first_tile, 0), n_steps);

  // ------------------------------------------------ Q's rows, on their way
  constexpr int kQChunks = DP / 8;  // of 16 bytes per row; a row's lanes are neighbours
  constexpr int kQRowsAtOnce = 256 / kQChunks, kQRounds = 2 * kTile / kQRowsAtOnce;
  const int q_chunk = threadIdx.x % kQChunks, q_first = threadIdx.x / kQChunks;
  uint4 q_held[kQRounds];
  if (warp < 8) {
    const uint16_t* src = a.q + static_cast<int64_t>(hk) * a.group * a.d + 8 * q_chunk;
    RowWalk at(row_0 + q_first, a.group, kQRowsAtOnce);
#pragma unroll
    for (int k = 0; k < kQRounds; ++k, at.next()) {
      q_held[k] = make_uint4(0, 0, 0, 0);
      if (q_first + k * kQRowsAtOnce < rows0 + rows1 && 8 * q_chunk < a.d)
        q_held[k] = __ldg(reinterpret_cast<const uint4*>(src + (seq.row0 + at.token) * a.q_ld + at.head * a.d));
    }
  }

  // ------------------------------------------------ set-up
  auto bar = [&](const uint64_t& x) { return smem_u32(&x); };
  const int n_items = 2 * n_steps;  // operand tiles: K V K V ...
  const int32_t* table = a.table + static_cast<int64_t>(b) * a.ld_table;
  // TMA, straight from the pages: a page to a lane
  auto bring = [&](int it) {
    const int page_size = 1 << a.page_log2;
    const int key0 = (first_tile + (it >> 1)) * kTile, st = it % C::kStages;
    const int pages = min(kTile >> a.page_log2, (vis_max - key0 + page_size - 1) >> a.page_log2);
    int page = 0;
    if (lane < pages) {
      page = __ldg(table + (key0 >> a.page_log2) + lane);
      if (page < 0 || page >= a.n_pages) {
        sh.bad_page = 1;  // read page 0 in its place; the rows become NaN
        page = 0;
      }
    }
    const uint32_t full = bar(sh.full[st]);
    if (lane == 0)
      mbar_arrive_expect_tx(full, static_cast<uint32_t>(pages * page_size) * (kE4m3 ? DP : 128 * C::kHalves));
    __syncwarp();
    if (lane < pages) {
      const CUtensorMap* map = (it & 1) ? &map_v : &map_k;
      const uint32_t dst = s_stage + st * C::kStageBytes;
      if constexpr (kE4m3) {
        tma_load_page(dst + C::kRawAt + lane * page_size * DP, map, full, 0, 0, 0, hk, page);
      } else {
#pragma unroll
        for (int h = 0; h < C::kHalves; ++h)
          tma_load_page(dst + h * C::kBlockBytes + lane * page_size * 128, map, full, 64 * h, 0, 0, hk, page);
      }
    }
  };
  if (warp == 9) {
    if (lane == 0) {
      for (int i = 0; i < C::kStages; ++i) {
        mbar_init(bar(sh.full[i]), 1);
        mbar_init(bar(sh.ready[i]), kE4m3 ? 4 : 2);
        mbar_init(bar(sh.empty[i]), 1);
      }
      mbar_init(bar(sh.s_free), 4);
      mbar_init(bar(sh.scales_ready), 4);
      mbar_init(bar(sh.refs_ready), 1);
      mbar_init(bar(sh.q_ready), 8);
      for (int i = 0; i < 2; ++i) {
        mbar_init(bar(sh.s_ready[i]), 1);
        mbar_init(bar(sh.p_ready[i]), 4);
        mbar_init(bar(sh.p_free[i]), 1);
      }
      sh.abort = 0;
      sh.bad_page = 0;
      sh.any_bad = 0;
      fence_mbar_init();
    }
    __syncwarp();
    for (int it = 0; it < min(C::kStages, n_items); ++it) bring(it);  // no one to wait for
  }
  constexpr int kBads = kE4m3 ? 1 : kMaxChannels;
  if (warp == 10)
    for (int i = lane; i < kBads; i += 32) sh.first_bad[i] = 0x7FFFFFFF;
  if (warp == 8) {
    tmem_alloc(smem_u32(&sh.tmem), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm_s = sh.tmem, tm_p = sh.tmem + 128, tm_o = sh.tmem + 256;  // + 64 i, + 128 i
  int* const status = a.status;
  volatile int* const abort_flag = &sh.abort;
  // a bounded wait of the whole warp, which goes on or gives up together
  auto warp_wait = [&](const uint64_t& x, int phase) -> bool {
    return warp_wait1(bar(x), phase & 1, status, abort_flag);
  };
  // one arrival per warp, after every lane's accesses
  auto warp_arrive = [&](const uint64_t& x) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(x));
  };

  if (warp >= 8) {
    regs_dec<C::kOtherRegs>();
    if (warp == 9) {
      // ---------------------------------------------- TMA
      int issued = min(C::kStages, n_items);
      for (int it = issued; it < n_items; ++it) {
        if (!warp_wait(sh.empty[it % C::kStages], it / C::kStages - 1)) break;
        bring(it);
        issued = it + 1;
      }
      // after an abort nobody else waits for the copies in flight
      if (*abort_flag) {
        for (int it = max(0, issued - C::kStages); it < issued; ++it)
          mbar_wait(bar(sh.full[it % C::kStages]), (it / C::kStages) & 1, status, nullptr);
      }
    } else if (warp == 8) {
      // ---------------------------------------------- tcgen05.mma
      constexpr uint32_t kFormat = kE4m3 ? 0u : (1u << 7) | (1u << 10);  // fp16 or bf16 operands
      const uint32_t idesc_s = (1u << 4) | kFormat | (kTile / 8 << 17) | (kTile / 16 << 24);
      const uint32_t idesc_o = (1u << 4) | kFormat | (1u << 16) |
                               (static_cast<uint32_t>(a.d / 8) << 17) | (kTile / 16 << 24);
      const int k_steps = a.d / 16;
      const bool full_d = a.d == DP;
      const uint32_t one = elect_one();
      int used = 0;  // products that went through S
      auto wait2 = [&](uint32_t x, int phase_x, uint32_t y, int phase_y) -> bool {
        const bool ok = warp_wait2(x, phase_x & 1, y, phase_y & 1, status, abort_flag);
        tc_fence_after();
        return ok;
      };
      // an operand tile is in shared memory: bf16 keys come straight from the TMA,
      // everything else through other warps
      const uint32_t full0 = bar(sh.full[0]), ready0 = bar(sh.ready[0]);
      auto item = [&](int it) -> uint32_t {
        return (!kE4m3 && !(it & 1) ? full0 : ready0) + 8 * (it % C::kStages);
      };
      // Only a descriptor's start address changes: its low word by constants, so that the
      // one issuing lane spends a few instructions per product (a loop that built
      // descriptors took 150 cycles for each product of 64).
      const uint32_t k_hi = static_cast<uint32_t>(sw128_kmajor_desc(0) >> 32);
      const uint32_t k_lo = static_cast<uint32_t>(sw128_kmajor_desc(0));
      const uint32_t v_hi = static_cast<uint32_t>(value_desc(0, C::kBlockBytes) >> 32);
      const uint32_t v_lo = static_cast<uint32_t>(value_desc(0, C::kBlockBytes));
      auto scores = [&](int i, int j) {  // S = Q_i K_j^T, when the last S is read and K_j there
        const int it = 2 * j, st = it % C::kStages;
        // before the first there is no S to wait for
        if (!wait2(item(it), it / C::kStages, used > 0 ? bar(sh.s_free) : item(it),
                   used > 0 ? used - 1 : it / C::kStages))
          return false;
        ++used;
        const uint32_t q = k_lo + desc_addr(base + i * C::kTileBytes);
        const uint32_t k = k_lo + desc_addr(s_stage + st * C::kStageBytes);
        auto step = [&](int s) {
          const uint32_t off = ((s >> 2) * C::kBlockBytes + (s & 3) * 32) >> 4;
          mma_ss(tm_s, desc64(q + off, k_hi), desc64(k + off, k_hi), idesc_s, s > 0, one);
        };
        if (full_d) {
#pragma unroll
          for (int s = 0; s < DP / 16; ++s) step(s);
        } else {
#pragma unroll 1
          for (int s = 0; s < k_steps; ++s) step(s);
        }
        commit(bar(sh.s_ready[i]), one);
        return true;
      };
      auto values = [&](int i, int j) {  // O_i += P_i V_j
        const int it = 2 * j + 1, st = it % C::kStages;
        if (!wait2(item(it), it / C::kStages, bar(sh.p_ready[i]), j)) return false;
        const uint32_t v = v_lo + desc_addr(s_stage + st * C::kStageBytes);
#pragma unroll
        for (int s = 0; s < kTile / 16; ++s)
          mma_ts(tm_o + 128 * i, tm_p + 64 * i + 8 * s, desc64(v + s * 128, v_hi), idesc_o,
                 j > 0 || s > 0, one);
        commit(bar(sh.p_free[i]), one);
        return true;
      };
      bool ok = warp_wait(sh.q_ready, 0);
      if (ok && n_steps > 0) {
        if (steps0 > 0) ok = scores(0, 0);
        if (ok && steps1 > 0) ok = scores(1, 0);
        if (ok) commit(bar(sh.empty[0]), one);
      }
      for (int j = 0; j < n_steps && ok; ++j) {
        if (j + 1 < steps0) ok = scores(0, j + 1);
        if (ok && j < steps0) ok = values(0, j);
        if (ok && j + 1 < steps1) ok = scores(1, j + 1);
        if (ok && j + 1 < n_steps) commit(bar(sh.empty[(2 * j + 2) % C::kStages]), one);
        if (ok && j < steps1) ok = values(1, j);
        if (ok) commit(bar(sh.empty[(2 * j + 1) % C::kStages]), one);
      }
    } else if (!kE4m3 && warp >= 10) {
      // ---------------------------------------------- values that not every row sees
      for (int it = 0; it < n_items; ++it) {  // keys too: a stage holds either in turn
        const int st = it % C::kStages, key0 = (first_tile + (it >> 1)) * kTile;
        if (!warp_wait(sh.full[st], it / C::kStages)) break;
        if ((it & 1) && key0 + kTile > vis_min) {
          // 64 rows by 128 bytes at a time, a lane's eight loads under way together
          const int pc = lane & 7, r_of = 32 * (warp - 10) + (lane >> 3);
#pragma unroll 1
          for (int h = 0; h < C::kHalves; ++h) {
            uint8_t* v = smem + 2 * C::kTileBytes + st * C::kStageBytes + h * C::kBlockBytes + pc * 16;
#pragma unroll 1
            for (int first = max(vis_min - key0, 0); first < kTile; first += 64) {
              uint32_t found = 0;  // bit k: this lane's piece of row first + 4 k + r_of
              uint4 x[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const int r = first + 4 * k + r_of;
                x[k] = r < kTile ? *reinterpret_cast<const uint4*>(v + r * 128) : make_uint4(0, 0, 0, 0);
              }
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const int r = first + 4 * k + r_of;
                // an exponent of ones carries into the sign's place
                const uint32_t carry = ((x[k].x & 0x7F807F80u) + 0x00800080u) | ((x[k].y & 0x7F807F80u) + 0x00800080u) |
                                       ((x[k].z & 0x7F807F80u) + 0x00800080u) | ((x[k].w & 0x7F807F80u) + 0x00800080u);
                if (r < kTile && key0 + r >= vis_max)
                  *reinterpret_cast<uint4*>(v + r * 128) = make_uint4(0, 0, 0, 0);
                else if (carry & 0x80008000u)
                  found |= 1u << k;
              }
              for (; found; found &= found - 1) {
                const int r = first + 4 * (__ffs(found) - 1) + r_of, ch = h * 64 + ((pc ^ (r & 7)) << 3);
                uint32_t* w = reinterpret_cast<uint32_t*>(v + r * 128);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  uint32_t both = w[k];
                  if ((both & 0x7F80u) == 0x7F80u) {
                    atomicMin(&sh.first_bad[ch + 2 * k], key0 + r);
                    both &= 0xFFFF0000u;
                  }
                  if ((both & 0x7F800000u) == 0x7F800000u) {
                    atomicMin(&sh.first_bad[ch + 2 * k + 1], key0 + r);
                    both &= 0x0000FFFFu;
                  }
                  w[k] = both;
                }
                sh.any_bad = 1;
              }
            }
          }
          fence_proxy_async_smem();
        }
        warp_arrive(sh.ready[st]);
      }
    } else if (kE4m3 && warp >= 12) {
      // ---------------------------------------------- codes to fp16 operand tiles, scales
      // Warp w has rows 32 w .. 32 w + 31 of a tile, four lanes a row: codes 16 c .. and
      // 64 + 16 c .. of it (c = lane & 3).  Neighbouring groups of four take rows r and
      // r ^ 5, so that neither the reads nor the writes meet in a bank.
      const int w = warp - 12, t = threadIdx.x - 384;
      const int c = lane & 3, pair_row = (lane >> 3) & 3;
      const int row8 = (lane & 4) ? pair_row ^ 5 : pair_row;  // of eight
      const int row0 = 32 * w + row8;
      constexpr int kPer = DP / 64;                 // 16-byte pieces of codes per row and lane
      constexpr int kSwizzle = DP == 128 ? 7 : 0;   // of the codes' 128-byte rows
      // Thread t has key t of a tile: its scales are looked up a step ahead, its page two.
      const int64_t head = static_cast<int64_t>(hk) << a.page_log2;
      const int page_mask = (1 << a.page_log2) - 1;
      auto page_of = [&](int j) -> int {
        const int key = (first_tile + j) * kTile + t;
        return j < n_steps && key < vis_max ? __ldg(table + (key >> a.page_log2)) : -1;
      };
      auto scale_of = [&](const float* scales, int page) -> float {
        if (page < 0 || page >= a.n_pages) return 0.f;
        return __ldg(scales + page * a.ld_scale_page + head + (t & page_mask));
      };
      // numbers order like their bits; what is not finite counts as 0, and 0 not at all
      auto bits_of = [](float x) { return fabsf(x) < INFINITY ? __float_as_uint(fabsf(x)) : 0u; };
      int page = page_of(0);
      float k_now = scale_of(a.k_scale, page), v_now = scale_of(a.v_scale, page);
      page = page_of(1);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t bits = bits_of(i ? v_now : k_now);
        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, bits);
        const uint32_t low = __reduce_min_sync(0xFFFFFFFFu, bits - 1u);
        if (lane == 0) {
          sh.tops[i][w] = top;
          sh.lows[i][w] = low;
        }
      }
      warp_arrive(sh.scales_ready);
      const bool begun = warp_wait(sh.scales_ready, 0);
      // The least bits of the keys' and values' scales in range, and whether (keys 1, values 2) they
      // left it, so that each is divided by a power of two of its own.
      uint32_t least[2], apart = 0u;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t *tops = sh.tops[i], *lows = sh.lows[i];
        const uint32_t top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
        const uint32_t low = min(min(lows[0], lows[1]), min(lows[2], lows[3]));
        const int ref = min(max(top == 0u ? 127 : static_cast<int>(top >> 23) + 1, 20), 240);  // biased
        least[i] = static_cast<uint32_t>(ref - kScalesBelow) << 23;
        if (low != 0xFFFFFFFFu &&
            (low + 1u < least[i] || top >= static_cast<uint32_t>(ref + kScalesAbove) << 23))
          apart |= 1u << i;
        if (t == 0) (i ? sh.v_ref : sh.k_ref) = pow2(ref - 127);
      }
      if (t == 0) {
        sh.k_from = apart & 1u ? 0 : 0x7FFFFFFF;
        sh.v_from = apart & 2u ? 0 : 0x7FFFFFFF;
        sh.apart_from = apart ? 0 : 0x7FFFFFFF;
        mbar_arrive(bar(sh.refs_ready));
      }
      auto out_of_range = [&](int i, float x) {
        const uint32_t bits = bits_of(x);
        return bits != 0u && bits - least[i] >= static_cast<uint32_t>(kScalesBelow + kScalesAbove) << 23;
      };
      // An operand tile: codes to fp16 times their keys' factors.  What the places of this step's
      // powers held was last read in step j - 3, which is over since the stage of this step's
      // keys, where that one's values were, was free for the copy.
      auto convert = [&](int it, float now) -> bool {
        const int st = it % C::kStages, j = it >> 1, key0 = (first_tile + j) * kTile;
        if (!warp_wait(sh.full[st], it / C::kStages)) return false;
        // a value vector that is NaN and that some row must not see becomes zeros, and is noted
        if ((it & 1) && !(fabsf(now) < INFINITY) && key0 + t >= vis_min) {
          if (key0 + t < vis_max) {
            atomicMin(&sh.first_bad[0], key0 + t);
            sh.any_bad = 1;
          }
          now = 0.f;
        }
        // this key's factor as the sum of two fp16: keys use both, so that a product has
        // its own rounding only (a score is 128 of them), values the first
        float f = now * __uint_as_float((static_cast<uint32_t>(127 + 127 + 3 - kScalesBelow) << 23) - (it & 1 ? least[1] : least[0]));
        if (apart & (it & 1 ? 2u : 1u)) {
          int e;
          f = scale_parts(now, &e);
          (it & 1 ? sh.v_pow : sh.k_pow)[j % 3][t] = static_cast<uint16_t>((127 + e) << 7);
        }
        const __half f_hi = __float2half_rn(f);
        const __half f_lo = __float2half_rn(f - __half2float(f_hi));
        const uint32_t factors = static_cast<uint32_t>(__half_as_ushort(f_hi)) |
                                 (static_cast<uint32_t>(__half_as_ushort(f_lo)) << 16);
        uint8_t* stage = smem + 2 * C::kTileBytes + st * C::kStageBytes;
        uint4 x[4][kPer];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int p = 0; p < kPer; ++p)
            x[k][p] = *reinterpret_cast<const uint4*>(stage + C::kRawAt + (row0 + 8 * k) * DP +
                                                      (((c + 4 * p) ^ (row8 & kSwizzle)) << 4));
        if (key0 + kTile > vis_max) {  // rows from vis_max on are not this sequence's
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (key0 + row0 + 8 * k >= vis_max)
#pragma unroll
              for (int p = 0; p < kPer; ++p) x[k][p] = make_uint4(0, 0, 0, 0);
        }
        __syncwarp();  // the rows' codes are read: their place may be written
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t both = __shfl_sync(0xFFFFFFFFu, factors, row8 + 8 * k);
          const uint32_t hi = __byte_perm(both, 0, 0x1010), lo = __byte_perm(both, 0, 0x3232);
#pragma unroll
          for (int p = 0; p < kPer; ++p) {
            const uint32_t u[4] = {x[k][p].x, x[k][p].y, x[k][p].z, x[k][p].w};
            uint32_t o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint32_t code = e4m3x2_f16x2(u[e >> 1], e & 1);
              if (it & 1) {
                asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(o[e]) : "r"(code), "r"(hi));
              } else {
                asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(o[e]) : "r"(code), "r"(lo));
                asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(o[e]) : "r"(code), "r"(hi));
              }
            }
            uint8_t* row = stage + p * C::kBlockBytes + (row0 + 8 * k) * 128;
            *reinterpret_cast<uint4*>(row + (((2 * c) ^ row8) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
            *reinterpret_cast<uint4*>(row + (((2 * c + 1) ^ row8) << 4)) =
                make_uint4(o[4], o[5], o[6], o[7]);
          }
        }
        fence_proxy_async_smem();
        return true;
      };
      // Keys and values in turn, by the same instructions: twice the code costs its fetch.
      float k_next = 0.f, v_next = 0.f;
#pragma unroll 1
      for (int it = 0; it < n_items && begun; ++it) {
        const int j = it >> 1;
        if (!(it & 1)) {
          k_next = scale_of(a.k_scale, page);
          v_next = scale_of(a.v_scale, page);
          page = page_of(j + 2);
        }
        if (!convert(it, it & 1 ? v_now : k_now)) break;
        // Whether the next step's scales are in range, settled before this step's values are
        // ready: who has waited for those knows.
        if (it & 1) {
          if (!warp_wait(sh.scales_ready, j + 1)) break;
          const uint32_t* fars = sh.far[j & 1];
          const uint32_t far = fars[0] | fars[1] | fars[2] | fars[3];
          if (far & ~apart) {
            if (t == 0) {
              if (far & ~apart & 1u) sh.k_from = j + 1;
              if (far & ~apart & 2u) sh.v_from = j + 1;
              if (apart == 0u) sh.apart_from = j + 1;
            }
            apart |= far;
          }
          k_now = k_next;
          v_now = v_next;
        }
        warp_arrive(sh.ready[it % C::kStages]);
        if (!(it & 1)) {
          const uint32_t far = (__any_sync(0xFFFFFFFFu, out_of_range(0, k_next)) ? 1u : 0u) |
                               (__any_sync(0xFFFFFFFFu, out_of_range(1, v_next)) ? 2u : 0u);
          if (lane == 0) sh.far[j & 1][w] = far;
          warp_arrive(sh.scales_ready);
        }
      }
    }
    __syncwarp();
    if (cluster > 1) {  // the parts are there; they have been read
      cluster_sync();
      cluster_sync();
    }
  } else {
    regs_inc<C::kSoftmaxRegs>();
    const int i = warp >> 2;      // this thread's tile and its row there
    const int r = threadIdx.x & 127;
    float row_factor = a.scale_log2;  // of the scores, to log2 units
    // ------------------------------------------------ Q into the swizzled operand tiles
#pragma unroll
    for (int k = 0; k < kQRounds; ++k) {
      const int at = q_first + k * kQRowsAtOnce, tile = at / kTile, tr = at % kTile;
      *reinterpret_cast<uint4*>(smem + tile * C::kTileBytes + (q_chunk >> 3) * C::kBlockBytes + tr * 128 +
                                (((q_chunk & 7) ^ (tr & 7)) << 4)) = q_held[k];
    }
    if constexpr (kE4m3) {
      // to fp16: a thread its row, in short loops, since code that runs once per block
      // costs its fetch
      asm volatile("bar.sync 2, 256;" ::: "memory");
      uint8_t* row = smem + i * C::kTileBytes + r * 128;
      auto piece = [&](int c) {
        return reinterpret_cast<uint4*>(row + (c >> 3) * C::kBlockBytes + (((c & 7) ^ (r & 7)) << 4));
      };
      uint32_t tops = 0;  // of the low and the high halves
#pragma unroll 4
      for (int c = 0; c < kQChunks; ++c) {
        const uint4 x = *piece(c);
        tops = __vmaxu2(__vmaxu2(tops, __vmaxu2(x.x & 0x7FFF7FFFu, x.y & 0x7FFF7FFFu)),
                        __vmaxu2(x.z & 0x7FFF7FFFu, x.w & 0x7FFF7FFFu));
      }
      float up;
      row_factor = f16_row_scale(max(tops << 16, tops & 0xFFFF0000u), a.scale_log2, &up) / kCodeScale;
#pragma unroll 4
      for (int c = 0; c < kQChunks; ++c) {
        const uint4 x = *piece(c);
        uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[e] = pack_f16(__uint_as_float(w[e] << 16) * up, __uint_as_float(w[e] & 0xFFFF0000u) * up);
        *piece(c) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    fence_proxy_async_smem();
    warp_arrive(sh.q_ready);
    // ------------------------------------------------ softmax: one row per thread
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t ts = tm_s + lanes, tp = tm_p + 64 * i + lanes, to = tm_o + 128 * i + lanes;
    const int rows = i ? rows1 : rows0, steps = i ? steps1 : steps0;
    const bool live = r < rows;
    const bool warp_live = 32 * (warp & 3) < rows;
    const uint32_t row0 = static_cast<uint32_t>(r0) + i * kTile;
    const int vis = live ? visible(row0 + r) : 0;
    const int64_t tree_row = seq.row0 + (live ? row_token(row0 + r, a.group) : 0);
    // least visible count in the warp: steps below it need no mask
    const int vis_low = kTree ? vis_min : __reduce_min_sync(0xFFFFFFFFu, vis);
    // P = exp2(x + ref), l its sum, 0 until the row has seen a key: ref is minus the row's maximum
    // when it was last set, and kPBits more where that is exact enough (P up to 2^(11 + kSlack)
    // is a number of fp16, 2^(16 + kSlack) is not)
    auto ref_of = [](float top) -> float { return kE4m3 && fabsf(top) < 0x1p22f ? kPBits - top : -top; };
    float l = 0.f, ref = 0.f;
    bool alive = true;
    // e4m3: the scores' factor, and the step from which keys or values are divided by their own
    // scales' powers of two.  From then on O is in units of 2^v_exp / kPScale, which may fall by
    // v_room.
    float k_factor = row_factor;
    volatile int *const apart_from = &sh.apart_from, *const k_from = &sh.k_from, *const v_from = &sh.v_from;
    int apart = 0x7FFFFFFF, v_exp = kLeastExp;
    float v_room = kAllRoom;
    if (kE4m3 && warp_live && steps > 0) {
      alive = warp_wait(sh.refs_ready, 0);
      k_factor = fmaxf(row_factor * sh.k_ref, 0x1p-126f);
      apart = *apart_from;
    }
    int j = 0;
    // The steps before `apart`, or the others.
    auto go = [&](auto apart_) {
      constexpr bool kApart = decltype(apart_)::value;
      for (; j < steps && alive && (kApart || j < apart); ++j) {
        if (!warp_wait(sh.s_ready[i], j)) { alive = false; break; }
        tc_fence_after();
        if (!warp_live) {  // no rows of its own: P's lanes hold what they hold, nobody reads O's
          tc_fence_before();
          warp_arrive(sh.s_free);
          if (j > 0 && !warp_wait(sh.p_free[i], j - 1)) { alive = false; break; }
          warp_arrive(sh.p_ready[i]);
          continue;
        }
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32_async(ts + 32 * c, s[c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_wait_ld_pin(s[c]);
        tc_fence_before();
        warp_arrive(sh.s_free);
        const int key0 = (first_tile + j) * kTile;
        const bool edge = key0 + kTile > vis_low;
        float factor = k_factor;
        if constexpr (kE4m3) {  // the values' tile is converted right after the keys'
          if (!warp_wait(sh.ready[(2 * j + 1) % C::kStages], (2 * j + 1) / C::kStages)) {
            alive = false;
            break;
          }
          if (!kApart) apart = *apart_from;  // j + 1 at least
        }
        if constexpr (kApart) {
          if (j >= *k_from) {
            const float whole = row_factor * kCodeScale;
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int k = 0; k < 32; k += 2) {
                float f0, f1;
                powers_at(sh.k_pow[j % 3], 32 * c + k, f0, f1);
                s[c][k] = __float_as_uint(__uint_as_float(s[c][k]) * (whole * f0));
                s[c][k + 1] = __float_as_uint(__uint_as_float(s[c][k + 1]) * (whole * f1));
              }
          } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int k = 0; k < 32; ++k) s[c][k] = __float_as_uint(__uint_as_float(s[c][k]) * factor);
          }
          factor = 1.f;
        }
        if (edge) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t seen = 0u;
            if constexpr (kTree) {
              const int end = vis - (key0 + 32 * c);  // no key of the sequence from there on
              if (end > 0)
                seen = tree_bits(a, tree_row, key0 + 32 * c - prefix) & (end >= 32 ? 0xFFFFFFFFu : (1u << end) - 1u);
            }
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (kTree ? !((seen >> k) & 1u) : key0 + 32 * c + k >= vis) s[c][k] = 0xFF800000u;
          }
        }
        float top[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          top[c] = fmaxf(__uint_as_float(s[c][0]), __uint_as_float(s[c][1]));
#pragma unroll
          for (int k = 2; k < 32; k += 2)
            top[c] = max3(top[c], __uint_as_float(s[c][k]), __uint_as_float(s[c][k + 1]));
        }
        const float most = max3(fmaxf(top[0], top[1]), top[2], top[3]) * factor;
        if constexpr (kApart) {
          // Each value's power of two goes into its weight.
          const bool v_apart = j >= *v_from;
          const float v_unit = sh.v_ref / kCodeScale;
          const float top_was = l == 0.f ? -INFINITY : -ref, top_now = fmaxf(top_was, most);
          const float ref_new = top_now == -INFINITY ? 0.f : -top_now;
          float turn = l == 0.f ? 0.f : fast_exp2(ref_new - ref);  // of O
          v_room = l == 0.f ? kAllRoom : v_room + (top_now - top_was);
          ref = ref_new;
          l *= turn;
          float sum = 0.f, heaviest = 0.f;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
              float f0 = v_unit, f1 = v_unit;
              if (v_apart) powers_at(sh.v_pow[j % 3], 32 * c + k, f0, f1);
              const float p0 = fast_exp2(__uint_as_float(s[c][k]) + ref), p1 = fast_exp2(__uint_as_float(s[c][k + 1]) + ref);
              sum += p0 + p1;
              f0 *= p0;
              f1 *= p1;
              heaviest = max3(heaviest, f0, f1);
              s[c][k] = __float_as_uint(f0);
              s[c][k + 1] = __float_as_uint(f1);
            }
          l += sum;
          const int over = exponent_of(heaviest) - v_exp;  // of 2^11
          int up = 0;
          if (heaviest > 0.f && over > 3) {
            up = over;
            v_room = 0.f;
          } else if (heaviest > 0.f && over < -5) {
            up = -min(min(static_cast<int>(v_room), v_exp - kLeastExp), -over);
            if (v_room < 0.5f * kAllRoom) up = max(up, -120);  // what O can take at a time
            v_room += static_cast<float>(up);
          }
          if (heaviest > 0.f && v_room > 0.5f * kAllRoom) v_room = 0.f;
          v_exp += up;
          turn = turn * pow2(-(up / 2)) * pow2(-(up - up / 2));
          if (j > 0) {
            alive = warp_wait(sh.p_free[i], j - 1);
            tc_fence_after();
            if (alive && __any_sync(0xFFFFFFFFu, turn != 1.f)) {
#pragma unroll 1
              for (int c = 0; c < a.d; c += 16) tmem_scale_x16(to + c, turn);
            }
          }
          const float unit = exp_scale(v_exp);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t p[32];
#pragma unroll
            for (int k = 0; k < 64; k += 2) {
              const int c = 2 * h + (k >> 5);
              p[k >> 1] = pack_f16(__uint_as_float(s[c][k & 31]) * unit, __uint_as_float(s[c][(k & 31) + 1]) * unit);
            }
            if (alive) tmem_st_x32(tp + 32 * h, p);
          }
          if (!alive) break;
          tmem_wait_st();
          tc_fence_before();
          warp_arrive(sh.p_ready[i]);
          continue;
        }
        const bool move = most + ref > (kE4m3 ? kPBits : 0.f) + kSlack || (l == 0.f && most > -INFINITY);
        const bool big = fabsf(most) >= 0x1p20f && fabsf(most) < INFINITY;
        if (__any_sync(0xFFFFFFFFu, move || big)) {
          // The product s factor is not rounded before ref is added to it below, most is: where
          // scores are big the difference would count.
          if (__any_sync(0xFFFFFFFFu, big)) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int k = 0; k < 32; ++k) s[c][k] = __float_as_uint(__uint_as_float(s[c][k]) * factor);
            factor = 1.f;
          }
          const float ref_new = move ? ref_of(most) : ref;
          const float shrink = l == 0.f ? 0.f : fast_exp2(ref_new - ref);
          ref = ref_new;
          l *= shrink;
          if (j > 0) {
            if (!warp_wait(sh.p_free[i], j - 1)) { alive = false; break; }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < a.d; c += 16) tmem_scale_x16(to + c, shrink);
          }
        }
        const uint64_t factor2 = pair(factor, factor), ref2 = pair(ref, ref);
        uint64_t l2[2] = {0, 0};
        auto half = [&](int h) {
          uint32_t p[32];
#pragma unroll
          for (int k = 0; k < 64; k += 2) {
            const int c = 2 * h + (k >> 5);
            const uint64_t x = fma2(pair(__uint_as_float(s[c][k & 31]), __uint_as_float(s[c][(k & 31) + 1])),
                                    factor2, ref2);
            float p0, p1;
            unpair(x, p0, p1);
            const uint64_t y = pair(fast_exp2(p0), fast_exp2(p1));
            l2[(k >> 1) & 1] = add2(l2[(k >> 1) & 1], y);
            unpair(y, p0, p1);
            p[k >> 1] = kE4m3 ? pack_f16(p0, p1) : pack_bf16(p0, p1);
          }
          if (h == 0 && j > 0) {  // the product that read the last P
            alive = warp_wait(sh.p_free[i], j - 1);
            tc_fence_after();
          }
          tmem_st_x32(tp + 32 * h, p);
        };
        half(0);
        half(1);
        if (!alive) break;
        tmem_wait_st();
        tc_fence_before();
        warp_arrive(sh.p_ready[i]);
        float l0, l1;
        unpair(add2(l2[0], l2[1]), l0, l1);
        l += l0 + l1;
      }
    };
    go(std::false_type{});
    const bool rest = kE4m3 && warp_live && alive && j < steps;
    if (rest) {
      if (j > 0) {
        v_exp = exponent_of(sh.v_ref / kCodeScale) + static_cast<int>(kPBits);
        v_room = 0.f;
      }
      go(std::bool_constant<kE4m3>{});
    }
    if (steps > 0 && alive) alive = warp_wait(sh.p_free[i], steps - 1);
    // (Q's rows come from all warps: one whose tile has no keys may be here before they are in place, and goes
    // through them on its way out.)
    if (steps == 0 && alive) alive = warp_wait(sh.q_ready, 0);
    tc_fence_after();
    // ---------------------------------------------- out
    const bool have = steps > 0 && alive;
    if (!alive || sh.bad_page) l = __uint_as_float(0x7FC00000u);
    if (sh.bad_page && threadIdx.x == 0) paged_report(a.status);
    // O is in units of P's power of two, which l has too, and of the values'
    if (cluster == 1) {
      const float v_back = !kE4m3 ? 1.f
                           : rest ? pow2(v_exp - static_cast<int>(kPBits))
                                  : sh.v_ref / kCodeScale;
      // through this warp's rows of Q's tile, which no product needs any more, so that
      // rows leave whole (a row per thread at 16 bytes a store took 7 us per block)
      const float inv = 1.f / l;
      const bool some_bad = sh.any_bad;
      uint8_t* stage = smem + i * C::kTileBytes + 32 * (warp & 3) * (2 * DP);
      if (warp_live) {
#pragma unroll 1
        for (int c = 0; c < DP / 32; ++c) {
          float o[32];
          if (have) {
            tmem_ld_32x32b_x32_sync(to + 32 * c, o);
          } else {
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = 0.f;
          }
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = l == 0.f ? 0.f : o[k] * inv * v_back;
          if (some_bad) {
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (sh.first_bad[kE4m3 ? 0 : 32 * c + k] < vis &&
                  (!kTree || tree_sees_bad<kE4m3>(a, seq, table, hk, tree_row, 32 * c + k)))
                o[k] = __uint_as_float(0x7FC00000u);
          }
#pragma unroll
          for (int k = 0; k < 32; k += 8)
            *reinterpret_cast<uint4*>(stage + lane * (2 * DP) + (((4 * c + k / 8) ^ (lane & 7)) << 4)) =
                make_uint4(pack_bf16(o[k], o[k + 1]), pack_bf16(o[k + 2], o[k + 3]),
                           pack_bf16(o[k + 4], o[k + 5]), pack_bf16(o[k + 6], o[k + 7]));
        }
        __syncwarp();
        constexpr int kChunks = DP / 8;
        const int chunk = lane % kChunks;
        RowWalk at(row0 + 32 * (warp & 3) + lane / kChunks, a.group, 32 / kChunks);
        uint16_t* const out = a.out + static_cast<int64_t>(hk) * a.group * a.d + 8 * chunk;
#pragma unroll 4
        for (int k = 0; k < kChunks; ++k, at.next()) {
          const int q = lane / kChunks + k * (32 / kChunks);
          if (q < rows - 32 * (warp & 3) && 8 * chunk < a.d)
            *reinterpret_cast<uint4*>(out + (seq.row0 + at.token) * a.out_ld + at.head * a.d) =
                *reinterpret_cast<const uint4*>(stage + q * (2 * DP) + ((chunk ^ (q & 7)) << 4));
        }
      }
    } else {
      // The cluster's blocks share out the unit's rows, and each sends every other its part
      // of that one's rows: O [32 rows][channel / 4][row] by fours, so that a warp's stores
      // are contiguous, and m and l.  Stores into another block's shared memory are not
      // waited for; loads from it, which take a microsecond each, made the join 11 us; it takes 5.
      const int log2_rows = 8 - (31 - __clz(cluster)), rows_of = 1 << log2_rows;
      const int mine = i * kTile + r;
      const int slot = (split << log2_rows) + (mine & (rows_of - 1));
      cluster_sync();  // every block's products have read their operands
      const uint32_t there = map_to_cta(base, mine >> log2_rows);
      if (warp_live) {
#pragma unroll 1
        for (int c = 0; c < DP / 32; ++c) {
          float o[32];
          if (have) {
            tmem_ld_32x32b_x32_sync(to + 32 * c, o);
          } else {
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = 0.f;
          }
          const uint32_t dst = there + (((slot >> 5) * (DP / 4) + 8 * c) * 32 + (slot & 31)) * 16;
#pragma unroll
          for (int k = 0; k < 32; k += 4)
            st_cluster_f32x4(dst + 128 * k, o[k], o[k + 1], o[k + 2], o[k + 3]);
        }
      }
      st_cluster_f32x2(there + C::kPartMl + 8 * slot, l == 0.f ? -INFINITY : -ref, l);
      // the values' power of two goes with a part, not into it: sums that are not yet divided by l would leave f32
      if constexpr (kE4m3)
        st_cluster_s32(there + C::kPartUnit + 4 * slot,
                       rest ? v_exp - static_cast<int>(kPBits) : exponent_of(sh.v_ref / kCodeScale));
      if (sh.any_bad) {
        for (int at = threadIdx.x; at < cluster * kBads; at += 256)
          min_cluster_s32(map_to_cta(smem_u32(&sh.first_bad[at % kBads]), at / kBads), sh.first_bad[at % kBads]);
        if (threadIdx.x < cluster) st_cluster_s32(map_to_cta(smem_u32(&sh.any_bad), threadIdx.x), 1);
      }
      cluster_sync();
      // A warp joins eight rows at a time, lane (x, q) channels 4 x + 16 t of row q: all of
      // a part's loads are under way together, and free of bank conflicts.
      const bool some_bad = sh.any_bad;
      const int row_end = rows0 + rows1 - (split << log2_rows);  // of this block's rows
      const int q = lane & 7, x = lane >> 3;
      for (int first = 8 * warp; first < min(rows_of, row_end); first += 64) {
        const int row = first + q;
        float top = -INFINITY, sum = 0.f;
        for (int c = 0; c < cluster; ++c)
          top = fmaxf(top, *reinterpret_cast<const float*>(smem + C::kPartMl + 8 * ((c << log2_rows) + row)));
        float y[DP / 16][4] = {};
        // y is in units of 2^unit, about the largest of the parts' units times their weights
        int unit = -4096;
        if constexpr (kE4m3) {
          for (int c = 0; c < cluster; ++c) {
            const int at = (c << log2_rows) + row;
            const float m = *reinterpret_cast<const float*>(smem + C::kPartMl + 8 * at);
            if (m > -INFINITY)
              unit = max(unit, *reinterpret_cast<const int*>(smem + C::kPartUnit + 4 * at) +
                                   static_cast<int>(fmaxf(m - top, -1024.f)));
          }
        }
#pragma unroll 1
        for (int c = 0; c < cluster; ++c) {
          const int at = (c << log2_rows) + row;
          const float2 ml = *reinterpret_cast<const float2*>(smem + C::kPartMl + 8 * at);
          float4 o[DP / 16];
#pragma unroll
          for (int t = 0; t < DP / 16; ++t)
            o[t] = *reinterpret_cast<const float4*>(smem + (((at >> 5) * (DP / 4) + 4 * t + x) * 32 + (at & 31)) * 16);
          // a part without keys has l = 0 (or NaN, which has to stay)
          const float weight = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - top);
          sum += ml.x == -INFINITY ? ml.y : weight * ml.y;
          float of_o = weight;
          if constexpr (kE4m3)
            of_o = ml.x == -INFINITY ? 0.f
                                     : fast_exp2((ml.x - top) + static_cast<float>(
                                           *reinterpret_cast<const int*>(smem + C::kPartUnit + 4 * at) - unit));
          if (of_o != 0.f) {  // else what is there may be anything
#pragma unroll
            for (int t = 0; t < DP / 16; ++t) {
              y[t][0] += of_o * o[t].x;
              y[t][1] += of_o * o[t].y;
              y[t][2] += of_o * o[t].z;
              y[t][3] += of_o * o[t].w;
            }
          }
        }
        if (row >= row_end) continue;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        if constexpr (kE4m3) {  // in two steps: the unit has more than f32's exponents
          unit = min(max(unit, -250), 250);
          const float one = inv * pow2(unit / 2), two = pow2(unit - unit / 2);
#pragma unroll
          for (int t = 0; t < DP / 16; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[t][e] = y[t][e] * one * two;
        } else {
#pragma unroll
          for (int t = 0; t < DP / 16; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[t][e] *= inv;
        }
        const uint32_t of_unit = row_0 + (split << log2_rows) + row, token = row_token(of_unit, a.group);
        uint16_t* const out = a.out + (seq.row0 + token) * a.out_ld +
                              (static_cast<int64_t>(hk) * a.group + of_unit - token * a.group) * a.d + 4 * x;
        if (some_bad) {
          const int vis_q = visible(of_unit);
#pragma unroll
          for (int t = 0; t < DP / 16; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (sh.first_bad[kE4m3 ? 0 : 16 * t + 4 * x + e] < vis_q &&
                  (!kTree || tree_sees_bad<kE4m3>(a, seq, table, hk, seq.row0 + token, 16 * t + 4 * x + e)))
                y[t][e] = __uint_as_float(0x7FC00000u);
        }
#pragma unroll
        for (int t = 0; t < DP / 16; ++t)
          if (16 * t < a.d)  // d is a multiple of 16
            *reinterpret_cast<uint2*>(out + 16 * t) =
                make_uint2(pack_bf16(y[t][0], y[t][1]), pack_bf16(y[t][2], y[t][3]));
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(sh.tmem, 512);
  }
}

// What a device has, asked for once: how many clusters of 1, 2, 4 and 8 blocks run at a time
// (a block fills an SM, and a cluster has to find its SMs in one part of the chip: 15 of 8
// blocks on 148 SMs).  Also lets the kernel have its shared memory, and checks that the
// launch brings the registers that the warps share out among themselves.
template <bool kE4m3, int DP, bool kTree>
cudaError_t configure_mma(cudaLaunchConfig_t cfg, const int** clusters) {
  using C = MmaCfg<kE4m3, DP>;
  static std::atomic<bool> done[64] = {};
  static int fit[64][4];
  static std::mutex once;
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
  if (dev >= 64) return cudaErrorInvalidDevice;
  *clusters = fit[dev];
  if (done[dev].load(std::memory_order_acquire)) return cudaSuccess;
  const std::lock_guard<std::mutex> lock(once);
  if (done[dev].load(std::memory_order_relaxed)) return cudaSuccess;  // meanwhile
  cudaFuncAttributes attr;
  if (cudaError_t e = cudaFuncGetAttributes(&attr, paged_mma_kernel<kE4m3, DP, kTree>); e != cudaSuccess)
    return e;
  if (attr.numRegs * C::kThreads <
      256 * C::kSoftmaxRegs + (C::kThreads - 256) * C::kOtherRegs)
    return cudaErrorInvalidConfiguration;
  if (cudaError_t e = cudaFuncSetAttribute(paged_mma_kernel<kE4m3, DP, kTree>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
      e != cudaSuccess)
    return e;
  int found[4] = {device_sm_count()};
  for (int i = 1; i < 4; ++i) {
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = 1u << i;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    cfg.gridDim = dim3(1u << i);
    cfg.attrs = &cluster;
    cfg.numAttrs = 1;
    if (cudaError_t e = cudaOccupancyMaxActiveClusters(&found[i], paged_mma_kernel<kE4m3, DP, kTree>, &cfg);
        e != cudaSuccess)
      return e;
  }
  for (int i = 0; i < 4; ++i) fit[dev][i] = found[i];
  done[dev].store(true, std::memory_order_release);
  return cudaSuccess;
}

template <bool kE4m3, int DP, bool kTree>
cudaError_t launch_mma(const PagedArgs& a, cudaStream_t stream) {
  using C = MmaCfg<kE4m3, DP>;
  CUtensorMap mk, mv;
  const int row_bytes = kE4m3 ? DP : 128, box_rows = 1 << a.page_log2;
  if (!make_page_map(&mk, a.k, a, row_bytes, box_rows, 1) ||
      !make_page_map(&mv, a.v, a, row_bytes, box_rows, 1))
    return cudaErrorInvalidValue;
  const int64_t most_rows = static_cast<int64_t>(a.max_q) * a.group;
  const int row_units = static_cast<int>((most_rows + 2 * kTile - 1) / (2 * kTile));
  const int64_t units = static_cast<int64_t>(a.B) * a.H_kv * row_units;
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  const int* at_a_time;
  if (cudaError_t e = configure_mma<kE4m3, DP, kTree>(cfg, &at_a_time); e != cudaSuccess) return e;
  // How many blocks share a unit's keys: what takes clearly the fewest rounds of steps
  // (a step is 3000 to 3900 cycles), if every sequence were as long as the table allows.  A
  // block costs about three steps more than its keys, a split one six and more: its
  // part goes through distributed shared memory.  Trees are of sequences at different points of their
  // answers: there the longest unit takes its time whatever the others do, and with the longest first all are
  // through about a third of a unit behind the mean of half the table's length; what gains more by this, in
  // proportion, than it loses by the first.  (16 trees of 33 to 64 nodes, 8 e4m3 heads of 4 query heads and 128
  // channels: over 2000 to 16384 tokens 278 us whole, 160 in two, 195 in four; over 16384 each 318, 337 and
  // 355; over 2048 each 51, 70 and 100.  80 units of 64 rows over 3000 tokens each, bf16, 44 whole, 55 in two;
  // ragged 42 and 31.)  Clearly the fewest is a tenth fewer, of trees a twelfth: in between, parts save ragged contexts
  // more than they cost equal ones (whole and in two, bf16 and e4m3: 16 trees of 80 nodes over 8576 tokens, 8 heads,
  // ragged 97 and 73, 127 and 86, equal 97 and 113, 134 and 143; 9 over 5248, 12 heads, ragged 62 and 39, 79 and 48,
  // equal 63 and 79, 83 and 97; 3 over 1152, 16 heads, either 21 and 18, 26 and 22).
  const int64_t steps = ((static_cast<int64_t>(a.max_pages) << a.page_log2) + kTile - 1) / kTile;
  auto cost_of = [&](int c, int64_t fit) -> double {
    const int64_t own = (steps + c - 1) / c, more = c == 1 ? 3 : 6 + c / 4;
    const double equal = static_cast<double>((units + fit - 1) / fit * (own + more));
    if (!kTree || a.B == 1) return equal;
    return std::sqrt(equal * static_cast<double>(std::max(own + more, units * (own / 2 + more) / fit + own / 3)));
  };
  int cluster = 1;
  double best = cost_of(1, at_a_time[0]);
  for (int i = 1; 1 << i <= kMaxSplit; ++i) {
    const int c = 1 << i;
    if (at_a_time[i] < 1) break;
    const double cost = cost_of(c, at_a_time[i]);
    if (10.0 * cost < (kTree ? 9.2 : 9.0) * best) {
      best = cost;
      cluster = c;
    }
  }
  if (units * cluster > 0x7FFFFFFFll) return cudaErrorInvalidConfiguration;
  cfg.gridDim = dim3(static_cast<unsigned>(units * cluster));
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(cluster);
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, paged_mma_kernel<kE4m3, DP, kTree>, mk, mv, a, row_units, cluster);
}

template <bool kTree>
cudaError_t launch_many_rows(const PagedArgs& a, cudaStream_t stream) {
  const bool e4m3 = a.k_scale != nullptr;
  if (a.d <= 64) return e4m3 ? launch_mma<true, 64, kTree>(a, stream) : launch_mma<false, 64, kTree>(a, stream);
  return e4m3 ? launch_mma<true, 128, kTree>(a, stream) : launch_mma<false, 128, kTree>(a, stream);
}

}  // namespace

cudaError_t launch_paged_attention_mma(const PagedArgs& a, cudaStream_t stream) {
  return a.tree != nullptr ? launch_many_rows<true>(a, stream) : launch_many_rows<false>(a, stream);
}

}  // namespace dwa
