// paged_attention_mma.cu — attention of a chunk of new tokens over the paged
// cache on tcgen05: prompts in pieces, long drafts, anything with many rows per
// key/value head.
//
// A block takes 256 rows of one key/value head (a row is one (new token, query
// head), token-major) as two tiles of 128, and goes once over the keys they may
// see, 128 at a time:
//
//   S_i = Q_i K^T        tcgen05, Q and K in shared memory, S_i in TMEM
//   P_i = exp2(S_i - m)  one thread per row: running maximum, sum, P_i back to TMEM
//   O_i += P_i V         tcgen05, P_i from TMEM, V in shared memory, O_i in TMEM
//
// TMEM is full: two S of 128 columns (P_i takes the first half of S_i's), two O
// of 128.  The tiles run in turn, so that one's products overlap the other's
// exponentials: per 128 keys the two products take 2 x 1024 cycles of the tensor
// pipe and the exponentials 32768 / 16 = 2048 cycles of the special-function
// units.  m only moves when a row's maximum grew by more than 2^kSlack (the
// result does not depend on m; P stays below 2^kSlack), so O is hardly ever
// rescaled, and then by the row's own thread.
//
// Warps 0-3 and 4-7: the rows of tile 0 and 1.  Warp 8: issues every tcgen05.mma.
// Warp 9: TMA, one box of 64 channels per page, straight from the pages into the
// swizzled operand tiles.  bf16 caches: warps 10-11 look over the values of tiles
// that end behind what every row sees, since 0 * NaN would reach rows that must
// not see it.  e4m3 caches: warps 12-15 turn codes into fp16 (exact) operand
// tiles, Q is scaled per row by a power of two into fp16, and P carries the
// values' scales relative to a running power of two.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "dwa_internal.h"
#include "paged_attention.cuh"
#include "sm100_ptx.cuh"

namespace dwa {

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

bool make_page_map(CUtensorMap* map, const void* ptr, const PagedArgs& a, int row_bytes, int box_rows) {
  auto encode = tensor_map_encoder();
  if (!encode) return false;
  const bool e4m3 = a.k_scale != nullptr;
  const uint64_t es = e4m3 ? 1 : 2;
  const uint64_t page = 1ull << a.page_log2;
  // a page's heads, then the pages; a single page may have any stride
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.d), page, static_cast<cuuint64_t>(a.H_kv),
                        static_cast<cuuint64_t>(a.n_pages)};
  cuuint64_t strides[3] = {a.d * es, page * a.d * es, a.ld_page * es};
  cuuint32_t box[4] = {static_cast<cuuint32_t>(row_bytes / es), static_cast<cuuint32_t>(box_rows), 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return encode(map, e4m3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                row_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace {

constexpr int kTile = 128;     // rows per tile, keys per step
constexpr int kMaxChannels = 128;
constexpr float kSlack = 4.f;  // log2 of how far P may grow before m follows

template <bool kE4m3, int DP>
struct MmaCfg {
  static constexpr int kThreads = kE4m3 ? 512 : 384;
  static constexpr int kSoftmaxRegs = kE4m3 ? 176 : 208;
  static constexpr int kOtherRegs = kE4m3 ? 80 : 88;
  static constexpr int kHalves = DP / 64;               // 128-byte wide column blocks
  static constexpr int kBlockBytes = kTile * 128;       // one of them: 16 KB
  static constexpr int kTileBytes = kHalves * kBlockBytes;
  static constexpr int kStages = kE4m3 ? 3 : 5;         // operand tiles (K and V in turn)
  static constexpr int kRaw = kE4m3 ? 3 : 0;            // code tiles
  static constexpr int kRawBytes = kTile * DP;
  static constexpr int kSmem = 1024 + 2 * kTileBytes + kStages * kTileBytes + kRaw * kRawBytes;
};

template <bool kE4m3>
struct MmaShared {
  uint64_t full[5], ready[5], empty[5], raw_full[3], raw_empty[3];
  uint64_t s_ready[2], p_ready[2], done[2];
  uint32_t tmem;
  int abort;
  int bad_page;
  int any_bad;
  int first_bad[kMaxChannels];  // least key with a value that is not finite
  // e4m3 only: what a row of Q was divided by, with the scale; the keys' and
  // values' scales of four steps
  float q_factor[kE4m3 ? 2 * kTile : 1];
  __align__(16) float scales[kE4m3 ? 4 : 1][2][kE4m3 ? kTile : 4];
};

// ---------------------------------------------------------------- tcgen05 pieces
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t add) {
  umma_bf16_ss(d, a, b, idesc, add);
}
// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(add)
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

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x,
                                            int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

template <int kRegs>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

// What a block works on.
struct Unit {
  PagedSeq seq;
  int hk;
  int64_t r0;        // its first row of the sequence's rows
  int rows[2];       // rows of each tile
  int steps[2];      // key tiles of each tile
  int n_steps;       // of the block
  int vis_min, vis_max;
};

template <bool kE4m3, int DP>
__global__ void __launch_bounds__(MmaCfg<kE4m3, DP>::kThreads, 1)
    paged_mma_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                     const PagedArgs a, const int row_units) {
  using C = MmaCfg<kE4m3, DP>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ MmaShared<kE4m3> sh;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
  // [Q tile 0][Q tile 1][operand stages][code stages]
  const uint32_t s_stage = base + 2 * C::kTileBytes;
  const uint32_t s_raw = s_stage + C::kStages * C::kTileBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ------------------------------------------------ the block's work
  Unit u;
  int64_t unit = blockIdx.x;
  // late rows (more keys) first
  const int ru = row_units - 1 - static_cast<int>(unit / (static_cast<int64_t>(a.B) * a.H_kv));
  unit %= static_cast<int64_t>(a.B) * a.H_kv;
  u.hk = static_cast<int>(unit % a.H_kv);
  const int b = static_cast<int>(unit / a.H_kv);
  u.seq = paged_seq(a, b);
  if (u.seq.bad && u.hk == 0 && ru == 0 && threadIdx.x == 0) paged_report(a.status);
  const int64_t all_rows = static_cast<int64_t>(u.seq.n) * a.group;
  u.r0 = static_cast<int64_t>(ru) * 2 * kTile;
  if (u.r0 >= all_rows) return;
  if (u.seq.bad) {
    const int64_t stride = static_cast<int64_t>(row_units) * 2 * kTile;
    for (int64_t r = u.r0; r < all_rows; r += stride)
      for (int i = threadIdx.x; i < 2 * kTile * a.d; i += C::kThreads) {
        const int64_t row = r + i / a.d;
        if (row < all_rows)
          a.out[(u.seq.row0 + row / a.group) * a.out_ld +
                (static_cast<int64_t>(u.hk) * a.group + row % a.group) * a.d + i % a.d] = 0x7FC0u;
      }
    return;
  }
  u.vis_min = paged_visible(u.seq, static_cast<int>(u.r0 / a.group));
  u.vis_max = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t left = all_rows - u.r0 - i * kTile;
    u.rows[i] = static_cast<int>(left < 0 ? 0 : left < kTile ? left : kTile);
    u.steps[i] = 0;
    if (u.rows[i] > 0) {
      const int vis = paged_visible(
          u.seq, static_cast<int>((u.r0 + i * kTile + u.rows[i] - 1) / a.group));
      u.steps[i] = (vis + kTile - 1) / kTile;
      u.vis_max = max(u.vis_max, vis);
    }
  }
  u.n_steps = max(u.steps[0], u.steps[1]);

  // ------------------------------------------------ set-up
  auto bar = [&](const uint64_t& x) { return smem_u32(&x); };
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(bar(sh.full[i]), 1);
      mbar_init(bar(sh.ready[i]), kE4m3 ? 128 : 64);
      mbar_init(bar(sh.empty[i]), 1);
    }
    for (int i = 0; i < C::kRaw; ++i) {
      mbar_init(bar(sh.raw_full[i]), 1);
      mbar_init(bar(sh.raw_empty[i]), 128);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(sh.s_ready[i]), 1);
      mbar_init(bar(sh.p_ready[i]), 128);
      mbar_init(bar(sh.done[i]), 1);
    }
    sh.abort = 0;
    sh.bad_page = 0;
    sh.any_bad = 0;
    fence_mbar_init();
  }
  if (threadIdx.x < kMaxChannels) sh.first_bad[threadIdx.x] = 0x7FFFFFFF;
  if (warp == 8) {
    tmem_alloc(smem_u32(&sh.tmem), 512);
    tmem_relinquish();
  }
  // Q into the swizzled operand tiles: 16 bytes (8 channels) per thread
  {
    constexpr int kChunks = DP / 8;  // per row; a row's threads are neighbours in a warp
    for (int i = threadIdx.x; i < 2 * kTile * kChunks; i += C::kThreads) {
      const int r = i / kChunks, c = i % kChunks;
      const int64_t row = u.r0 + r;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (row < all_rows && 8 * c < a.d)
        x = __ldg(reinterpret_cast<const uint4*>(
            a.q + (u.seq.row0 + row / a.group) * a.q_ld +
            (static_cast<int64_t>(u.hk) * a.group + row % a.group) * a.d + 8 * c));
      if constexpr (kE4m3) {
        uint32_t w[4] = {x.x, x.y, x.z, x.w};
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) top = max(top, max((w[k] << 16) & 0x7FFF0000u, w[k] & 0x7FFF0000u));
#pragma unroll
        for (int o = kChunks / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        float f0, f1;
        const float factor = f16_row_scale(top, a.scale_log2, &f0, &f1);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w[k] = pack_f16(__uint_as_float(w[k] << 16) * f0 * f1,
                           __uint_as_float(w[k] & 0xFFFF0000u) * f0 * f1);
        x = make_uint4(w[0], w[1], w[2], w[3]);
        if (c == 0)
          sh.q_factor[r] = factor;
      }
      const int tile = r / kTile, tr = r % kTile;
      *reinterpret_cast<uint4*>(smem + tile * C::kTileBytes + (c >> 3) * C::kBlockBytes + tr * 128 +
                                (((c & 7) ^ (tr & 7)) << 4)) = x;
    }
  }
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  const uint32_t tm_s[2] = {tmem, tmem + 128}, tm_o[2] = {tmem + 256, tmem + 384};
  int* const status = a.status;
  volatile int* const abort_flag = &sh.abort;
  const int n_items = 2 * u.n_steps;

  if (warp >= 8) {
   regs_dec<C::kOtherRegs>();
   if (warp == 9) {
    // ------------------------------------------------ TMA: K_0 V_0 K_1 V_1 ...
    const int per_tile = kTile >> a.page_log2;  // pages
    const int32_t* table = a.table + static_cast<int64_t>(b) * a.ld_table;
    const int page_size = 1 << a.page_log2;
    int issued = 0;
    for (int it = 0; it < n_items; ++it) {
      const int key0 = (it >> 1) * kTile;
      constexpr int kRing = kE4m3 ? C::kRaw : C::kStages;
      const int st = it % kRing;
      const uint32_t full = kE4m3 ? bar(sh.raw_full[st]) : bar(sh.full[st]);
      const uint32_t empty = kE4m3 ? bar(sh.raw_empty[st]) : bar(sh.empty[st]);
      const int pages = min(per_tile, (u.vis_max - key0 + page_size - 1) >> a.page_log2);
      int page = 0;
      if (lane < pages) {
        page = __ldg(table + (key0 >> a.page_log2) + lane);
        if (page < 0 || page >= a.n_pages) {
          sh.bad_page = 1;  // read page 0 in its place; the rows become NaN
          page = 0;
        }
      }
      if (it >= kRing && !mbar_wait(empty, ((it / kRing) - 1) & 1, status, abort_flag)) break;
      __syncwarp();
      const uint32_t box = static_cast<uint32_t>(page_size) * 128;
      if (lane == 0)
        mbar_arrive_expect_tx(full, static_cast<uint32_t>(pages) *
                                        (kE4m3 ? static_cast<uint32_t>(page_size) * DP
                                               : box * C::kHalves));
      __syncwarp();
      if (lane < pages) {
        const CUtensorMap* map = (it & 1) ? &map_v : &map_k;
        if constexpr (kE4m3) {
          tma_load_4d(s_raw + st * C::kRawBytes + lane * page_size * DP, map, full, 0, 0, u.hk, page);
        } else {
#pragma unroll
          for (int h = 0; h < C::kHalves; ++h)
            tma_load_4d(s_stage + st * C::kTileBytes + h * C::kBlockBytes + lane * box, map, full,
                        64 * h, 0, u.hk, page);
        }
      }
      issued = it + 1;
    }
    // after an abort nobody else waits for the copies in flight
    if (*abort_flag) {
      constexpr int kRing = kE4m3 ? C::kRaw : C::kStages;
      for (int it = max(0, issued - kRing); it < issued; ++it)
        mbar_wait(kE4m3 ? bar(sh.raw_full[it % kRing]) : bar(sh.full[it % kRing]),
                  (it / kRing) & 1, status, nullptr);
    }
  } else if (warp == 8) {
    // ------------------------------------------------ tcgen05.mma
    if (lane == 0) {
      constexpr uint32_t kFormat = kE4m3 ? 0u : (1u << 7) | (1u << 10);  // fp16 or bf16 operands
      const uint32_t idesc_s = (1u << 4) | kFormat | (kTile / 8 << 17) | (kTile / 16 << 24);
      const uint32_t idesc_o = (1u << 4) | kFormat | (1u << 16) |
                               (static_cast<uint32_t>(a.d / 8) << 17) | (kTile / 16 << 24);
      const int k_steps = a.d / 16;
      bool alive = true;
      auto item_ready = [&](int it) {  // an operand tile is in shared memory
        const int st = it % C::kStages;
        const uint32_t parity = (it / C::kStages) & 1;
        // bf16 keys come straight from the TMA, everything else through other warps
        const uint32_t x = !kE4m3 && !(it & 1) ? bar(sh.full[st]) : bar(sh.ready[st]);
        alive = alive && mbar_wait(x, parity, status, abort_flag);
        return alive;
      };
      auto scores = [&](int i, int j) {
        const uint32_t q = base + i * C::kTileBytes;
        const uint32_t k = s_stage + ((2 * j) % C::kStages) * C::kTileBytes;
        for (int s = 0; s < k_steps; ++s) {
          const uint32_t off = (s >> 2) * C::kBlockBytes + (s & 3) * 32;
          mma_ss(tm_s[i], sw128_kmajor_desc(q + off), sw128_kmajor_desc(k + off), idesc_s, s > 0);
        }
        umma_commit(bar(sh.s_ready[i]));
      };
      auto values = [&](int i, int j) {
        const uint32_t v = s_stage + ((2 * j + 1) % C::kStages) * C::kTileBytes;
#pragma unroll
        for (int s = 0; s < kTile / 16; ++s)
          mma_ts(tm_o[i], tm_s[i] + 8 * s, value_desc(v + s * 2048, C::kBlockBytes), idesc_o,
                 j > 0 || s > 0);
      };
      if (u.n_steps > 0 && item_ready(0)) {
        tc_fence_after();
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (u.steps[i] > 0) scores(i, 0);
        umma_commit(bar(sh.empty[0]));
        for (int j = 0; j < u.n_steps && alive; ++j) {
          if (!item_ready(2 * j + 1)) break;
          if (j + 1 < u.n_steps && !item_ready(2 * j + 2)) break;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (j < u.steps[i]) {
              if (!mbar_wait(bar(sh.p_ready[i]), j & 1, status, abort_flag)) { alive = false; break; }
              tc_fence_after();
              values(i, j);
              if (j + 1 == u.steps[i]) umma_commit(bar(sh.done[i]));
            }
            if (i == 1) umma_commit(bar(sh.empty[(2 * j + 1) % C::kStages]));
            if (j + 1 < u.steps[i]) scores(i, j + 1);
          }
          if (alive && j + 1 < u.n_steps) umma_commit(bar(sh.empty[(2 * j + 2) % C::kStages]));
        }
      }
    }
  } else if (!kE4m3 && warp >= 10) {
    // ------------------------------------------------ values that not every row sees
    const int t = threadIdx.x - 320;
    for (int it = 0; it < n_items; ++it) {  // keys too: a stage holds either in turn
      const int st = it % C::kStages, key0 = (it >> 1) * kTile;
      if (!mbar_wait(bar(sh.full[st]), (it / C::kStages) & 1, status, abort_flag)) break;
      if ((it & 1) && key0 + kTile > u.vis_min) {
        uint8_t* v = smem + 2 * C::kTileBytes + st * C::kTileBytes;
        const int first = max(u.vis_min - key0, 0);
        for (int i = t; i < (kTile - first) * C::kHalves * 8; i += 64) {
          const int pc = i & 7, r = first + (i >> 3) / C::kHalves, h = (i >> 3) % C::kHalves;
          uint4* p = reinterpret_cast<uint4*>(v + h * C::kBlockBytes + r * 128 + pc * 16);
          if (key0 + r >= u.vis_max) {
            *p = make_uint4(0, 0, 0, 0);
            continue;
          }
          const uint4 x = *p;
          uint32_t w[4] = {x.x, x.y, x.z, x.w};
          bool found = false;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            found = found || (w[k] & 0x7F80u) == 0x7F80u || (w[k] & 0x7F800000u) == 0x7F800000u;
          if (found) {
            const int ch = h * 64 + ((pc ^ (r & 7)) << 3);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if ((w[k] & 0x7F80u) == 0x7F80u) {
                atomicMin(&sh.first_bad[ch + 2 * k], key0 + r);
                w[k] &= 0xFFFF0000u;
              }
              if ((w[k] & 0x7F800000u) == 0x7F800000u) {
                atomicMin(&sh.first_bad[ch + 2 * k + 1], key0 + r);
                w[k] &= 0x0000FFFFu;
              }
            }
            sh.any_bad = 1;
            *p = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        fence_proxy_async_smem();
      }
      mbar_arrive(bar(sh.ready[st]));
    }
  } else if (kE4m3 && warp >= 12) {
    // ------------------------------------------------ codes to fp16 operand tiles, scales
    const int t = threadIdx.x - 384;
    const int32_t* table = a.table + static_cast<int64_t>(b) * a.ld_table;
    constexpr int kRaw = C::kRaw > 0 ? C::kRaw : 1;
    for (int it = 0; it < n_items; ++it) {
      const int st = it % C::kStages, rs = it % kRaw, j = it >> 1;
      const int key = j * kTile + t;
      // this thread's key's scale; the slot was last read in step j - 4, which is over
      // before the operand stage that this tile goes to is free
      float scale = 0.f;
      if (key < u.vis_max) {
        const int page = __ldg(table + (key >> a.page_log2));
        if (page >= 0 && page < a.n_pages)
          scale = __ldg(((it & 1) ? a.v_scale : a.k_scale) + page * a.ld_scale_page +
                        (static_cast<int64_t>(u.hk) << a.page_log2) + (key & ((1 << a.page_log2) - 1)));
      }
      if (!mbar_wait(bar(sh.raw_full[rs]), (it / kRaw) & 1, status, abort_flag)) break;
      if (it >= C::kStages &&
          !mbar_wait(bar(sh.empty[st]), ((it / C::kStages) - 1) & 1, status, abort_flag))
        break;
      sh.scales[j & 3][it & 1][t] = scale;
      const uint8_t* src = smem + 2 * C::kTileBytes + C::kStages * C::kTileBytes + rs * C::kRawBytes;
      constexpr int kSwizzle = DP == 128 ? 7 : 0;  // of the code tile's 128-byte rows
      uint8_t* dst = smem + 2 * C::kTileBytes + st * C::kTileBytes;
      constexpr int kChunks = DP / 16;  // 16 codes each
#pragma unroll 4
      for (int i = t; i < kTile * kChunks; i += 128) {
        const int r = i / kChunks, c = i % kChunks;
        uint4 x = *reinterpret_cast<const uint4*>(src + r * DP + ((c ^ (r & kSwizzle)) << 4));
        if (j * kTile + r >= u.vis_max) x = make_uint4(0, 0, 0, 0);  // not this sequence's
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
        uint32_t o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
              static_cast<__nv_fp8x2_storage_t>(w[k >> 1] >> (16 * (k & 1))), __NV_E4M3);
          o[k] = static_cast<uint32_t>(h.x) | (static_cast<uint32_t>(h.y) << 16);
        }
        uint8_t* row = dst + (c >> 2) * C::kBlockBytes + r * 128;
        const int c0 = 2 * (c & 3);
        *reinterpret_cast<uint4*>(row + ((c0 ^ (r & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<uint4*>(row + (((c0 + 1) ^ (r & 7)) << 4)) =
            make_uint4(o[4], o[5], o[6], o[7]);
      }
      fence_proxy_async_smem();
      mbar_arrive(bar(sh.raw_empty[rs]));
      mbar_arrive(bar(sh.ready[st]));
    }
   }
  } else {
    regs_inc<C::kSoftmaxRegs>();
    // ------------------------------------------------ softmax: one row per thread
    const int i = warp >> 2;
    const int r = threadIdx.x & 127;
    const uint32_t lanes = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t ts = tm_s[i] + lanes, to = tm_o[i] + lanes;
    const int64_t row = u.r0 + i * kTile + r;
    const bool live = r < u.rows[i];
    const int vis = live ? paged_visible(u.seq, static_cast<int>(row / a.group)) : 0;
    // least visible count in the tile: steps below it need no mask
    const int vis_min = u.rows[i] == kTile
        ? paged_visible(u.seq, static_cast<int>((u.r0 + i * kTile) / a.group)) : 0;
    const float factor = kE4m3 ? sh.q_factor[i * kTile + r] : a.scale_log2;
    float m = -INFINITY, l = 0.f;
    float v_ref = 0.f, v_mul = 0.f;  // power of two at or above the values' scales; kPScale over it
    bool alive = true;
    for (int j = 0; j < u.steps[i]; ++j) {
      if (!mbar_wait(bar(sh.s_ready[i]), j & 1, status, abort_flag)) { alive = false; break; }
      tc_fence_after();
      const int key0 = j * kTile;
      const bool edge = key0 + kTile > vis_min;
      if constexpr (kE4m3) {
        // the step's scales: the values' tile is converted right after the keys'
        if (!mbar_wait(bar(sh.ready[(2 * j + 1) % C::kStages]), ((2 * j + 1) / C::kStages) & 1, status,
                       abort_flag)) { alive = false; break; }
      }
      const float* ks = sh.scales[kE4m3 ? j & 3 : 0][0];
      const float* vs = sh.scales[kE4m3 ? j & 3 : 0][1];
      float s[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32_sync(ts + 32 * c, s[c]);
      if constexpr (kE4m3) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int k = 0; k < 32; k += 4) {
            const float4 x = *reinterpret_cast<const float4*>(ks + 32 * c + k);
            s[c][k] *= x.x; s[c][k + 1] *= x.y; s[c][k + 2] *= x.z; s[c][k + 3] *= x.w;
          }
      }
      if (edge) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (key0 + 32 * c + k >= vis) s[c][k] = -INFINITY;
      }
      float t0 = -INFINITY, t1 = -INFINITY, t2 = -INFINITY, t3 = -INFINITY;
#pragma unroll
      for (int k = 0; k < 32; ++k) {
        t0 = fmaxf(t0, s[0][k]); t1 = fmaxf(t1, s[1][k]);
        t2 = fmaxf(t2, s[2][k]); t3 = fmaxf(t3, s[3][k]);
      }
      const float top = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3)) * factor;
      float v_top = 0.f;
      if constexpr (kE4m3) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v_top = fmaxf(v_top, vs[lane + 32 * k]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v_top = fmaxf(v_top, __shfl_xor_sync(0xFFFFFFFFu, v_top, o));
      }
      const bool move = top > m + kSlack || (m == -INFINITY && top > m) || (kE4m3 && v_top > v_ref);
      if (__any_sync(0xFFFFFFFFu, move)) {
        const float m_new = fmaxf(m, top);
        const float shrink = m == -INFINITY ? 0.f : fast_exp2(m - m_new);
        float shrink_o = shrink;
        if constexpr (kE4m3) {
          if (v_top > v_ref) {  // the next power of two (v_ref is warp-uniform)
            const float up = power_above(v_top);
            shrink_o = v_ref == 0.f ? 0.f : shrink * (v_ref / up);
            v_ref = up;
            v_mul = kPScale / up;
          }
        }
        m = m_new;
        l *= shrink;
        if (j > 0) {
#pragma unroll 1
          for (int c = 0; c < a.d; c += 16) tmem_scale_x16(to + c, shrink_o);
        }
      }
      const float base_m = m == -INFINITY ? 0.f : m;
      float l0 = 0.f, l1 = 0.f;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        uint32_t p[32];
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2)
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            const int c = 2 * hf + c2;
            float p0 = fast_exp2(fmaf(s[c][k], factor, -base_m));
            float p1 = fast_exp2(fmaf(s[c][k + 1], factor, -base_m));
            l0 += p0;
            l1 += p1;
            if constexpr (kE4m3) {
              const float2 x = *reinterpret_cast<const float2*>(vs + 32 * c + k);
              p0 *= x.x * v_mul;
              p1 *= x.y * v_mul;
              if (edge) {  // a masked key's scale may be anything
                if (key0 + 32 * c + k >= vis) p0 = 0.f;
                if (key0 + 32 * c + k + 1 >= vis) p1 = 0.f;
              }
              p[16 * c2 + (k >> 1)] = pack_f16(p0, p1);
            } else {
              p[16 * c2 + (k >> 1)] = pack_bf16(p0, p1);
            }
          }
        tmem_st_x32(ts + 32 * hf, p);
      }
      l += l0 + l1;
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(bar(sh.p_ready[i]));
    }
    if (u.steps[i] > 0 && alive) alive = mbar_wait(bar(sh.done[i]), 0, status, abort_flag);
    tc_fence_after();
    // ---------------------------------------------- out
    const bool nothing = u.steps[i] == 0;
    float inv = l == 0.f ? 0.f : 1.f / l;
    if constexpr (kE4m3) inv *= v_ref / kPScale;
    const bool bad = !alive || sh.bad_page;
    const bool some_bad = !kE4m3 && sh.any_bad;
    uint16_t* dst = a.out + (u.seq.row0 + row / a.group) * a.out_ld +
                    (static_cast<int64_t>(u.hk) * a.group + row % a.group) * a.d;
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) {
      float o[32];
      if (nothing || !alive) {
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = 0.f;
      } else {
        tmem_ld_32x32b_x32_sync(to + 32 * c, o);
      }
      if (live) {
#pragma unroll
        for (int k = 0; k < 32; k += 8) {
          if (32 * c + k < a.d) {
            float x[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              x[q] = o[k + q] * inv;
              // a row without keys has nothing in O
              if (l == 0.f) x[q] = 0.f;
              if (some_bad && sh.first_bad[32 * c + k + q] < vis) x[q] = __uint_as_float(0x7FC00000u);
              if (bad) x[q] = __uint_as_float(0x7FC00000u);
            }
            *reinterpret_cast<uint4*>(dst + 32 * c + k) =
                make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]),
                           pack_bf16(x[6], x[7]));
          }
        }
      }
    }
    if (sh.bad_page && threadIdx.x == 0) paged_report(a.status);
    tc_fence_before();
  }
  __syncwarp();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Once per device: the shared memory limit, and that the launch brings the
// registers that the warps share out among themselves.
template <bool kE4m3, int DP>
cudaError_t configure_mma() {
  using C = MmaCfg<kE4m3, DP>;
  static std::atomic<bool> done[64] = {};
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
  if (dev < 64 && done[dev].load(std::memory_order_acquire)) return cudaSuccess;
  cudaFuncAttributes attr;
  if (cudaError_t e = cudaFuncGetAttributes(&attr, paged_mma_kernel<kE4m3, DP>); e != cudaSuccess)
    return e;
  if (attr.numRegs * C::kThreads <
      256 * C::kSoftmaxRegs + (C::kThreads - 256) * C::kOtherRegs)
    return cudaErrorInvalidConfiguration;
  if (cudaError_t e = cudaFuncSetAttribute(paged_mma_kernel<kE4m3, DP>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
      e != cudaSuccess)
    return e;
  if (dev < 64) done[dev].store(true, std::memory_order_release);
  return cudaSuccess;
}

template <bool kE4m3, int DP>
cudaError_t launch_mma(const PagedArgs& a, cudaStream_t stream) {
  using C = MmaCfg<kE4m3, DP>;
  CUtensorMap mk, mv;
  const int row_bytes = kE4m3 ? DP : 128, page = 1 << a.page_log2;
  if (!make_page_map(&mk, a.k, a, row_bytes, page) || !make_page_map(&mv, a.v, a, row_bytes, page))
    return cudaErrorInvalidValue;
  const int64_t most_rows = static_cast<int64_t>(a.max_q) * a.group;
  const int row_units = static_cast<int>((most_rows + 2 * kTile - 1) / (2 * kTile));
  const int64_t blocks = static_cast<int64_t>(a.B) * a.H_kv * row_units;
  if (blocks > 0x7FFFFFFFll) return cudaErrorInvalidConfiguration;
  if (cudaError_t e = configure_mma<kE4m3, DP>(); e != cudaSuccess) return e;
  paged_mma_kernel<kE4m3, DP>
      <<<static_cast<unsigned>(blocks), C::kThreads, C::kSmem, stream>>>(mk, mv, a, row_units);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_attention_mma(const PagedArgs& a, cudaStream_t stream) {
  const bool e4m3 = a.k_scale != nullptr;
  if (a.d <= 64) return e4m3 ? launch_mma<true, 64>(a, stream) : launch_mma<false, 64>(a, stream);
  return e4m3 ? launch_mma<true, 128>(a, stream) : launch_mma<false, 128>(a, stream);
}

}  // namespace dwa
