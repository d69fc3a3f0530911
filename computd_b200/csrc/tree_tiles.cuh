// tree_tiles.cuh — what the kernels of tree_attention.cu and tree_attention_short.cu share: their
// tcgen05 instructions and descriptors, bounded waits, numbers across lanes, and steps over numbers far apart.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "f32x2.cuh"
#include "paged_attention.cuh"
#include "sm100_ptx.cuh"

namespace dwa {
namespace {

constexpr int kTile = 128;           // keys per step
constexpr int kBlock = kTile * 128;  // bytes of 128 rows of 128 bytes
// Minus the reference of a column that has seen no score yet: any score moves it, but a score of minus infinity
// (from which minus infinity could not be subtracted) keeps the weight 0.
constexpr float kUnset = 0x1.FFFFFEp127f;

__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
// D[tmem] (+)= A[smem] B[smem]^T, by the elected lane of a converged warp
template <bool kF8>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add,
                                       uint32_t one) {
  if constexpr (kF8)
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(one)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(one)
        : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar, uint32_t one) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
      "r"(one)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// Uses of the registers stay behind it.
__device__ __forceinline__ void tmem_wait_x16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
                 "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]),
                 "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ float tmem_ld_x1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr) : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r) : : "memory");
  return __uint_as_float(r);
}
__device__ __forceinline__ void tmem_st_x1(uint32_t taddr, float x) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(__float_as_uint(x)) : "memory");
}

// 16 keys of an operand whose other axis lies along rows of 128 bytes (64 16-bit elements, the
// next 64 kBlock on), a key to a row, 128-byte swizzle.
__device__ __forceinline__ uint64_t by_key_desc(uint32_t addr) {
  uint64_t desc = 0;
  desc |= static_cast<uint64_t>((addr >> 4) & 0x3FFFu);
  desc |= static_cast<uint64_t>((kBlock >> 4) & 0x3FFFu) << 16;  // LBO: 64 elements on
  desc |= static_cast<uint64_t>(1024u >> 4) << 32;               // SBO: 8 keys on
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
// A bounded wait of a whole converged warp, which goes on or gives up together.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int* status, volatile int* abort_flag) {
  constexpr uint32_t kAll = 0xFFFFFFFFu;
  if (__all_sync(kAll, mbar_test(bar, parity))) return true;
  const uint64_t t0 = globaltimer_ns();
  while (true) {
    if (__all_sync(kAll, mbar_try_wait(bar, parity))) return true;
    if (__any_sync(kAll, *abort_flag != 0)) return false;
    if (__any_sync(kAll, globaltimer_ns() - t0 > kWaitLimitNs)) {
      if (status) atomicCAS(status, 0, kStatusTimeout);
      *abort_flag = 1;
      __syncwarp();
      return false;
    }
  }
}
// The same for two at once.
__device__ __forceinline__ bool warp_wait2(uint32_t x, uint32_t parity_x, uint32_t y, uint32_t parity_y, int* status,
                                           volatile int* abort_flag) {
  if (__all_sync(0xFFFFFFFFu, mbar_test(x, parity_x) & mbar_test(y, parity_y))) return true;
  return warp_wait(x, parity_x, status, abort_flag) && warp_wait(y, parity_y, status, abort_flag);
}
// The kThreads threads of a named barrier together; whether any asks.
template <int kThreads>
__device__ __forceinline__ bool group_any(int id, bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
      "barrier.cta.red.or.pred p, %2, %3, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(x)), "r"(id), "n"(kThreads)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void group_sync(int id) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(id) : "memory"); }
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float fast_log2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Numbers by the order of signed integers (NaN above, or below, all).
__device__ __forceinline__ int ordered(float x) {
  const int i = __float_as_int(x);
  return i ^ ((i >> 31) & 0x7FFFFFFF);
}
__device__ __forceinline__ float from_ordered(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7FFFFFFF)); }

// Sixteen columns' values of 32 lanes summed over the lanes: lane l gets column l / 2's.
__device__ __forceinline__ float sum16(float (&v)[16]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int w = 8, o = 16; w >= 1; w >>= 1, o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int k = 0; k < w; ++k) {
      const float send = up ? v[k] : v[k + w], keep = up ? v[k + w] : v[k];
      v[k] = keep + __shfl_xor_sync(0xFFFFFFFFu, send, o);
    }
  }
  return v[0] + __shfl_xor_sync(0xFFFFFFFFu, v[0], 1);
}
// The largest of a warp's numbers (NaN counts for nothing).
__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xFFFFFFFF;" : "=f"(y) : "f"(x));
  return y;
}

// ---------------------------------------------------------------- careful steps
// A step's weights are 2^(S - a) with a reference a that stays unless a score passes a limit, and over an e4m3
// cache times the value's scale over one power of two for all tiles.  That has its range: where scores are 2^kBig
// and more, f32's steps at their size are a good part of 1, and a difference of numbers rounded apart is off by
// them; and a value's scale 2^90 away from the first tile's largest leaves fp16 (that of a vector of zeros, 2^-126, is).  From the first tile with either
// on, a warpgroup's steps of the unit are careful ones:
//   t = S rounded to f32 as a number of its own, b = the column's maximum of t so far,
//   weights 2^(t - b), at most 1, in the sum; in the product, over an e4m3 cache, m 2^((t - b) + e - d), where the
//   value's scale is m 2^e and d follows the largest of (t - b) + e, so that the row's largest is 2^10 at least
//   (and every weight down to 2^-24 of it keeps fp16's 11 bits).
// So O is in units of 2^(b + d).  b and d only meet differences: sums of both would lose d beside a large b.
// (Three passes over the scores, a column at a time: 16 trees of 20 to 32 nodes over 300 to 4096 tokens, 16 heads of 128,
// with scores of 2^24, bf16 97 us instead of 56, e4m3 124 instead of 53.)
constexpr float kBig = 0x1p20f;
constexpr float kLeastUnit = -0x1p100f;  // the exponent d where nothing has any weight

// The sixteen columns of a warpgroup, in shared memory.
struct CarefulColumns {
  float* neg_b;      // minus b
  float* d;          // e4m3
  int* most;         // across keys, ordered; minus infinity between uses
  float* shrink_l;   // of the sums, and of O
  float* shrink_o;
  const float* f;    // e4m3: the scores' factors
};

// The weights of this thread's key in sixteen columns, whose scores are at TMEM column `ts`, into its row of P
// (at columns c0 .. and, bf16, the second parts kApart further) and their sums l.  `to`: O's columns, rescaled
// where they move and have_o says that there are any; the products into them so far are done.  hidden: columns
// that do not see the key.  The 128 threads of named barrier `id` together.
template <bool kE4m3, int kApart>
__device__ __forceinline__ void careful_step(const CarefulColumns& at, int id, uint32_t ts, uint32_t to, bool have_o,
                                             uint32_t hidden, float scale_log2, float sk, float sv, uint8_t* prow, int c0,
                                             uint64_t (&l)[8]) {
  const int t = threadIdx.x & 127, lane = threadIdx.x & 31;
  int exp_v = 0;
  const float m = kE4m3 ? scale_parts(sv, &exp_v) : 1.f;
  const float e_v = static_cast<float>(exp_v);
  auto together = [&]() {
    group_sync(id);
    __syncwarp();
  };
  // (A load of the whole warp: it stands in no branch that threads may take apart.)
  auto score = [&](int e) -> float {
    const float s = tmem_ld_x1(ts + e);
    const float x = kE4m3 ? __fmul_rn(__fmul_rn(s, at.f[e]), sk) : __fmul_rn(s, scale_log2);
    return (hidden >> e) & 1u ? -INFINITY : x;
  };
  // columns' maxima of `value` across the keys, which NaN is not among
  auto maxima = [&](auto&& value) {
    float most = -INFINITY;
#pragma unroll 1
    for (int e = 0; e < 16; ++e) {
      const float largest = warp_max(value(e, score(e)));
      if ((lane & 15) == e) most = largest;
    }
    if (lane < 16 && most == most) atomicMax(&at.most[lane], ordered(most));
    together();
  };
  maxima([](int, float x) -> float { return x; });
  if (t < 16) {
    const float was = -at.neg_b[t], now = fmaxf(was, from_ordered(at.most[t]));
    at.shrink_l[t] = at.shrink_o[t] = fast_exp2(was - now);
    if constexpr (kE4m3) at.d[t] = fmaxf(at.d[t] + (was - now), kLeastUnit);
    at.neg_b[t] = -now;
    at.most[t] = ordered(-INFINITY);
  }
  together();
  if constexpr (kE4m3) {
    maxima([&](int e, float x) -> float { return m != 0.f ? (x + at.neg_b[e]) + e_v : -INFINITY; });
    if (t < 16) {
      const float was = at.d[t], now = fmaxf(was, from_ordered(at.most[t]) - 10.f);
      at.shrink_o[t] = fast_exp2(was - now);
      at.d[t] = now;
      at.most[t] = ordered(-INFINITY);
    }
    together();
  }
  if (have_o) {
#pragma unroll 1
    for (int e = 0; e < 16; ++e) {
      const float by = at.shrink_o[e];
      if (by == 1.f) continue;  // the same for all threads
#pragma unroll
      for (int h = 0; h < (kE4m3 ? 1 : 2); ++h) tmem_st_x1(to + kApart * h + e, tmem_ld_x1(to + kApart * h + e) * by);
    }
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
  }
#pragma unroll 1
  for (int e = 0; e < 16; e += 2) {
    float w[2], p[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float x = score(e + k), rel = x + at.neg_b[e + k];
      w[k] = x == -INFINITY ? 0.f : fast_exp2(rel);
      p[k] = w[k];
      if constexpr (kE4m3) {
        p[k] = fast_exp2((rel + e_v) - at.d[e + k]) * m;
        if (m == 0.f || ((hidden >> (e + k)) & 1u)) p[k] = 0.f;  // d says nothing of the one, the other's scale may be anything
      }
    }
    const uint64_t by = pair(at.shrink_l[e], at.shrink_l[e + 1]), more = pair(w[0], w[1]);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (2 * k == e) l[k] = fma2(l[k], by, more);
    auto put = [&](int c, uint32_t v) {
      *reinterpret_cast<uint32_t*>(prow + (((c >> 3) ^ (t & 7)) << 4) + 2 * (c & 7)) = v;
    };
    if constexpr (kE4m3) {
      put(c0 + e, pack_f16(p[0], p[1]));
    } else {
      const uint32_t hi = pack_bf16(p[0], p[1]);
      put(c0 + e, hi);
      put(kApart + c0 + e,
          pack_bf16(p[0] - __uint_as_float(hi << 16), p[1] - __uint_as_float(hi & 0xFFFF0000u)));
    }
  }
}

}  // namespace
}  // namespace dwa
