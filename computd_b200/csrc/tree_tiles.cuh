// tree_tiles.cuh — what the kernels of tree_attention.cu and tree_attention_short.cu share: their
// tcgen05 instructions and descriptors, bounded waits, and numbers across lanes.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

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

}  // namespace
}  // namespace dwa
