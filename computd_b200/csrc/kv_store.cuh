// kv_store.cuh — what the kernels that put keys and values into the paged cache share
// (kv_cache.cu, kv_append.cu): e4m3 codes and their scale, and which of a call's tokens stay
// where slots repeat.
#pragma once

#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "f32x2.cuh"
#include "paged_attention.cuh"

namespace dwa {

// x / b correctly rounded, given y = 1 / b correctly rounded: with q = x y the remainder
// x - q b is exact in an fma, and q + remainder y is the rounded quotient (Markstein,
// 1990), as long as nothing underflows on the way.
__device__ __forceinline__ float quotient(float x, float b, float y) {
  const float q = x * y;
  return fmaf(fmaf(-q, b, x), y, q);
}

__device__ __forceinline__ uint4 codes16(const float (&x)[16]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    u[i] = static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(x[4 * i], x[4 * i + 1]),
                                                          __NV_SATFINITE, __NV_E4M3)) |
           static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + 2], x[4 * i + 3]),
                                                          __NV_SATFINITE, __NV_E4M3)) << 16;
  return make_uint4(u[0], u[1], u[2], u[3]);
}
// The codes of sixteen values of a vector, given its largest magnitude (finite), and its scale.
__device__ __forceinline__ uint4 quantised16(float (&x)[16], float amax, float* scale) {
  // Tiny vectors are scaled up by 2^100, exactly, so that no remainder underflows: amax is
  // above 2^-70 or the scale above 2^-26 then.  (Remainders of quotients above 2^-11 are
  // above 2^-137; smaller quotients give the code 0 either way.)
  float up = 1.f, down = 1.f, least = 0x1p-126f, most = amax;
  if (!(amax > 0x1p-70f)) {
    up = 0x1p100f;
    down = 0x1p-100f;
    least = 0x1p-26f;
    most *= up;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] *= up;
  }
  const float s = fmaxf(quotient(most, 448.f, 1.f / 448.f), least);
  const float y = __frcp_rn(s);
  const uint64_t neg2 = pair(-y, -y), s2 = pair(s, s);
#pragma unroll
  for (int i = 0; i < 16; i += 2) {  // as quotient(), but of -x: so the remainder of a zero, +0, leaves it its sign
    const uint64_t v = pair(x[i], x[i + 1]), q = mul2(v, neg2);
    unpair(fma2(fma2(q, s2, v), neg2, q), x[i], x[i + 1]);
  }
  uint4 w = codes16(x);  // |x / s| <= 448 (1 + 2^-23), which rounds to 448 at most
  w = make_uint4(w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u);
  *scale = s * down;
  return w;
}

constexpr int kFilterBits = 8192;  // a block's slots' low bits

// The slots of a block's tokens t0 .. t0 + n - 1 of T, and which of them are not written: those
// without a slot (-1; any other outside the cache is reported), and those whose slot a later
// token of the launch names, which has to stay whichever block writes first.  The block looks
// the slots after its own up in a filter of its own slots' low bits.  Ends with the block's
// threads together.
template <int kThreads>
__device__ __forceinline__ void settle_slots(const int64_t* slots, int64_t T, int64_t t0, int n, int64_t n_slots,
                                             int64_t* own, int* dropped, uint32_t* filter, int32_t* status) {
  for (int i = threadIdx.x; i < kFilterBits / 32; i += kThreads) filter[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int64_t s = slots[t0 + i];
    const bool fine = s >= 0 && s < n_slots;
    if (!fine && s != -1) paged_report(status);
    own[i] = s;
    dropped[i] = fine ? 0 : 1;
    if (fine) atomicOr(&filter[(s & (kFilterBits - 1)) >> 5], 1u << (s & 31));
  }
  __syncthreads();
  constexpr int kBatch = 8;  // slots that a thread looks at together
  for (int64_t t = t0 + 1 + threadIdx.x; t < T; t += kBatch * kThreads) {
    int64_t s[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      s[j] = t + j * kThreads < T ? __ldg(slots + t + j * kThreads) : -1;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (s[j] >= 0 && ((filter[(s[j] & (kFilterBits - 1)) >> 5] >> (s[j] & 31)) & 1u)) {
        const int before = static_cast<int>(min(t + j * kThreads - t0, static_cast<int64_t>(n)));
        for (int i = 0; i < before; ++i)
          if (own[i] == s[j]) dropped[i] = 1;
      }
    }
  }
  __syncthreads();
}

inline int log2_at_least(int n) {
  int l = 0;
  while ((1 << l) < n) ++l;
  return l;
}

}  // namespace dwa
