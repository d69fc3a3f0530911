// kv_cache.cu — writing new tokens' keys and values into the paged cache
// (bf16, or e4m3 with one f32 scale per (token, head)) and reading them back.
//
// Both are one pass over the data and bound by HBM: per (token, head) vector
// of d values the write reads 2 d bytes (bf16) and writes d + 4, the read the
// reverse.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "dwa_internal.h"
#include "dwa_retrieval.h"

namespace dwa {

namespace {

constexpr int kWriteThreads = 256;
constexpr int kWriteBlocks = 4;    // per SM
constexpr int kGroupTokens = 64;   // tokens of a block checked for repeated slots at a time
constexpr int kFilterBits = 1024;  // their slots' low bits

__device__ __forceinline__ void report(int32_t* status) {
  if (status != nullptr) atomicCAS(status, 0, DWA_ERR_DEVICE_CHECK);
}

// Eight consecutive values of a source row: 16 bytes of bf16, or 32 of f32.
template <bool kBf16>
struct Raw8 {
  uint4 w[kBf16 ? 1 : 2];
};
template <bool kBf16>
__device__ __forceinline__ Raw8<kBf16> load8(const void* row, int64_t at) {
  Raw8<kBf16> r;
  if constexpr (kBf16) {
    r.w[0] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(row) + at));
  } else {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(row) + at);
    r.w[0] = __ldg(p);
    r.w[1] = __ldg(p + 1);
  }
  return r;
}
template <bool kBf16>
__device__ __forceinline__ void as_f32(const Raw8<kBf16>& r, float (&x)[8]) {
  if constexpr (kBf16) {
    const uint32_t u[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x[4 * i] = __uint_as_float(r.w[i].x); x[4 * i + 1] = __uint_as_float(r.w[i].y);
      x[4 * i + 2] = __uint_as_float(r.w[i].z); x[4 * i + 3] = __uint_as_float(r.w[i].w);
    }
  }
}

// Stores the eight values of this lane (of `lanes` lanes that hold one vector).
// Every lane of the warp takes part in the shuffles; `on` says whether it
// holds values, `keep` whether they are stored.
template <bool kE4m3>
__device__ __forceinline__ void store8(const float (&x)[8], bool on, bool keep, int lanes, int lane,
                                       void* cache, float* scales, int64_t row, int64_t srow, int d) {
  if constexpr (!kE4m3) {
    if (on && keep) {
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(cache) + row * d + 8 * lane) =
          make_uint4(u[0], u[1], u[2], u[3]);
    }
    return;
  }
  // The largest magnitude as bits: NaN orders above infinity above every finite number.
  uint32_t top = 0;
  if (on) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  }
  for (int o = lanes >> 1; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  const bool finite = top < 0x7F800000u;
  const float scale = finite ? fmaxf(__fdiv_rn(__uint_as_float(top), 448.f), 0x1p-126f)
                             : __uint_as_float(0x7FC00000u);
  if (!keep) return;
  if (on) {
    // x / scale, |x / scale| <= 448 (1 + 2^-23), which rounds to 448 at most.  One
    // reciprocal for all: with y = 1 / scale rounded, q = x y, the remainder
    // x - q scale is exact in an fma and q + remainder y is the rounded quotient
    // (Markstein, 1990), as long as nothing underflows: scale above 2^-80 and
    // quotients above 2^-11 leave the remainder above 2^-138 (smaller quotients
    // give the code 0 either way).
    float q[8];
    if (scale > 0x1p-80f) {
      const float y = __frcp_rn(scale);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float q0 = x[i] * y;
        q[i] = fmaf(fmaf(-q0, scale, x[i]), y, q0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = finite ? __fdiv_rn(x[i], scale) : 0.f;
    }
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      w[i] = static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(q[4 * i], q[4 * i + 1]),
                                                            __NV_SATFINITE, __NV_E4M3)) |
             static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(
                 make_float2(q[4 * i + 2], q[4 * i + 3]), __NV_SATFINITE, __NV_E4M3)) << 16;
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(cache) + row * d + 8 * lane) =
        make_uint2(w[0], w[1]);
  }
  if (lane == 0) scales[srow] = scale;
}

struct WriteArgs {
  const void *k, *v;
  int64_t T;
  int H, d;
  int64_t k_tok, k_head, v_tok, v_head;
  const int64_t* slots;
  void *k_cache, *v_cache;
  float *k_scale, *v_scale;
  int64_t n_slots;
  int page_log2;
  int64_t ld_page, ld_scale_page;  // in vectors (rows of d) and in scales
  int64_t tokens_per_block;
  int lanes_log2;  // lanes per vector: the power of two >= d / 8
  int32_t* status;
};

// A block owns a run of tokens.  `lanes` neighbouring lanes hold one (token,
// head) vector of K and of V, 8 values each; the amax is a shuffle over them.
// Where slots repeat the last token must stay, whichever block writes first:
// each block drops its tokens whose slot a later token names.  It looks the
// slots after its own up in a filter of its own slots' low bits, so the whole
// list is read once per block (from L2: 19 MB in all for 8192 tokens, against
// the 200 MB of keys and values at 32 heads of 128).
template <bool kE4m3, bool kSrcBf16>
__global__ void __launch_bounds__(kWriteThreads, kWriteBlocks) kv_write_kernel(const WriteArgs a) {
  __shared__ int64_t own[kGroupTokens];
  __shared__ int dropped[kGroupTokens];
  __shared__ uint32_t filter[kFilterBits / 32];

  const int lanes = 1 << a.lanes_log2;
  const int lane = threadIdx.x & (lanes - 1);
  const int group = threadIdx.x >> a.lanes_log2;
  const int groups = kWriteThreads >> a.lanes_log2;
  const bool on = 8 * lane < a.d;
  const int64_t t_end = min((blockIdx.x + 1) * a.tokens_per_block, a.T);
  for (int64_t t0 = blockIdx.x * a.tokens_per_block; t0 < t_end; t0 += kGroupTokens) {
    const int n = static_cast<int>(min(t_end - t0, static_cast<int64_t>(kGroupTokens)));
    const int vectors = n * a.H;
    // a round's values are under way while the round before is stored, the first ones
    // while the slots are checked
    auto load = [&](int vec, Raw8<kSrcBf16>* k, Raw8<kSrcBf16>* v) {
      if (vec < vectors && on) {
        const int i = vec / a.H, h = vec - i * a.H;
        *k = load8<kSrcBf16>(a.k, (t0 + i) * a.k_tok + h * a.k_head + 8 * lane);
        *v = load8<kSrcBf16>(a.v, (t0 + i) * a.v_tok + h * a.v_head + 8 * lane);
      }
    };
    Raw8<kSrcBf16> k_now{}, v_now{};
    load(group, &k_now, &v_now);
    __syncthreads();
    for (int i = threadIdx.x; i < kFilterBits / 32; i += kWriteThreads) filter[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kWriteThreads) {
      const int64_t s = a.slots[t0 + i];
      const bool fine = s >= 0 && s < a.n_slots;
      if (!fine && s != -1) report(a.status);
      own[i] = s;
      dropped[i] = fine ? 0 : 1;
      if (fine) atomicOr(&filter[(s & (kFilterBits - 1)) >> 5], 1u << (s & 31));
    }
    __syncthreads();
    constexpr int kBatch = 8;  // slots that a thread looks at together
    for (int64_t t = t0 + 1 + threadIdx.x; t < a.T; t += kBatch * kWriteThreads) {
      int64_t s[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        s[j] = t + j * kWriteThreads < a.T ? __ldg(a.slots + t + j * kWriteThreads) : -1;
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        if (s[j] >= 0 && ((filter[(s[j] & (kFilterBits - 1)) >> 5] >> (s[j] & 31)) & 1u)) {
          const int before = static_cast<int>(min(t + j * kWriteThreads - t0, static_cast<int64_t>(n)));
          for (int i = 0; i < before; ++i)
            if (own[i] == s[j]) dropped[i] = 1;
        }
      }
    }
    __syncthreads();
    for (int base = 0; base < vectors; base += groups) {
      const int vec = base + group;
      Raw8<kSrcBf16> k_next{}, v_next{};
      load(vec + groups, &k_next, &v_next);
      const bool here = vec < vectors;
      const int i = here ? vec / a.H : 0, h = here ? vec - i * a.H : 0;
      const bool keep = here && !dropped[i];
      const int64_t s = keep ? own[i] : 0;
      const int64_t page = s >> a.page_log2, off = s & ((1 << a.page_log2) - 1);
      const int64_t in_page = (static_cast<int64_t>(h) << a.page_log2) + off;
      const int64_t row = page * a.ld_page + in_page;
      const int64_t srow = page * a.ld_scale_page + in_page;
      float x[8];
      as_f32(k_now, x);
      store8<kE4m3>(x, here && on, keep, lanes, lane, a.k_cache, a.k_scale, row, srow, a.d);
      as_f32(v_now, x);
      store8<kE4m3>(x, here && on, keep, lanes, lane, a.v_cache, a.v_scale, row, srow, a.d);
      k_now = k_next;
      v_now = v_next;
    }
  }
}

struct ReadArgs {
  const void *k_cache, *v_cache;
  const float *k_scale, *v_scale;
  const int64_t* slots;
  int64_t T;
  int H, d;
  int64_t n_slots;
  int page_log2;
  int64_t ld_page, ld_scale_page;
  uint16_t *k_out, *v_out;
  int lanes_log2;  // lanes per vector: the power of two >= d / 16
  int clear_skipped;
  int32_t* status;
};

constexpr int kReadThreads = 256;

// Sixteen values of this lane as bf16: one 16-byte load of codes (or two of
// bf16), two 16-byte stores.
template <bool kE4m3>
__device__ __forceinline__ void read16(const void* cache, const float* scales, int64_t row,
                                       int64_t srow, int d, int lane, bool fine, uint32_t fill,
                                       uint16_t* out) {
  uint32_t o[8];
  if (!fine) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = fill;
  } else if (kE4m3) {
    const uint4 w = __ldg(
        reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(cache) + row * d + 16 * lane));
    const float scale = __ldg(scales + srow);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
          static_cast<__nv_fp8x2_storage_t>(u[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
      const float2 f = __half22float2(__half2(h));
      const __nv_bfloat162 b = __floats2bfloat162_rn(f.x * scale, f.y * scale);
      o[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
  } else {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(cache) + row * d +
                                                    16 * lane);
    const uint4 w = __ldg(p), x = __ldg(p + 1);
    o[0] = w.x; o[1] = w.y; o[2] = w.z; o[3] = w.w;
    o[4] = x.x; o[5] = x.y; o[6] = x.z; o[7] = x.w;
  }
  uint4* dst = reinterpret_cast<uint4*>(out + 16 * lane);
  dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
  dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
}

template <bool kE4m3>
__global__ void __launch_bounds__(kReadThreads) kv_read_kernel(const ReadArgs a) {
  const int lane = threadIdx.x & ((1 << a.lanes_log2) - 1);
  const int64_t vec =
      (static_cast<int64_t>(blockIdx.x) * kReadThreads + threadIdx.x) >> a.lanes_log2;
  if (vec >= a.T * a.H || 16 * lane >= a.d) return;
  const int64_t t = vec / a.H;
  const int h = static_cast<int>(vec - t * a.H);
  const int64_t s = __ldg(a.slots + t);
  const bool skipped = s == -1;
  if (skipped && !a.clear_skipped) return;
  const bool fine = s >= 0 && s < a.n_slots;
  if (!fine && !skipped) report(a.status);
  const uint32_t fill = skipped ? 0u : 0x7FC07FC0u;  // zeros, or NaN for a slot outside the cache
  const int64_t page = s >> a.page_log2, off = s & ((1 << a.page_log2) - 1);
  const int64_t in_page = (static_cast<int64_t>(h) << a.page_log2) + off;
  const int64_t row = page * a.ld_page + in_page, srow = page * a.ld_scale_page + in_page;
  read16<kE4m3>(a.k_cache, a.k_scale, row, srow, a.d, lane, fine, fill, a.k_out + vec * a.d);
  read16<kE4m3>(a.v_cache, a.v_scale, row, srow, a.d, lane, fine, fill, a.v_out + vec * a.d);
}

int log2_at_least(int n) {
  int l = 0;
  while ((1 << l) < n) ++l;
  return l;
}

}  // namespace

cudaError_t launch_kv_write(const KvCacheView& c, const void* k, const void* v, int src_bf16,
                            int64_t T, int64_t k_tok, int64_t k_head, int64_t v_tok, int64_t v_head,
                            const int64_t* slots, int32_t* status, cudaStream_t stream) {
  WriteArgs a{};
  a.k = k; a.v = v; a.T = T; a.H = c.H; a.d = c.d;
  a.k_tok = k_tok; a.k_head = k_head; a.v_tok = v_tok; a.v_head = v_head;
  a.slots = slots;
  a.k_cache = const_cast<void*>(c.k); a.v_cache = const_cast<void*>(c.v);
  a.k_scale = const_cast<float*>(c.k_scale); a.v_scale = const_cast<float*>(c.v_scale);
  a.page_log2 = log2_at_least(c.page_size);
  a.n_slots = c.n_pages << a.page_log2;
  a.ld_page = c.ld_page / c.d; a.ld_scale_page = c.ld_scale_page;
  a.lanes_log2 = log2_at_least(c.d / 8);
  a.status = status;
  const int64_t most = static_cast<int64_t>(kWriteBlocks) * device_sm_count();
  a.tokens_per_block = (T + most - 1) / most;
  const unsigned grid = static_cast<unsigned>((T + a.tokens_per_block - 1) / a.tokens_per_block);
  if (c.k_scale != nullptr) {
    if (src_bf16) kv_write_kernel<true, true><<<grid, kWriteThreads, 0, stream>>>(a);
    else kv_write_kernel<true, false><<<grid, kWriteThreads, 0, stream>>>(a);
  } else {
    if (src_bf16) kv_write_kernel<false, true><<<grid, kWriteThreads, 0, stream>>>(a);
    else kv_write_kernel<false, false><<<grid, kWriteThreads, 0, stream>>>(a);
  }
  return cudaGetLastError();
}

cudaError_t launch_kv_read(const KvCacheView& c, const int64_t* slots, int64_t T, void* k_out,
                           void* v_out, int clear_skipped, int32_t* status, cudaStream_t stream) {
  ReadArgs a{};
  a.k_cache = c.k; a.v_cache = c.v; a.k_scale = c.k_scale; a.v_scale = c.v_scale;
  a.slots = slots; a.T = T; a.H = c.H; a.d = c.d;
  a.page_log2 = log2_at_least(c.page_size);
  a.n_slots = c.n_pages << a.page_log2;
  a.ld_page = c.ld_page / c.d; a.ld_scale_page = c.ld_scale_page;
  a.k_out = static_cast<uint16_t*>(k_out); a.v_out = static_cast<uint16_t*>(v_out);
  a.lanes_log2 = log2_at_least(c.d / 16);
  a.clear_skipped = clear_skipped;
  a.status = status;
  const int64_t per_block = kReadThreads >> a.lanes_log2;
  const unsigned grid = static_cast<unsigned>((T * c.H + per_block - 1) / per_block);
  if (c.k_scale != nullptr) kv_read_kernel<true><<<grid, kReadThreads, 0, stream>>>(a);
  else kv_read_kernel<false><<<grid, kReadThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace dwa
