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
#include "kv_store.cuh"
#include "paged_attention.cuh"

namespace dwa {

namespace {

constexpr int kWriteThreads = 256;
// Blocks per SM: bf16 into a bf16 cache (8191 tokens, 32 heads of 128: 55, 50, 50.5 us with 3,
// 4, 5), into codes (39.9, 42.3, 62.8), and f32 (with 1, 2, 3 into codes 83, 61, 67, into bf16
// 116, 77, 69).
template <bool kE4m3, bool kSrcBf16>
constexpr int kWriteBlocks = !kSrcBf16 ? 2 : kE4m3 ? 3 : 4;
constexpr int kBlockTokens = 32;  // at most; a longer call is cut into launches

// Values of a lane: sixteen make 16 bytes of codes, eight 16 bytes of bf16.
template <bool kE4m3>
constexpr int kLaneValues = kE4m3 ? 16 : 8;

// kN consecutive values of a source row.
template <bool kBf16, int kN>
struct Raw {
  uint4 w[kN / (kBf16 ? 8 : 4)];
};
template <bool kBf16, int kN>
__device__ __forceinline__ Raw<kBf16, kN> load_raw(const void* row, int64_t at) {
  Raw<kBf16, kN> r;
  const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(row) + at * (kBf16 ? 2 : 4));
#pragma unroll
  for (int i = 0; i < kN / (kBf16 ? 8 : 4); ++i) r.w[i] = __ldg(p + i);
  return r;
}
template <bool kBf16, int kN>
__device__ __forceinline__ void as_f32(const Raw<kBf16, kN>& r, float (&x)[kN]) {
#pragma unroll
  for (int i = 0; i < kN / (kBf16 ? 8 : 4); ++i) {
    const uint32_t u[4] = {r.w[i].x, r.w[i].y, r.w[i].z, r.w[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (kBf16) {
        x[8 * i + 2 * j] = __uint_as_float(u[j] << 16);
        x[8 * i + 2 * j + 1] = __uint_as_float(u[j] & 0xFFFF0000u);
      } else {
        x[4 * i + j] = __uint_as_float(u[j]);
      }
    }
  }
}

// Stores the eight values of this lane, rounded to bf16.
template <bool kBf16>
__device__ __forceinline__ void store_bf16(const Raw<kBf16, 8>& raw, uint16_t* dst) {
  if constexpr (kBf16) {
    *reinterpret_cast<uint4*>(dst) = raw.w[0];
  } else {
    float x[8];
    as_f32(raw, x);
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(dst) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}
// Stores the sixteen values of this lane (of `lanes` lanes that hold one vector) as codes.
// Every lane of the warp takes part in the shuffles; `on` says whether it
// holds values, `keep` whether they are stored.
template <bool kBf16>
__device__ __forceinline__ void store_e4m3(const Raw<kBf16, 16>& raw, bool on, bool keep, int lanes, int lane,
                                           uint8_t* cache, float* scales, int64_t row, int64_t srow, int d) {
  // The largest magnitude as bits: NaN orders above infinity above every finite number.
  uint32_t top = 0;
  if (on) {
    if constexpr (kBf16) {  // of both halves at once
      uint32_t tops = 0;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        tops = __vmaxu2(__vmaxu2(tops, __vmaxu2(raw.w[i].x & 0x7FFF7FFFu, raw.w[i].y & 0x7FFF7FFFu)),
                        __vmaxu2(raw.w[i].z & 0x7FFF7FFFu, raw.w[i].w & 0x7FFF7FFFu));
      top = max(tops << 16, tops & 0xFFFF0000u);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        top = max(max(top, max(raw.w[i].x & 0x7FFFFFFFu, raw.w[i].y & 0x7FFFFFFFu)),
                  max(raw.w[i].z & 0x7FFFFFFFu, raw.w[i].w & 0x7FFFFFFFu));
    }
  }
  for (int o = lanes >> 1; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  if (!keep) return;
  const float amax = __uint_as_float(top);
  const bool finite = top < 0x7F800000u;
  uint4 w = make_uint4(0, 0, 0, 0);
  float scale = __uint_as_float(0x7FC00000u);
  if (finite) {
    float x[16];
    as_f32(raw, x);
    w = quantised16(x, amax, &scale);
  }
  if (on) *reinterpret_cast<uint4*>(cache + row * d + 16 * lane) = w;
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
  int lanes_log2;  // lanes per vector: the power of two >= d / (values of a lane)
  int32_t* status;
};

// A block owns a run of tokens.  `lanes` neighbouring lanes hold one (token,
// head) vector of K and of V; the amax is a shuffle over them.
// Where slots repeat the last token must stay, whichever block writes first:
// each block drops its tokens whose slot a later token of the launch names.  It looks
// the slots after its own up in a filter of its own slots' low bits, so a launch's list
// is read once per block (from L2: 19 MB in all for 8192 tokens, against the 200 MB of
// keys and values at 32 heads of 128).  More tokens than the resident blocks take, 14,208 from
// bf16 to codes, are cut into launches, which the stream orders, so that time and looks grow
// as the tokens do: 1,000,000 tokens of 8 heads of 128 take 2.6 ms (with 16, 64, 128 tokens per
// block 2.6, 3.9, 8.3; in one launch 169), 20,000 47 us (50, 55, 55; 57).
template <bool kE4m3, bool kSrcBf16>
__global__ void __launch_bounds__(kWriteThreads, kWriteBlocks<kE4m3, kSrcBf16>)
    kv_write_kernel(const WriteArgs a) {
  __shared__ int64_t own[kBlockTokens];
  __shared__ int dropped[kBlockTokens];
  __shared__ uint32_t filter[kFilterBits / 32];

  const int lanes = 1 << a.lanes_log2;
  const int lane = threadIdx.x & (lanes - 1);
  const int group = threadIdx.x >> a.lanes_log2;
  const int groups = kWriteThreads >> a.lanes_log2;
  constexpr int kN = kLaneValues<kE4m3>;
  using Values = Raw<kSrcBf16, kN>;
  const bool on = kN * lane < a.d;
  const int64_t t0 = blockIdx.x * a.tokens_per_block;
  const int n = static_cast<int>(min(a.T - t0, a.tokens_per_block));
  const int vectors = n * a.H;
  // a round's values are under way while the round before is stored, the first ones
  // while the slots are checked
  auto load = [&](int i, int h, Values* k, Values* v) {
    if (i < n && on) {
      *k = load_raw<kSrcBf16, kN>(a.k, (t0 + i) * a.k_tok + h * a.k_head + kN * lane);
      *v = load_raw<kSrcBf16, kN>(a.v, (t0 + i) * a.v_tok + h * a.v_head + kN * lane);
    }
  };
  auto forward = [&](int* i, int* h) {  // to this group's next vector
    *h += groups;
    while (*h >= a.H) {
      *h -= a.H;
      ++*i;
    }
  };
  Values k_now{}, v_now{};
  int i_now = group / a.H, h_now = group % a.H;
  load(i_now, h_now, &k_now, &v_now);
  settle_slots<kWriteThreads>(a.slots, a.T, t0, n, a.n_slots, own, dropped, filter, a.status);
  for (int base = 0; base < vectors; base += groups) {
    int i_next = i_now, h_next = h_now;
    forward(&i_next, &h_next);
    Values k_next{}, v_next{};
    load(i_next, h_next, &k_next, &v_next);
    const bool here = i_now < n;
    const bool keep = here && !dropped[here ? i_now : 0];
    const int64_t s = keep ? own[i_now] : 0;
    const int64_t page = s >> a.page_log2, off = s & ((1 << a.page_log2) - 1);
    const int64_t in_page = (static_cast<int64_t>(h_now) << a.page_log2) + off;
    const int64_t row = page * a.ld_page + in_page;
    const int64_t srow = page * a.ld_scale_page + in_page;
    if constexpr (kE4m3) {
      store_e4m3(k_now, here && on, keep, lanes, lane, static_cast<uint8_t*>(a.k_cache), a.k_scale, row, srow, a.d);
      store_e4m3(v_now, here && on, keep, lanes, lane, static_cast<uint8_t*>(a.v_cache), a.v_scale, row, srow, a.d);
    } else if (on && keep) {
      store_bf16(k_now, static_cast<uint16_t*>(a.k_cache) + row * a.d + kN * lane);
      store_bf16(v_now, static_cast<uint16_t*>(a.v_cache) + row * a.d + kN * lane);
    }
    k_now = k_next;
    v_now = v_next;
    i_now = i_next;
    h_now = h_next;
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
  int lanes_log2;  // lanes per vector: the power of two >= d / 8
  int clear_skipped;
  int32_t* status;
};

constexpr int kReadThreads = 256;

constexpr int kReadVectors = 2;

// Eight values of a lane on their way: 8 bytes of codes and their scale, or 16 bytes of
// bf16.  (With sixteen a lane's two stores left half a sector each: twice the writes to
// L2, 82 us instead of 69 for 16384 tokens of 32 heads.)
template <bool kE4m3>
struct Held8 {
  uint4 w;
  float scale;
};
template <bool kE4m3>
__device__ __forceinline__ Held8<kE4m3> fetch8(const void* cache, const float* scales, int64_t row,
                                               int64_t srow, int d, int lane) {
  Held8<kE4m3> x;
  const char* p = static_cast<const char*>(cache) + (row * d + 8 * lane) * (kE4m3 ? 1 : 2);
  if constexpr (kE4m3) {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
    x.w = make_uint4(w.x, w.y, 0, 0);
    x.scale = __ldg(scales + srow);
  } else {
    x.w = __ldg(reinterpret_cast<const uint4*>(p));
  }
  return x;
}
// One 16-byte store of bf16; streaming, since the reader goes through it once.
template <bool kE4m3>
__device__ __forceinline__ void put8(const Held8<kE4m3>& x, uint16_t* out) {
  uint4 o = x.w;
  if constexpr (kE4m3) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
          static_cast<__nv_fp8x2_storage_t>((i < 2 ? x.w.x : x.w.y) >> (16 * (i & 1))), __NV_E4M3);
      const float2 f = __half22float2(__half2(h));
      const __nv_bfloat162 b = __floats2bfloat162_rn(f.x * x.scale, f.y * x.scale);
      r[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    o = make_uint4(r[0], r[1], r[2], r[3]);
  }
  __stcs(reinterpret_cast<uint4*>(out), o);
}

// A group of lanes brings kReadVectors (token, head) vectors of K and of V, a block's
// groups neighbouring ones at a time; all its loads are under way before the first store.
template <bool kE4m3>
__global__ void __launch_bounds__(kReadThreads) kv_read_kernel(const ReadArgs a) {
  const int lane = threadIdx.x & ((1 << a.lanes_log2) - 1);
  const int groups = kReadThreads >> a.lanes_log2;
  if (8 * lane >= a.d) return;
  const int64_t vectors = a.T * a.H;
  const int64_t vec0 = static_cast<int64_t>(blockIdx.x) * groups * kReadVectors + (threadIdx.x >> a.lanes_log2);
  int64_t s[kReadVectors];
  int h[kReadVectors];
#pragma unroll
  for (int i = 0; i < kReadVectors; ++i) {
    const int64_t vec = vec0 + static_cast<int64_t>(i) * groups;
    const int64_t t = vec / a.H;
    h[i] = static_cast<int>(vec - t * a.H);
    s[i] = vec < vectors ? __ldg(a.slots + t) : -1;
  }
  Held8<kE4m3> k[kReadVectors], v[kReadVectors];
#pragma unroll
  for (int i = 0; i < kReadVectors; ++i) {
    if (s[i] >= 0 && s[i] < a.n_slots) {
      const int64_t page = s[i] >> a.page_log2, off = s[i] & ((1 << a.page_log2) - 1);
      const int64_t in_page = (static_cast<int64_t>(h[i]) << a.page_log2) + off;
      const int64_t row = page * a.ld_page + in_page, srow = page * a.ld_scale_page + in_page;
      k[i] = fetch8<kE4m3>(a.k_cache, a.k_scale, row, srow, a.d, lane);
      v[i] = fetch8<kE4m3>(a.v_cache, a.v_scale, row, srow, a.d, lane);
    }
  }
#pragma unroll
  for (int i = 0; i < kReadVectors; ++i) {
    const int64_t vec = vec0 + static_cast<int64_t>(i) * groups;
    const bool skipped = s[i] == -1;
    if (vec >= vectors || (skipped && !a.clear_skipped)) continue;
    uint16_t* k_out = a.k_out + vec * a.d + 8 * lane;
    uint16_t* v_out = a.v_out + vec * a.d + 8 * lane;
    if (s[i] >= 0 && s[i] < a.n_slots) {
      put8<kE4m3>(k[i], k_out);
      put8<kE4m3>(v[i], v_out);
    } else {
      if (!skipped) paged_report(a.status);
      const uint32_t fill = skipped ? 0u : 0x7FC07FC0u;  // zeros, or NaN for a slot outside the cache
      *reinterpret_cast<uint4*>(k_out) = make_uint4(fill, fill, fill, fill);
      *reinterpret_cast<uint4*>(v_out) = make_uint4(fill, fill, fill, fill);
    }
  }
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
  a.lanes_log2 = log2_at_least(c.d / (c.k_scale != nullptr ? kLaneValues<true> : kLaneValues<false>));
  a.status = status;
  const bool e4m3 = c.k_scale != nullptr;
  const int per_sm = e4m3 ? (src_bf16 ? kWriteBlocks<true, true> : kWriteBlocks<true, false>)
                          : (src_bf16 ? kWriteBlocks<false, true> : kWriteBlocks<false, false>);
  const int64_t most = static_cast<int64_t>(per_sm) * device_sm_count();
  const int64_t launches = (T + most * kBlockTokens - 1) / (most * kBlockTokens);
  const int64_t share = (T + launches - 1) / launches;  // tokens of one
  const int64_t es = src_bf16 ? 2 : 4;
  for (int64_t t = 0; t < T; t += share) {
    a.T = std::min(share, T - t);
    a.k = static_cast<const char*>(k) + t * k_tok * es;
    a.v = static_cast<const char*>(v) + t * v_tok * es;
    a.slots = slots + t;
    a.tokens_per_block = (a.T + most - 1) / most;
    const unsigned grid = static_cast<unsigned>((a.T + a.tokens_per_block - 1) / a.tokens_per_block);
    if (e4m3) {
      if (src_bf16) kv_write_kernel<true, true><<<grid, kWriteThreads, 0, stream>>>(a);
      else kv_write_kernel<true, false><<<grid, kWriteThreads, 0, stream>>>(a);
    } else {
      if (src_bf16) kv_write_kernel<false, true><<<grid, kWriteThreads, 0, stream>>>(a);
      else kv_write_kernel<false, false><<<grid, kWriteThreads, 0, stream>>>(a);
    }
    if (cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  }
  return cudaSuccess;
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
  a.lanes_log2 = log2_at_least(c.d / 8);
  a.clear_skipped = clear_skipped;
  a.status = status;
  const int64_t per_block = (kReadThreads >> a.lanes_log2) * kReadVectors;
  const unsigned grid = static_cast<unsigned>((T * c.H + per_block - 1) / per_block);
  if (c.k_scale != nullptr) kv_read_kernel<true><<<grid, kReadThreads, 0, stream>>>(a);
  else kv_read_kernel<false><<<grid, kReadThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace dwa
