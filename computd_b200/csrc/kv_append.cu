// kv_append.cu — new tokens' queries and keys rotated for their positions, and keys and
// values put into the paged cache, in one pass.
//
// For x1 = x[0::2], x2 = x[1::2] and the token's row of the tables the rotated vector is
// [x1 cos - x2 sin, x1 sin + x2 cos].  bf16 tensors with bf16 tables round every product,
// sum and difference to bf16, so that the result is rope_qk's (lm_ops.cu) followed by
// kv_write's (kv_cache.cu) bit for bit.  Otherwise all is f32, with the second product's rounding
// error carried along (two more operations an output), so that an output whose products nearly
// cancel keeps its bits, and is rounded once where it is stored: to bf16, or relative to the
// vector's scale to e4m3.
//
// Bound by HBM: per token, d (2 (H + 2 H_kv) + 2 H) bytes and the cache's 4 d H_kv or
// 2 (d + 4) H_kv.  Apart, the two passes move the keys twice more, and the queries' pass knows no
// far positions but through a gathered copy of the tables.  8191 tokens, 32 over 8 heads of 128, bf16 with f32
// tables: 50 us, 4.1 TB/s, with the issue slots 58 % full and loads the longest stall; 64 tokens of 16 heads of
// 80 into an 8-bit cache 3.9 us, launch and one chain of loads.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "dwa_internal.h"
#include "kv_store.cuh"
#include "paged_attention.cuh"

namespace dwa {

namespace {

constexpr int kThreads = 256;
// Blocks per SM, which decide how many loads are under way: bf16 into a bf16 cache 2, 3, 4 (8191 tokens, 32 over 8 heads
// of 128: 69, 54, 50 us); codes and f32 need the registers.
template <bool kE4m3, bool kSrcBf16>
constexpr int kBlocks = !kSrcBf16 ? 2 : kE4m3 ? 3 : 4;
constexpr int kBlockTokens = 32;  // at most; a longer call is cut into launches

// Sixteen neighbouring values of a row.
template <bool kBf16>
struct Raw16 {
  uint4 w[kBf16 ? 2 : 4];
};
template <bool kBf16>
__device__ __forceinline__ Raw16<kBf16> load16(const void* base, int64_t at) {
  Raw16<kBf16> r;
  const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(base) + at * (kBf16 ? 2 : 4));
#pragma unroll
  for (int i = 0; i < (kBf16 ? 2 : 4); ++i) r.w[i] = __ldg(p + i);
  return r;
}
__device__ __forceinline__ void bf16x8(const uint4& w, float* x) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = __uint_as_float(u[j] << 16);
    x[2 * j + 1] = __uint_as_float(u[j] & 0xFFFF0000u);
  }
}
template <bool kBf16>
__device__ __forceinline__ void widen(const Raw16<kBf16>& r, float (&x)[16]) {
  if constexpr (kBf16) {
    bf16x8(r.w[0], x);
    bf16x8(r.w[1], x + 8);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[4 * i] = __uint_as_float(r.w[i].x);
      x[4 * i + 1] = __uint_as_float(r.w[i].y);
      x[4 * i + 2] = __uint_as_float(r.w[i].z);
      x[4 * i + 3] = __uint_as_float(r.w[i].w);
    }
  }
}

__device__ __forceinline__ float to_bf16(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }

// a b + c d, with c d's rounding error carried along.
__device__ __forceinline__ float two_products(float a, float b, float c, float d) {
  const float p = c * d;
  const float lost = fmaf(c, d, -p);
  const float r = fmaf(a, b, p);
  const float y = r + lost;
  return y == y ? y : r;  // an infinite product has no error to speak of
}

struct AppendArgs {
  const void *q, *k, *v;
  int64_t T;
  int H, H_kv, d;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;
  const void *cos, *sin;
  int64_t ld_table, n_positions;
  const int64_t* positions;  // null: a token's own number, from t_first on
  int64_t t_first;
  const int64_t* slots;
  void *k_cache, *v_cache;
  float *k_scale, *v_scale;
  int64_t n_slots;
  int page_log2;
  int64_t ld_page, ld_scale_page;  // in vectors (rows of d) and in scales
  uint16_t* q_out;
  int tokens_per_block, parts;  // blocks that share a run of tokens' vectors
  int lanes_log2;               // lanes per vector: the power of two >= d / 16
  int32_t* status;
};

// `lanes` neighbouring lanes hold one vector, sixteen values each; a block's groups go through
// the vectors of its tokens (token by token: queries, keys, values), a round's values under way
// while the round before is stored.
template <bool kE4m3, bool kSrcBf16, bool kTabBf16>
__global__ void __launch_bounds__(kThreads, kBlocks<kE4m3, kSrcBf16>) kv_append_kernel(const AppendArgs a) {
  __shared__ int64_t own[kBlockTokens];
  __shared__ int dropped[kBlockTokens];
  __shared__ uint32_t filter[kFilterBits / 32];

  const int lanes = 1 << a.lanes_log2;
  const int lane = threadIdx.x & (lanes - 1);
  const int groups = kThreads >> a.lanes_log2;
  const bool on = 16 * lane < a.d;
  const int run = static_cast<int>(blockIdx.x) / a.parts, part = static_cast<int>(blockIdx.x) % a.parts;
  const int64_t t0 = static_cast<int64_t>(run) * a.tokens_per_block;
  const int n = static_cast<int>(min(a.T - t0, static_cast<int64_t>(a.tokens_per_block)));
  const int per_token = a.H + 2 * a.H_kv;
  const int vectors = n * per_token;
  const int share = (vectors + a.parts - 1) / a.parts;
  const int first = part * share, last = min(first + share, vectors);

  int at = first + (threadIdx.x >> a.lanes_log2);  // this group's vector: j of token i
  int i = at / per_token, j = at - i * per_token;
  using Values = Raw16<kSrcBf16>;
  auto load = [&](int at, int i, int j) -> Values {
    Values x{};
    if (at < last && on) {
      const int64_t t = t0 + i;
      if (j < a.H) x = load16<kSrcBf16>(a.q, t * a.q_tok + j * a.q_head + 16 * lane);
      else if (j < a.H + a.H_kv) x = load16<kSrcBf16>(a.k, t * a.k_tok + (j - a.H) * a.k_head + 16 * lane);
      else x = load16<kSrcBf16>(a.v, t * a.v_tok + (j - a.H - a.H_kv) * a.v_head + 16 * lane);
    }
    return x;
  };
  Values now = load(at, i, j);
  settle_slots<kThreads>(a.slots, a.T, t0, n, a.n_slots, own, dropped, filter, a.status);

  float c[8], s[8];  // of token `held`, this lane's eight rotations
  int held = -1;
  for (int base = first; base < last; base += groups) {
    const int next_at = at + groups;
    int next_i = i, next_j = j + groups;
    while (next_j >= per_token) {
      next_j -= per_token;
      ++next_i;
    }
    const Values next = load(next_at, next_i, next_j);
    const bool here = at < last, turn = j < a.H + a.H_kv, query = j < a.H;
    float x[16];
    widen<kSrcBf16>(now, x);
    if (here && on && turn) {
      if (held != i) {
        held = i;
        const int64_t t = t0 + i;
        const int64_t pos = a.positions != nullptr ? __ldg(a.positions + t) : a.t_first + t;
        if (pos >= 0 && pos < a.n_positions) {
          const int64_t row = pos * a.ld_table + 8 * lane;
          if constexpr (kTabBf16) {
            bf16x8(__ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.cos) + row)), c);
            bf16x8(__ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.sin) + row)), s);
          } else {
            const float4* pc = reinterpret_cast<const float4*>(static_cast<const float*>(a.cos) + row);
            const float4* ps = reinterpret_cast<const float4*>(static_cast<const float*>(a.sin) + row);
            const float4 c0 = __ldg(pc), c1 = __ldg(pc + 1), s0 = __ldg(ps), s1 = __ldg(ps + 1);
            c[0] = c0.x; c[1] = c0.y; c[2] = c0.z; c[3] = c0.w;
            c[4] = c1.x; c[5] = c1.y; c[6] = c1.z; c[7] = c1.w;
            s[0] = s0.x; s[1] = s0.y; s[2] = s0.z; s[3] = s0.w;
            s[4] = s1.x; s[5] = s1.y; s[6] = s1.z; s[7] = s1.w;
          }
        } else {
          paged_report(a.status);
#pragma unroll
          for (int e = 0; e < 8; ++e) c[e] = s[e] = __uint_as_float(0x7FC00000u);
        }
      }
      float y[16];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x1 = x[2 * e], x2 = x[2 * e + 1];
        if constexpr (kSrcBf16 && kTabBf16) {
          y[e] = to_bf16(to_bf16(x1 * c[e]) - to_bf16(x2 * s[e]));
          y[8 + e] = to_bf16(to_bf16(x1 * s[e]) + to_bf16(x2 * c[e]));
        } else {
          y[e] = two_products(x1, c[e], -x2, s[e]);
          y[8 + e] = two_products(x1, s[e], x2, c[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = y[e];
    }
    // where the two runs of eight belong
    const int to0 = turn ? 8 * lane : 16 * lane, to1 = turn ? (a.d >> 1) + 8 * lane : 16 * lane + 8;
    const bool keep = here && !query && !dropped[here ? i : 0];
    const int64_t slot = keep ? own[i] : 0;
    const int64_t page = slot >> a.page_log2, off = slot & ((1 << a.page_log2) - 1);
    const int64_t in_page = (static_cast<int64_t>(turn ? j - a.H : j - a.H - a.H_kv) << a.page_log2) + off;
    const int64_t row = page * a.ld_page + in_page;
    if constexpr (kE4m3) {
      uint32_t top = 0;
      if (here && on && !query)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(x[e]) & 0x7FFFFFFFu);
      for (int o = lanes >> 1; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
      if (keep) {
        uint4 w = make_uint4(0, 0, 0, 0);
        float scale = __uint_as_float(0x7FC00000u);
        if (top < 0x7F800000u) w = quantised16(x, __uint_as_float(top), &scale);
        if (on) {
          uint8_t* cache = static_cast<uint8_t*>(turn ? a.k_cache : a.v_cache) + row * a.d;
          *reinterpret_cast<uint2*>(cache + to0) = make_uint2(w.x, w.y);
          *reinterpret_cast<uint2*>(cache + to1) = make_uint2(w.z, w.w);
        }
        if (lane == 0) (turn ? a.k_scale : a.v_scale)[page * a.ld_scale_page + in_page] = scale;
      }
    }
    if (on && (kE4m3 ? here && query : (here && query) || keep)) {
      uint16_t* dst = query ? a.q_out + ((t0 + i) * a.H + j) * a.d
                            : static_cast<uint16_t*>(turn ? a.k_cache : a.v_cache) + row * a.d;
      uint32_t u[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] = pack_bf16(x[2 * e], x[2 * e + 1]);
      *reinterpret_cast<uint4*>(dst + to0) = make_uint4(u[0], u[1], u[2], u[3]);
      *reinterpret_cast<uint4*>(dst + to1) = make_uint4(u[4], u[5], u[6], u[7]);
    }
    now = next;
    at = next_at;
    i = next_i;
    j = next_j;
  }
}

template <bool kE4m3, bool kSrcBf16>
void launch_one(const AppendArgs& a, bool tables_bf16, unsigned grid, cudaStream_t stream) {
  if (tables_bf16) kv_append_kernel<kE4m3, kSrcBf16, true><<<grid, kThreads, 0, stream>>>(a);
  else kv_append_kernel<kE4m3, kSrcBf16, false><<<grid, kThreads, 0, stream>>>(a);
}

}  // namespace

cudaError_t launch_kv_append(const KvCacheView& c, const KvAppendView& x, int64_t T, const int64_t* slots,
                             int32_t* status, cudaStream_t stream) {
  AppendArgs a{};
  a.q = x.q; a.k = x.k; a.v = x.v;
  a.H = x.q != nullptr ? x.H : 0; a.H_kv = c.H; a.d = c.d;
  a.q_tok = x.q_tok; a.q_head = x.q_head; a.k_tok = x.k_tok; a.k_head = x.k_head;
  a.v_tok = x.v_tok; a.v_head = x.v_head;
  a.cos = x.cos; a.sin = x.sin; a.ld_table = x.ld_table; a.n_positions = x.n_positions;
  a.k_cache = const_cast<void*>(c.k); a.v_cache = const_cast<void*>(c.v);
  a.k_scale = const_cast<float*>(c.k_scale); a.v_scale = const_cast<float*>(c.v_scale);
  a.page_log2 = log2_at_least(c.page_size);
  a.n_slots = c.n_pages << a.page_log2;
  a.ld_page = c.ld_page / c.d; a.ld_scale_page = c.ld_scale_page;
  a.lanes_log2 = log2_at_least(c.d / 16);
  a.status = status;
  const bool e4m3 = c.k_scale != nullptr;
  const int per_sm = e4m3 ? (x.src_bf16 ? kBlocks<true, true> : kBlocks<true, false>)
                          : (x.src_bf16 ? kBlocks<false, true> : kBlocks<false, false>);
  const int64_t most = static_cast<int64_t>(per_sm) * device_sm_count();
  const int64_t launches = (T + most * kBlockTokens - 1) / (most * kBlockTokens);
  const int64_t share = (T + launches - 1) / launches;  // tokens of one
  const int64_t es = x.src_bf16 ? 2 : 4;
  const int groups = kThreads >> a.lanes_log2;
  for (int64_t t = 0; t < T; t += share) {
    a.T = std::min(share, T - t);
    a.t_first = t;
    a.q = x.q != nullptr ? static_cast<const char*>(x.q) + t * x.q_tok * es : nullptr;
    a.k = static_cast<const char*>(x.k) + t * x.k_tok * es;
    a.v = static_cast<const char*>(x.v) + t * x.v_tok * es;
    a.q_out = x.q_out != nullptr ? static_cast<uint16_t*>(x.q_out) + t * a.H * a.d : nullptr;
    a.positions = x.positions != nullptr ? x.positions + t : nullptr;
    a.slots = slots + t;
    a.tokens_per_block = static_cast<int>((a.T + most - 1) / most);
    const int64_t runs = (a.T + a.tokens_per_block - 1) / a.tokens_per_block;
    // a few tokens' vectors are shared out until every block has one round of them
    const int64_t rounds = (static_cast<int64_t>(a.tokens_per_block) * (a.H + 2 * a.H_kv) + groups - 1) / groups;
    a.parts = static_cast<int>(std::max<int64_t>(1, std::min(rounds, most / runs)));
    const unsigned grid = static_cast<unsigned>(runs * a.parts);
    if (e4m3) {
      if (x.src_bf16) launch_one<true, true>(a, x.tables_bf16, grid, stream);
      else launch_one<true, false>(a, x.tables_bf16, grid, stream);
    } else {
      if (x.src_bf16) launch_one<false, true>(a, x.tables_bf16, grid, stream);
      else launch_one<false, false>(a, x.tables_bf16, grid, stream);
    }
    if (cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace dwa
