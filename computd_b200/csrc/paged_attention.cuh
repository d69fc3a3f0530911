// paged_attention.cuh — what the two kernels of the attention over the paged
// cache share (paged_attention.cu: few rows per key/value head;
// paged_attention_mma.cu: many).
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace dwa {

struct PagedArgs {
  const uint16_t* q;
  uint16_t* out;
  int64_t q_ld, out_ld;  // elements between tokens
  const void *k, *v;
  const float *k_scale, *v_scale;
  int64_t ld_page, ld_scale_page;  // elements, scales
  int64_t n_pages;
  const int32_t* table;
  int64_t ld_table;
  int max_pages, page_log2;
  const int32_t* lengths;
  const int32_t* q_start;  // null: `even` rows per sequence
  int64_t T;
  int even, max_q;
  int B, H, H_kv, group;  // group = H / H_kv query heads per key/value head
  int d;
  float scale_log2;  // scale * log2(e)
  int32_t* status;
};

// One sequence as the device finds it.
struct PagedSeq {
  int64_t row0;   // first row of q
  int n;          // new tokens
  int length;     // cached tokens, the new ones with them
  bool bad;       // its rows get NaN
};

__device__ __forceinline__ void paged_report(int32_t* status) {
  if (status != nullptr) atomicCAS(status, 0, 5 /* DWA_ERR_DEVICE_CHECK */);
}

__device__ __forceinline__ PagedSeq paged_seq(const PagedArgs& a, int b) {
  PagedSeq s;
  if (a.q_start != nullptr) {
    const int64_t lo = __ldg(a.q_start + b), hi = __ldg(a.q_start + b + 1);
    const bool fine = lo >= 0 && lo <= hi && hi <= a.T;
    s.row0 = fine ? lo : 0;
    s.n = fine ? static_cast<int>(hi - lo) : 0;  // rows that cannot be told apart stay as they are
    s.bad = !fine;
  } else {
    s.row0 = static_cast<int64_t>(b) * a.even;
    s.n = a.even;
    s.bad = false;
  }
  s.length = __ldg(a.lengths + b);
  if (s.length < 0 || s.length > (static_cast<int64_t>(a.max_pages) << a.page_log2) ||
      s.n > a.max_q) {
    s.bad = true;
    s.length = 0;
  }
  return s;
}

// Tokens that new token i may see.
__device__ __forceinline__ int paged_visible(const PagedSeq& s, int i) {
  return max(s.length - s.n + i + 1, 0);
}

}  // namespace dwa
