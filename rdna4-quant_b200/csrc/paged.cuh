// Shared by the paged-cache and likelihood kernels: the checked view of
// r4q_paged_cache and the status bits that r4q_kernel_status reports.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/r4q.h"

namespace r4q {

constexpr int kHeadDim = 128;
constexpr int kWaitPolls = 1 << 22;  // of a bounded wait of these kernels, before it gives up
constexpr int kPagedTimeout = 1;   // a bounded wait gave up
constexpr int kPagedBadPage = 2;   // a row, position, length or page id outside the cache

// x / d for 0 <= x < 2^31 by a multiplication: m = ceil(2^(31 + s) / d), 2^(s-1) < d <= 2^s
// (Granlund and Montgomery, Division by invariant integers using multiplication, 1994)
struct FastDiv {
  uint32_t m;
  int s;
  __device__ __forceinline__ int div(int x) const { return (int)(((uint64_t)m * (uint32_t)x) >> (31 + s)); }
};
inline FastDiv fast_div(uint32_t d) {
  int s = 0;
  while ((1ull << s) < d) ++s;
  return FastDiv{(uint32_t)(((1ull << (31 + s)) + d - 1) / d), s};
}

struct PagedView {
  uint8_t *k, *v;
  long k_stride, v_stride;         // bytes between pages
  int n_pages, page, Hk;
  const int* table;
  long ld_table;
  int seqs, max_blocks;
  const float *k_scale, *v_scale;  // [Hk] or null
};

// Checks the caller's description and fills the view; `what` names the caller.
int paged_view(const char* what, const r4q_paged_cache* c, PagedView* out);
// Polls that a launch gives its waits: kWaitPolls, or what r4q_debug_wait_limit set.  The
// wait for copies still in flight after that always has kWaitPolls.
int wait_polls();
// Where the attention's and the likelihood kernels' status words lie on the current device.
cudaError_t paged_attn_status_word(int** word);
cudaError_t logprob_status_word(int** word);

}  // namespace r4q
