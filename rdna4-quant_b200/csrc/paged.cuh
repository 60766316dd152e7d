// Shared by the paged-cache kernels: the checked view of r4q_paged_cache and
// the status bits that r4q_paged_status reports.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/r4q.h"

namespace r4q {

constexpr int kHeadDim = 128;
constexpr int kPagedTimeout = 1;   // a bounded wait gave up
constexpr int kPagedBadPage = 2;   // a row, position, length or page id outside the cache

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
// Status word of the attention kernels (the device is idle).
cudaError_t paged_attn_status(int clear, int* word);

}  // namespace r4q
