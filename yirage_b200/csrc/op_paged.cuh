// Device side of what the paged-cache operators share: the cache as a kernel argument.
#pragma once
#include <cuda_runtime.h>

#include "op_num.cuh"
#include "paged_index.h"

namespace ypk {

struct PagedView {
  char *k, *v;
  int64_t stride_page, stride_token, stride_head;   // elements of 16 bits
  const int *indptr, *indices, *last, *qo;
  int *status;
  int num_pages, page_size, kv_heads, num_requests, num_indices;
};

__device__ __forceinline__ void paged_flag(const PagedView &c, int bit) {
  if (c.status) atomicOr(c.status, bit);
}

}  // namespace ypk
