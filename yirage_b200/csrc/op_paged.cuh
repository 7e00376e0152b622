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

// n / d for 0 <= n < 2^31 and 1 <= d < 2^31 without a division: with l = ceil(log2 d) and
// mul = floor(2^32 (2^l - d) / d) + 1, n / d = (n + mulhi(n, mul)) >> l (Granlund and Montgomery,
// "Division by invariant integers using multiplication", 1994).
struct FastDivisor {
  uint32_t mul, shift;
};
inline FastDivisor fast_divisor(int d) {
  uint32_t l = 0;
  while ((uint64_t(1) << l) < uint64_t(d)) ++l;
  return {uint32_t((((uint64_t(1) << l) - d) << 32) / d + 1), l};
}
__device__ __forceinline__ uint32_t fast_div(uint32_t n, const FastDivisor &d) {
  return (n + __umulhi(n, d.mul)) >> d.shift;
}

__device__ __forceinline__ void paged_flag(const PagedView &c, int bit) {
  if (c.status) atomicOr(c.status, bit);
}

}  // namespace ypk
