// Host side of what the paged-cache operators share.
#pragma once
#include "op_common.h"
#include "op_paged.cuh"

namespace ypk {

// Checks the cache description; `what` names the call in messages.
int paged_check(const char *what, const ypk_paged_cache *c, bool append);
PagedView paged_view(const ypk_paged_cache *c);

// Rows of query heads, by strides in elements: do the bytes from the first to the last of them
// touch the other's?
struct HeadRows {
  const void *at;
  int64_t token, group, head;      // strides
};
inline bool heads_touch(const HeadRows &a, const HeadRows &b, int rows, int kv_heads, int group, int head_dim) {
  const auto end = [&](const HeadRows &h) {
    return reinterpret_cast<uintptr_t>(h.at) +
           2 * uint64_t((rows - 1) * h.token + (kv_heads - 1) * h.group + (group - 1) * h.head + head_dim);
  };
  return reinterpret_cast<uintptr_t>(a.at) < end(b) && reinterpret_cast<uintptr_t>(b.at) < end(a);
}

}  // namespace ypk
