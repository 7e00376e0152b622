// Host side of what the paged-cache operators share.
#pragma once
#include "op_common.h"
#include "op_paged.cuh"
#include "strided_rows.h"

namespace ypk {

// Checks the cache description; `what` names the call in messages.
int paged_check(const char *what, const ypk_paged_cache *c, bool append);
PagedView paged_view(const ypk_paged_cache *c);

// Rows of heads by strides in elements of 16 bits, as strided_rows.h takes them.
inline StridedRows head_rows(const void *at, int64_t tokens, int64_t token, int64_t groups, int64_t group,
                             int64_t heads, int64_t head, int64_t head_dim) {
  return {int64_t(reinterpret_cast<uintptr_t>(at)) / 2, head_dim, {token, group, head}, {tokens, groups, heads}};
}
inline StridedRows cache_rows(const ypk_paged_cache *c, const void *at) {
  return head_rows(at, c->num_pages, c->stride_page, c->page_size, c->stride_token, c->num_kv_heads, c->stride_head,
                   c->head_dim);
}

}  // namespace ypk
