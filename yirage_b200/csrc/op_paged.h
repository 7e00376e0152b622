// Host side of what the paged-cache operators share.
#pragma once
#include "op_common.h"
#include "op_paged.cuh"

namespace ypk {

// Checks the cache description; `what` names the call in messages.
int paged_check(const char *what, const ypk_paged_cache *c, bool append);
PagedView paged_view(const ypk_paged_cache *c);

}  // namespace ypk
