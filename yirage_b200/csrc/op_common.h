// What the handle-free operators (op_*.cu) share with the rest of the C ABI.
#pragma once
#include <cuda_runtime.h>

#include "../../include/ypk.h"

namespace ypk {

// Sets the message that ypk_last_error(NULL) returns on this thread; gives `code` back.
int op_fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));

inline bool op_aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline int op_launched(const char *what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return op_fail(YPK_ERR_CUDA, "%s: launch: %s", what, cudaGetErrorString(e));
  return YPK_OK;
}

}  // namespace ypk
