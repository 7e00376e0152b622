// What the handle-free operators (op_*.cu) share with the rest of the C ABI.
#pragma once
#include <cuda_runtime.h>

#include "../../include/ypk.h"

namespace ypk {

// Sets the message that ypk_last_error(NULL) returns on this thread; gives `code` back.
int op_fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));

// The current device and its SM count, asked for once per device.
struct DeviceInfo {
  int device, sms;
};
int op_device(const char *what, DeviceInfo *d);

inline bool op_aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Launches kernel(args) on clusters of `cluster` CTAs (0: none), set up while the kernel before it on
// the stream still ends: every kernel launched with this calls op_wait_for_previous() before it
// touches memory, so it sees what an ordinary launch would.  Back to back that saves 1.4 to
// 2.6 us a call.  (Kernels that let their successors start before they end were slower: the
// waiting CTAs take the place, and the even spread, of the running ones.)
template <class Args>
int op_launch(const char *what, void (*kernel)(Args), dim3 grid, int threads, int shared, int cluster,
              cudaStream_t stream, const Args &args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args);
  if (e != cudaSuccess) return op_fail(YPK_ERR_CUDA, "%s: launch: %s", what, cudaGetErrorString(e));
  return YPK_OK;
}

}  // namespace ypk
