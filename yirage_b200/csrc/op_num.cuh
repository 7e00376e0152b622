// 16-bit element types of the handle-free operators: widening two at a time, rounding once.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace ypk {

struct OpBf16 {
  static __device__ __forceinline__ float2 widen(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t round2(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return reinterpret_cast<const uint32_t &>(h);
  }
};

struct OpF16 {
  static __device__ __forceinline__ float2 widen(uint32_t v) {
    return __half22float2(reinterpret_cast<const __half2 &>(v));
  }
  static __device__ __forceinline__ uint32_t round2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return reinterpret_cast<const uint32_t &>(h);
  }
};

// Eight elements of 16 bits (one 16-byte load) as floats, and back.
template <class T>
__device__ __forceinline__ void op_widen8(const uint4 &v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = T::widen(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

template <class T>
__device__ __forceinline__ uint4 op_round8(const float (&x)[8]) {
  return make_uint4(T::round2(x[0], x[1]), T::round2(x[2], x[3]), T::round2(x[4], x[5]), T::round2(x[6], x[7]));
}

}  // namespace ypk
