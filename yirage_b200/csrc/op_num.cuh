// 16-bit element types of the handle-free operators: widening two at a time, rounding once.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace ypk {

// In every kernel of op_launch (op_common.h), before it touches memory: until the kernel before it
// on the stream has ended and its writes are there.  What the kernel before may have written
// (inputs, page tables, weights: all of it) is read behind this with ordinary loads only: a load that
// says its data is never written (ld.global.nc, __ldg) may be moved above it, and says something
// untrue, as this kernel is already there while the one before still writes.
__device__ __forceinline__ void op_wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// 16 bytes that are read once (to leave the caches first).
__device__ __forceinline__ uint4 op_load_once(const uint4 *p) {
  uint4 v;
  asm volatile("ld.global.cs.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

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

// Pairs of fp32 in one 64-bit register: one instruction for both, each rounded as usual.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 halves(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// Eight elements of 16 bits (one 16-byte load) as floats or pairs, and back.
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
__device__ __forceinline__ void op_widen8(const uint4 &v, f32x2 (&x)[4]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = T::widen(w[i]);
    x[i] = pair(f.x, f.y);
  }
}

template <class T>
__device__ __forceinline__ uint4 op_round8(const f32x2 (&x)[4]) {
  const float2 a = halves(x[0]), b = halves(x[1]), c = halves(x[2]), d = halves(x[3]);
  return make_uint4(T::round2(a.x, a.y), T::round2(b.x, b.y), T::round2(c.x, c.y), T::round2(d.x, d.y));
}

}  // namespace ypk
