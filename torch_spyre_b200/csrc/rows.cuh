// Rows of head vectors in registers: vector conversions between the row types
// and fp32, and the rotary turn of a pair.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <math_constants.h>

#include "common.cuh"

namespace b200kv {

// Eight 16-bit elements of one 16-byte vector as fp32, and back (rounded to
// nearest even once).
__device__ __forceinline__ void unpack8(uint4 v, float (&f)[8], __half) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
__device__ __forceinline__ void unpack8(uint4 v, float (&f)[8], __nv_bfloat16) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8], T t) {
  return make_uint4(pack2(f[0], f[1], t), pack2(f[2], f[3], t), pack2(f[4], f[5], t), pack2(f[6], f[7], t));
}

__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ void from_float(__half &d, float x) { d = __float2half_rn(x); }
__device__ __forceinline__ void from_float(__nv_bfloat16 &d, float x) { d = __float2bfloat16_rn(x); }
__device__ __forceinline__ void from_float(float &d, float x) { d = x; }

// The turn of one pair.  Every product and sum is rounded to fp32 by itself
// (no contraction to fma), so a row that is quantised afterwards falls on the
// same step whichever kernel or host code computed it.
__device__ __forceinline__ void turn_pair(float a, float b, float cosv, float sinv, float &ra, float &rb) {
  ra = __fsub_rn(__fmul_rn(a, cosv), __fmul_rn(b, sinv));
  rb = __fadd_rn(__fmul_rn(b, cosv), __fmul_rn(a, sinv));
}

inline bool aligned_to(const void *p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace b200kv
