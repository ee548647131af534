// The 8-bit rows of the dense-layer operators: scales, rounding, packing (definition: dense_int8.cu).
#pragma once

#include "dense_gemm.cuh"

namespace dense {
namespace {

struct RowScale {
  float inverse, scale;
  bool bad;
};
__device__ __forceinline__ RowScale row_scale(float amax) {
  RowScale r;
  r.bad = !(amax < __int_as_float(0x7F800000));
  const bool zero = amax < 0x1p-119f;
  r.inverse = r.bad || zero ? 0.0f : __fdiv_rn(127.0f, amax);
  r.scale = r.bad ? __int_as_float(0x7FFFFFFF) : zero ? 0.0f : __fdiv_rn(amax, 127.0f);
  return r;
}
// The integer nearest to x * inverse (ties to even) in the low byte: adding 1.5 * 2^23 leaves it in the last bits.
__device__ __forceinline__ uint32_t quantized(float x, float inverse) {
  return __float_as_uint(__fadd_rn(__fmul_rn(x, inverse), 12582912.0f));
}
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float(float x) { return x; }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

}  // namespace
}  // namespace dense
