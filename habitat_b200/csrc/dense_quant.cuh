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

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// quantized() of four values, packed.  The conversion instruction and the packing one saturate, which with ReLU leaves 0 of what is
// negative, by however much (6 instructions for four results, 9 with maxima and sums with 1.5 * 2^23).
template <bool kRelu>
__device__ __forceinline__ uint32_t quantized4(float2 a, float2 b, float inverse) {
  const float2 scale = make_float2(inverse, inverse);
  const float2 x = mul2(a, scale), y = mul2(b, scale);
  uint32_t high, r;
  if (kRelu) {
    asm("cvt.pack.sat.u8.s32.b32 %0, %1, %2, %3;" : "=r"(high) : "r"(__float2int_rn(y.y)), "r"(__float2int_rn(y.x)), "r"(0));
    asm("cvt.pack.sat.u8.s32.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(__float2int_rn(x.y)), "r"(__float2int_rn(x.x)), "r"(high));
  } else {
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(high) : "r"(__float2int_rn(y.y)), "r"(__float2int_rn(y.x)), "r"(0));
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(__float2int_rn(x.y)), "r"(__float2int_rn(x.x)), "r"(high));
  }
  return r;
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
