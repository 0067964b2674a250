// Scales and values of 8-bit rows, as every kernel that leaves them computes them.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <stdint.h>

namespace mb {
namespace f8 {

constexpr int BLOCK = 128;           // columns that share a scale
constexpr float TOP = 448.f;         // the largest E4M3 value
constexpr float LEAST = 1e-10f;      // scales of empty blocks stay above zero (the weights' quantiser has the same bound)

// A maximum that keeps NaN: a block that holds one gets the scale NaN, and so does what is multiplied with it.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float scale_of(float amax) { return __fdiv_rn(max_nan(amax, LEAST), TOP); }

// Four values over their scale -> four E4M3 bytes, the first in the lowest (nearest even; at most 448 by the choice of the scale).
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

}  // namespace f8
}  // namespace mb
