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

// g / (1 + e^-g) from the hardware's approximations of 2^x and 1 / x, without their care for results below 2^-126 (a sixth of a gate-up tile's
// output): exact to a few units in the last place and |g| 2^-24 relative, where the sums before it are to about 10 units. A divisor above
// 2^126 gives zero, as fp32 would within 1e-36; -infinity gives NaN, as the formula does.
__device__ __forceinline__ float silu(float g) {
  constexpr float LOG2E = 1.4426950408889634f;
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -LOG2E));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return g * r;
}

// Four values over their scale -> four E4M3 bytes, the first in the lowest (nearest even; at most 448 by the choice of the scale).
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

}  // namespace f8
}  // namespace mb
