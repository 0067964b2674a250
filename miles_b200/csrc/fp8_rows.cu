// Kernels that leave 8-bit rows: E4M3 values with one fp32 scale for each row and 128 columns, s = max(amax, 1e-10) / 448, q = e4m3(x / s).
//
//   quantize_rows : of bf16 activations
//   rmsnorm_rows  : of RMSNorm(x + residual) * w; the sum leaves in bf16 (the statistics are those of what is stored), and the normalised
//                   rows in bf16 as well where a router wants them. They are rounded to 8 bits once, from 32.
//   permute_rows  : of rows in expert order, values and scales
//
// All are bound by memory. A thread holds 8 columns at a time, so that 16 neighbours hold a block of 128 and find its largest value by four
// shuffles. x / s is an IEEE division: the values are then those of the formula bit for bit, and the units have time for it.
//
// Reference counterpart: the per-token-group quantisers of the serving engines' FP8 path, and the block format of miles/utils/fp8_kernel.py:24-79.
#include <cuda_runtime.h>

#include "fp8_block.h"
#include "fp8_math.cuh"
#include "pdl.cuh"

namespace mb {
namespace {

using bf16 = __nv_bfloat16;
using f8::BLOCK;

__device__ __forceinline__ void unpack8(const uint4& r, float (&f)[8]) {
  const __nv_bfloat162* v = reinterpret_cast<const __nv_bfloat162*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __bfloat1622float2(v[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint4 r;
  __nv_bfloat162* v = reinterpret_cast<__nv_bfloat162*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  return r;
}

// The scale of the block whose 128 columns 16 neighbouring threads hold; every thread of the warp takes part.
__device__ __forceinline__ float block_scale(const float (&f)[8]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = f8::max_nan(m, fabsf(f[i]));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = f8::max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  return f8::scale_of(m);
}
__device__ __forceinline__ uint2 over_scale(const float (&f)[8], float s) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __fdiv_rn(f[i], s);
  return make_uint2(f8::pack_e4m3(v[0], v[1], v[2], v[3]), f8::pack_e4m3(v[4], v[5], v[6], v[7]));
}

// One CTA per row and 2048 columns.
__global__ void __launch_bounds__(256)
quantize_kernel(const bf16* __restrict__ x, long long ldx, int K, uint8_t* __restrict__ q, float* __restrict__ s) {
  pdl_enter();
  const long long row = blockIdx.x;
  const int c = (blockIdx.y * 256 + threadIdx.x) * 8;
  float f[8] = {};
  if (c < K) unpack8(*reinterpret_cast<const uint4*>(x + row * ldx + c), f);
  const float sc = block_scale(f);
  if (c >= K) return;
  *reinterpret_cast<uint2*>(q + row * K + c) = over_scale(f, sc);
  if ((threadIdx.x & 15) == 0) s[row * ((K + BLOCK - 1) / BLOCK) + c / BLOCK] = sc;
}

// One CTA per row, VPT times 8 columns of it per thread in registers.
template <int THREADS, int VPT>
__global__ void __launch_bounds__(THREADS)
rmsnorm_kernel(const bf16* __restrict__ x, long long ldx, const bf16* __restrict__ res, long long ldr, const bf16* __restrict__ w, float eps, int H,
               uint8_t* __restrict__ q, float* __restrict__ s, bf16* __restrict__ sum, bf16* __restrict__ y) {
  pdl_enter();
  __shared__ float red[THREADS / 32];
  const long long row = blockIdx.x;
  float f[VPT][8];
  float ss = 0.f;
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int c = (v * THREADS + threadIdx.x) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[v][i] = 0.f;
    if (c < H) {
      unpack8(*reinterpret_cast<const uint4*>(x + row * ldx + c), f[v]);
      if (res) {
        float g[8];
        unpack8(*reinterpret_cast<const uint4*>(res + row * ldr + c), g);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[v][i] += g[i];
        const uint4 h = pack8(f[v]);  // rounded as it is stored, so that the statistics are those of the stored row
        *reinterpret_cast<uint4*>(sum + row * H + c) = h;
        unpack8(h, f[v]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += f[v][i] * f[v][i];
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
  __syncthreads();
  float tot = 0.f;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) tot += red[i];
  const float r = rsqrtf(tot / H + eps);
  const int blocks = (H + BLOCK - 1) / BLOCK;
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int c = (v * THREADS + threadIdx.x) * 8;
    if (c < H) {
      float g[8];
      unpack8(*reinterpret_cast<const uint4*>(w + c), g);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[v][i] = f[v][i] * r * g[i];
    }
    const float sc = block_scale(f[v]);
    if (c < H) {
      *reinterpret_cast<uint2*>(q + row * H + c) = over_scale(f[v], sc);
      if ((threadIdx.x & 15) == 0) s[row * blocks + c / BLOCK] = sc;
      if (y) *reinterpret_cast<uint4*>(y + row * H + c) = pack8(f[v]);
    }
  }
}

// A warp per row.
__global__ void __launch_bounds__(256)
permute_kernel(const uint8_t* __restrict__ x, const float* __restrict__ xs, const int* __restrict__ src, const int* __restrict__ num_tiles,
               int top_k, long long rows, long long T, int K, uint8_t* __restrict__ q, float* __restrict__ s) {
  pdl_enter();
  const long long live = min(static_cast<long long>(num_tiles[1]), rows);
  const int lane = threadIdx.x & 31, blocks = (K + BLOCK - 1) / BLOCK, pieces = K / 16;
  for (long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5); row < live; row += static_cast<long long>(gridDim.x) * 8) {
    const int pair = src[row];
    const long long from = pair < 0 ? -1 : pair / top_k;
    const bool there = from >= 0 && from < T;
    const uint4* a = reinterpret_cast<const uint4*>(x + (there ? from : 0) * K);
    uint4* b = reinterpret_cast<uint4*>(q + row * K);
    for (int c = lane; c < pieces; c += 32) b[c] = there ? a[c] : make_uint4(0, 0, 0, 0);
    for (int c = lane; c < blocks; c += 32) s[row * blocks + c] = there ? xs[from * blocks + c] : f8::LEAST / f8::TOP;
  }
}

}  // namespace

cudaError_t fp8_quantize_rows(const void* x, long long ldx, long long T, int K, uint8_t* q, float* s, cudaStream_t stream) {
  if (T <= 0) return cudaSuccess;
  return pdl_launch(quantize_kernel, dim3(static_cast<unsigned>(T), (K + 2047) / 2048), 256, 0, stream, static_cast<const bf16*>(x), ldx, K, q, s);
}

cudaError_t fp8_rmsnorm_rows(const void* x, long long ldx, const void* residual, long long ldr, const void* w, float eps, long long T, int H,
                             uint8_t* q, float* s, void* sum, void* y, cudaStream_t stream) {
  if (T <= 0) return cudaSuccess;
  const auto go = [&](auto kernel, int threads) {
    return pdl_launch(kernel, static_cast<unsigned>(T), threads, 0, stream, static_cast<const bf16*>(x), ldx, static_cast<const bf16*>(residual), ldr,
                      static_cast<const bf16*>(w), eps, H, q, s, static_cast<bf16*>(sum), static_cast<bf16*>(y));
  };
  if (H <= 2048) return go(rmsnorm_kernel<256, 1>, 256);
  if (H <= 4096) return go(rmsnorm_kernel<256, 2>, 256);
  if (H <= 8192) return go(rmsnorm_kernel<256, 4>, 256);
  return go(rmsnorm_kernel<1024, 4>, 1024);
}

cudaError_t fp8_permute_rows(const uint8_t* x, const float* xs, const int* src, const int* num_tiles, int top_k, long long rows, long long T, int K,
                             uint8_t* q, float* s, cudaStream_t stream) {
  if (rows <= 0) return cudaSuccess;
  const long long grid = (rows + 7) / 8;
  return pdl_launch(permute_kernel, static_cast<unsigned>(grid < 148 * 16 ? grid : 148 * 16), 256, 0, stream, x, xs, src, num_tiles, top_k, rows, T, K, q, s);
}

}  // namespace mb
