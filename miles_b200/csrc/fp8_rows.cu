// Kernels that leave 8-bit rows: E4M3 values with one fp32 scale for each row and 128 columns, s = max(amax, 1e-10) / 448, q = e4m3(x / s).
//
//   quantize_rows : of bf16 activations
//   rmsnorm_rows  : of RMSNorm(x + residual) * w; the sum leaves in bf16 (the statistics are those of what is stored), and the normalised
//                   rows in bf16 as well where a router wants them. They are rounded to 8 bits once, from 32.
//   permute_rows  : of rows in expert order, values and scales
//
// All are bound by memory. Neighbouring threads hold a block of 128 columns and find its largest value by shuffles. The values are those of the
// formula bit for bit; dividing by IEEE division costs as much time as memory does (16384 rows of 4096 with residual, 472 MB: 107 us).
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

// The scale of the block whose 128 columns 128 / 8 N neighbouring threads hold; every thread of the warp takes part.
template <int N>
__device__ __forceinline__ float block_scale(const float (&f)[N][8]) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) m = f8::max_nan(m, fabsf(f[j][i]));
#pragma unroll
  for (int o = BLOCK / 8 / N / 2; o > 0; o >>= 1) m = f8::max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  return f8::scale_of(m);
}
// f / s, rounded as a division rounds: a quotient from the correctly rounded reciprocal, corrected by its exact remainder (Markstein, IBM Journal of
// Research and Development 34, 1990). Remainders too small for fp32 belong to quotients that are zero in 8 bits.
__device__ __forceinline__ uint2 over_scale(const float (&f)[8], float s) {
  float v[8];
  const float inv = __fdiv_rn(1.f, s);
  if (s < __int_as_float(0x7f800000)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float t = f[i] * inv;
      v[i] = fmaf(fmaf(-t, s, f[i]), inv, t);
    }
  } else {  // an infinity or NaN in the block: finite values over it are zero
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = f[i] * inv;
  }
  return make_uint2(f8::pack_e4m3(v[0], v[1], v[2], v[3]), f8::pack_e4m3(v[4], v[5], v[6], v[7]));
}

// A thread takes 16 columns. (16384 rows of 4096, 201 MB: with 8 columns a thread 44 us, so 38.)
__global__ void __launch_bounds__(256)
quantize_kernel(const bf16* __restrict__ x, long long ldx, long long T, int K, uint8_t* __restrict__ q, float* __restrict__ s) {
  pdl_enter();
  const int blocks = (K + BLOCK - 1) / BLOCK;
  const long long block = static_cast<long long>(blockIdx.x) * 32 + threadIdx.x / 8;  // of all rows'
  const long long row = block / blocks;
  const int b = static_cast<int>(block - row * blocks), c = b * BLOCK + (threadIdx.x & 7) * 16;
  const bool there = row < T && c < K;  // (K is a multiple of 16)
  float f[2][8] = {};
  if (there) {
    const uint4* src = reinterpret_cast<const uint4*>(x + row * ldx + c);
    const uint4 lo = src[0], hi = src[1];
    unpack8(lo, f[0]);
    unpack8(hi, f[1]);
  }
  const float sc = block_scale(f);
  if (!there) return;
  const uint2 lo = over_scale(f[0], sc), hi = over_scale(f[1], sc);
  *reinterpret_cast<uint4*>(q + row * K + c) = make_uint4(lo.x, lo.y, hi.x, hi.y);
  if ((threadIdx.x & 7) == 0) s[row * blocks + b] = sc;
}

// CTAs go through the rows, VPT times 8 columns of a row per thread in registers together with the weights of the norm, and ask for their
// next row before they sum up this one. 16384 rows of 4096, us, with residual (472 MB) / without (201 MB): a CTA a row 83 / 64, so 76 / 56.
template <int VPT, bool RES>
__global__ void __launch_bounds__(1024)
rmsnorm_kernel(const bf16* __restrict__ x, long long ldx, const bf16* __restrict__ res, long long ldr, const bf16* __restrict__ w, float eps, int T, int H,
               uint8_t* __restrict__ q, float* __restrict__ s, bf16* __restrict__ sum, bf16* __restrict__ y) {
  pdl_enter();
  __shared__ float red[2][32];
  const int threads = blockDim.x, warps = threads >> 5, blocks = (H + BLOCK - 1) / BLOCK;
  uint4 xr[VPT], rr[VPT], wr[VPT];
  const auto fetch = [&](long long row) {
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int c = (v * threads + threadIdx.x) * 8;
      xr[v] = c < H ? *reinterpret_cast<const uint4*>(x + row * ldx + c) : make_uint4(0, 0, 0, 0);
      if (RES) rr[v] = c < H ? *reinterpret_cast<const uint4*>(res + row * ldr + c) : make_uint4(0, 0, 0, 0);
    }
  };
  if (static_cast<int>(blockIdx.x) < T) fetch(blockIdx.x);
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const int c = (v * threads + threadIdx.x) * 8;
    wr[v] = c < H ? *reinterpret_cast<const uint4*>(w + c) : make_uint4(0, 0, 0, 0);
  }
  int turn = 0;
  for (long long row = blockIdx.x; row < T; row += gridDim.x, turn ^= 1) {
    float f[VPT][1][8];
    float ss = 0.f;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int c = (v * threads + threadIdx.x) * 8;
      float(&a)[8] = f[v][0];
      unpack8(xr[v], a);
      if (RES) {
        float g[8];
        unpack8(rr[v], g);
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] += g[i];
        const uint4 h = pack8(a);  // rounded as it is stored, so that the statistics are those of the stored row
        if (c < H) *reinterpret_cast<uint4*>(sum + row * H + c) = h;
        unpack8(h, a);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += a[i] * a[i];
    }
    if (row + gridDim.x < T) fetch(row + gridDim.x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if ((threadIdx.x & 31) == 0) red[turn][threadIdx.x >> 5] = ss;
    __syncthreads();
    float tot = 0.f;
    for (int i = 0; i < warps; ++i) tot += red[turn][i];
    const float r = rsqrtf(tot / H + eps);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int c = (v * threads + threadIdx.x) * 8;
      float(&a)[8] = f[v][0];
      float g[8];
      unpack8(wr[v], g);
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = a[i] * r * g[i];
      const float sc = block_scale(f[v]);
      if (c < H) {
        *reinterpret_cast<uint2*>(q + row * H + c) = over_scale(a, sc);
        if ((threadIdx.x & 15) == 0) s[row * blocks + c / BLOCK] = sc;
        if (y) *reinterpret_cast<uint4*>(y + row * H + c) = pack8(a);
      }
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
  const long long grid = (T * ((K + BLOCK - 1) / BLOCK) + 31) / 32;
  if (grid > 0x7fffffffll) return cudaErrorInvalidValue;
  return pdl_launch(quantize_kernel, dim3(static_cast<unsigned>(grid)), 256, 0, stream, static_cast<const bf16*>(x), ldx, T, K, q, s);
}

cudaError_t fp8_rmsnorm_rows(const void* x, long long ldx, const void* residual, long long ldr, const void* w, float eps, long long T, int H,
                             uint8_t* q, float* s, void* sum, void* y, cudaStream_t stream) {
  if (T <= 0) return cudaSuccess;
  if (T > 0x7fffffffll) return cudaErrorInvalidValue;
  // few rows: as many threads as can share a row (its latency counts); many: two pieces a thread, for more bytes under way
  const int vpt = H > 16384 ? 4 : H > 8192 || T > 592 ? 2 : 1;
  const int threads = (H / 8 + vpt * 32 - 1) / (vpt * 32) * 32;
  const long long most = 148ll * (vpt == 1 ? 4 : 2048 / threads > 0 ? 2048 / threads : 1);
  const auto go = [&](auto kernel) {
    return pdl_launch(kernel, static_cast<unsigned>(T < most ? T : most), threads, 0, stream, static_cast<const bf16*>(x), ldx,
                      static_cast<const bf16*>(residual), ldr, static_cast<const bf16*>(w), eps, static_cast<int>(T), H, q, s, static_cast<bf16*>(sum),
                      static_cast<bf16*>(y));
  };
  if (vpt == 1) return residual ? go(rmsnorm_kernel<1, true>) : go(rmsnorm_kernel<1, false>);
  if (vpt == 2) return residual ? go(rmsnorm_kernel<2, true>) : go(rmsnorm_kernel<2, false>);
  return residual ? go(rmsnorm_kernel<4, true>) : go(rmsnorm_kernel<4, false>);
}

cudaError_t fp8_permute_rows(const uint8_t* x, const float* xs, const int* src, const int* num_tiles, int top_k, long long rows, long long T, int K,
                             uint8_t* q, float* s, cudaStream_t stream) {
  if (rows <= 0) return cudaSuccess;
  const long long grid = (rows + 7) / 8;
  return pdl_launch(permute_kernel, static_cast<unsigned>(grid < 148 * 16 ? grid : 148 * 16), 256, 0, stream, x, xs, src, num_tiles, top_k, rows, T, K, q, s);
}

}  // namespace mb
