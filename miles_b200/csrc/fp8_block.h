// Serving in block-scaled 8 bits: E4M3 activations with one fp32 scale for each row and 128 columns ("8-bit rows"), E4M3 weights with one
// for each 128 x 128. Kernels that leave such rows are in fp8_rows.cu, products in fp8_gemm.cu.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace mb {

struct Fp8Gemm {
  int M, N, K;  // rows of x; rows of one matrix of W (both halves of a gate-up matrix); contraction, a multiple of 16
  const uint8_t* x;   // [M, K], row pitch ldx bytes (a multiple of 16)
  long long ldx;
  const float* xs;    // [M, ceil(K / 128)]
  const uint8_t* w;   // [groups][N, K]
  const float* ws;    // [groups][halves * ceil(N / halves / 128), ceil(K / 128)]; halves: 2 if gated, else 1
  int groups;
  const int* tile_group;   // null (one matrix for all rows), or [max_tiles][4] = {matrix, first row, rows (<= 128), 0} ...
  const int* num_tiles;    // ... of which as many as this device scalar says are live
  int max_tiles;
  void* y;            // bf16 [M, N], row pitch ldy elements; null if gated
  long long ldy;
  const void* residual;    // bf16 [M, N] with row pitch ldr that is added before the rounding, or null
  long long ldr;
  uint8_t* q;         // gated: silu(gate) * up as 8-bit rows [M, N / 2] ...
  float* s;           // ... and their scales [M, ceil(N / 2 / 128)]
  int* status;        // device status word (0 = ok), may be null
  void* workspace;    // fp8_gemm_workspace bytes, 16-byte aligned
};
long long fp8_gemm_workspace(const Fp8Gemm& p);
// Launches of a product by expert of `rows` rows with matrices [N, K] and a list of max_tiles row tiles: one, and one to join row tiles where pairs
// of CTAs compute it.
int fp8_grouped_launches(long long rows, int groups, int N, int K, bool gated, int max_tiles);
// Launches on `stream`. Returns 0 or -1 with the reason in fp8_last_error().
int fp8_gemm_launch(const Fp8Gemm& p, cudaStream_t stream);
const char* fp8_last_error();

// 8-bit rows of x (bf16 [T, K], row pitch ldx elements).
cudaError_t fp8_quantize_rows(const void* x, long long ldx, long long T, int K, uint8_t* q, float* s, cudaStream_t stream);
// 8-bit rows of RMSNorm(h) * w, h = x (+ residual, rounded to bf16 and stored in sum); y, if given, receives them in bf16.
// x, residual: bf16 [T, H] with row pitches in elements.
cudaError_t fp8_rmsnorm_rows(const void* x, long long ldx, const void* residual, long long ldr, const void* w, float eps, long long T, int H,
                             uint8_t* q, float* s, void* sum, void* y, cudaStream_t stream);
// Rows of x in expert order: row i is that of token src[i] / top_k; negative entries leave zeros. Live rows: num_tiles[1].
cudaError_t fp8_permute_rows(const uint8_t* x, const float* xs, const int* src, const int* num_tiles, int top_k, long long rows, long long T, int K,
                             uint8_t* q, float* s, cudaStream_t stream);

}  // namespace mb
