// Products of 8-bit rows with block-scaled 8-bit weights for sm_100a:
//
//   y[t, n] = (residual[t, n] +) sum over blocks b of 128 along K of  xs[t, b] ws[n / 128, b] sum over k in b of x[t, k] w[n, k]
//
// in E4M3 with fp32 scales of any value, so that no scale can ride in the tensor core's own (power-of-two) ones: a block's product is
// computed by four tcgen05.mma into a TMEM buffer of its own, and eight warps add it, scaled, to sums in registers while the tensor core
// fills the next buffer. Per 128 x 256 x 128 block the tensor core needs 512 clocks, the warps about 256 multiply-adds per scheduler.
// The rows are one batch, or sorted by expert (row tiles {matrix, first row, rows} as the router's sort leaves them). A gate-up weight's
// tile takes 128 gate rows and their 128 up rows, so that silu(gate) * up leaves as a whole block of 128 columns of 8-bit rows, scaled by
// their largest value, without passing through memory in between.
//
//   warp 0     : TMA producer (128-byte swizzle)          warp 1 : TMEM allocator, tcgen05.mma issuer
//   warps 2..9 : sums of a tile in registers (two warps per 32 rows, half of the columns each), then rows of 64 bytes through shared memory
//
// Reference counterpart: the block-wise FP8 GEMMs of the serving engines that load its FP8 checkpoints (weight_block_size [128, 128]:
// miles/backends/megatron_utils/megatron_to_hf/processors/quantizer_fp8.py, miles/utils/fp8_kernel.py:24-79).
#include <cuda.h>
#include <string.h>

#include <atomic>
#include <mutex>
#include <string>

#include "fp8_block.h"
#include "fp8_math.cuh"
#include "ptx.cuh"

namespace mb {
namespace {

constexpr int BM = 128, BK = 128;
constexpr int HALF_BYTES = 128 * BK;  // 128 rows of one operand and stage
constexpr int THREADS = 320;
constexpr int EPI_WARPS = 8;
constexpr int STAGING = EPI_WARPS * 4096;

struct Args {
  int M, N, K;
  int halves, blocks_n, blocks_k;  // of a matrix; blocks of its scales
  const float* xs;
  const float* ws;
  int groups, max_tiles;
  const int* tile_group;
  const int* num_tiles;
  __nv_bfloat16* y;
  long long ldy;
  const __nv_bfloat16* residual;
  long long ldr;
  int vec_ok;
  uint8_t* q;
  float* s;
  int* status;
};

struct Tile {
  int row0, row_end, n0, group;  // rows of x; first column of y (or of silu(gate) * up)
};

__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "}\n"
      :
      : "r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor of kind::f8f6f4: fp32 accumulators (bit 4), E4M3 operands (0 at bits 7 and 10), both K-major.
__host__ __device__ constexpr uint32_t idesc_e4m3(int m, int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// The wait of a load from TMEM names its registers, so that nothing that reads them moves ahead of it while the next load is under way.
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// Whether every thread of the warp came out of its wait: the loads from TMEM behind it are the whole warp's.
__device__ __forceinline__ bool all_got(bool got) { return __all_sync(0xffffffffu, got); }

// Columns of a tile: BN of y, or BN / 2 of silu(gate) * up.
template <int BN, bool GATED>
__device__ __forceinline__ int column_tiles(const Args& p) {
  constexpr int COLS = GATED ? BN / 2 : BN;
  return (p.N / p.halves + COLS - 1) / COLS;
}
template <int BN, bool GATED>
__device__ __forceinline__ int tiles_of(const Args& p) {
  int m = (p.M + BM - 1) / BM;
  if (p.tile_group) m = min(max(*p.num_tiles, 0), p.max_tiles);
  return m * column_tiles<BN, GATED>(p);
}
template <int BN, bool GATED>
__device__ __forceinline__ Tile tile_at(const Args& p, int t) {
  const int n_tiles = column_tiles<BN, GATED>(p);
  Tile r;
  int mt = t / n_tiles, nt = t - mt * n_tiles;
  if (p.tile_group) {
    const int4 e = reinterpret_cast<const int4*>(p.tile_group)[mt];
    r.group = min(max(e.x, 0), p.groups - 1);
    r.row0 = min(max(e.y, 0), p.M);
    r.row_end = min(p.M, r.row0 + min(max(e.z, 0), BM));
  } else {
    // bands of eight row tiles, their columns outermost: CTAs that run together share tiles of W in L2
    constexpr int BAND = 8;
    const int m_tiles = (p.M + BM - 1) / BM;
    const int band = t / (BAND * n_tiles), first = band * BAND;
    const int rows = min(m_tiles - first, BAND), in_band = t - band * BAND * n_tiles;
    mt = first + in_band % rows;
    nt = in_band / rows;
    r.group = 0;
    r.row0 = mt * BM;
    r.row_end = min(p.M, r.row0 + BM);
  }
  r.n0 = nt * (GATED ? BN / 2 : BN);
  return r;
}

template <int BN, bool GATED, int STAGES>
__global__ void __launch_bounds__(THREADS, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const Args p) {
  constexpr int BUFS = 512 / BN;                        // TMEM holds this many blocks' products
  constexpr int STAGE = (BM + BN) * BK;
  constexpr int COLS = BN / 2;                          // of the tile, per thread
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t staging = base + STAGES * STAGE;
  __shared__ __align__(8) unsigned long long bars[2 * STAGES + 2 * BUFS + 1];
  __shared__ uint32_t tmem_slot_s;
  __shared__ int abort_s;
  volatile int* abort_flag = &abort_s;
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto tfull_bar = [&](int b) { return bar0 + 8u * (2 * STAGES + b); };
  auto tempty_bar = [&](int b) { return bar0 + 8u * (2 * STAGES + BUFS + b); };
  const uint32_t amax_bar = bar0 + 8u * (2 * STAGES + 2 * BUFS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    abort_s = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < BUFS; ++b) {
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), EPI_WARPS);
    }
    mbar_init(amax_bar, EPI_WARPS * 32);
    fence_barrier_init();
    prefetch_tensormap(&map_x);
    prefetch_tensormap(&map_w);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_slot_s), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_slot_s);
  const int total = tiles_of<BN, GATED>(p);
  const int half_n = p.N / p.halves;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < total; t += gridDim.x) {
        const Tile tl = tile_at<BN, GATED>(p, t);
        const int w0 = tl.group * p.N + tl.n0;
        const int w1 = GATED ? w0 + half_n : w0 + 128;  // the tile's second 128 rows of W
        for (int kb = 0; kb < p.blocks_k; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, ERR_WAIT_EMPTY)) {
            ok = false;
            break;
          }
          const uint32_t dst = base + stage * STAGE;
          mbar_expect_tx(full_bar(stage), STAGE);
          tma_load_2d(dst, &map_x, full_bar(stage), kb * BK, tl.row0);
          tma_load_2d(dst + HALF_BYTES, &map_w, full_bar(stage), kb * BK, w0);
          if (BN == 256) tma_load_2d(dst + 2 * HALF_BYTES, &map_w, full_bar(stage), kb * BK, w1);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) {  // copies in flight get a bounded time to land before shared memory is released
        const unsigned long long t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 2000000ull) {
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    constexpr uint32_t idesc = idesc_e4m3(BM, BN);
    int stage = 0, buf = 0;
    uint32_t phase = 0, tphase = 0;
    bool ok = true;
    for (int t = blockIdx.x; ok && t < total; t += gridDim.x) {
      for (int kb = 0; kb < p.blocks_k; ++kb) {
        ok = all_got(mbar_wait(tempty_bar(buf), tphase ^ 1u, abort_flag, p.status, ERR_WAIT_TMEM_EMPTY) &&
                     mbar_wait(full_bar(stage), phase, abort_flag, p.status, ERR_WAIT_FULL));
        if (!ok) break;
        tc_fence_after();
        if (lane == 0) {
          const uint32_t x = base + stage * STAGE, w = x + HALF_BYTES;
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            umma_f8(tmem + buf * BN, make_smem_desc(x + k * 32, 16, 1024), make_smem_desc(w + k * 32, 16, 1024), idesc, k > 0 ? 1u : 0u);
          umma_commit(empty_bar(stage));
          umma_commit(tfull_bar(buf));
        }
        __syncwarp();
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
        if (++buf == BUFS) {
          buf = 0;
          tphase ^= 1u;
        }
      }
    }
  } else {
    const int quad = warp & 3, side = (warp - 2) >> 2;  // rows of the tile that this warp reaches in TMEM; its half of the columns
    const uint32_t mine = staging + (warp - 2) * 4096;
    int buf = 0;
    uint32_t tphase = 0;
    int turn = 0;
    bool ok = true;
    for (int t = blockIdx.x; ok && t < total; t += gridDim.x, ++turn) {
      const Tile tl = tile_at<BN, GATED>(p, t);
      const int row = tl.row0 + quad * 32 + lane;
      const float* xs = p.xs + static_cast<long long>(min(row, p.M - 1)) * p.blocks_k;
      // scales of the weights' block(s) of this thread's columns: one for all, or the gate's and the up rows'
      const int nb = min(tl.n0 / 128 + (!GATED && BN == 256 ? side : 0), p.blocks_n / p.halves - 1);
      const float* ws0 = p.ws + (static_cast<long long>(tl.group) * p.blocks_n + nb) * p.blocks_k;
      const float* ws1 = ws0 + (GATED ? static_cast<long long>(p.blocks_n / 2) * p.blocks_k : 0);
      float acc[COLS];
#pragma unroll
      for (int i = 0; i < COLS; ++i) acc[i] = 0.f;
      float xn = xs[0], wn0 = ws0[0], wn1 = GATED ? ws1[0] : 0.f;
      for (int kb = 0; kb < p.blocks_k; ++kb) {
        const float c0 = xn * wn0, c1 = GATED ? xn * wn1 : c0;
        if (kb + 1 < p.blocks_k) {
          xn = xs[kb + 1];
          wn0 = ws0[kb + 1];
          if (GATED) wn1 = ws1[kb + 1];
        }
        ok = all_got(mbar_wait(tfull_bar(buf), tphase, abort_flag, p.status, ERR_WAIT_TMEM_FULL));
        if (!ok) break;
        tc_fence_after();
        // thread's columns: COLS from side * COLS on, or (gated) COLS / 2 gate columns and the same up columns
        const uint32_t from = tmem + buf * BN + (static_cast<uint32_t>(quad * 32) << 16);
        const auto col = [&](int c) {
          return static_cast<uint32_t>(GATED ? (c < COLS / 2 ? side * (COLS / 2) + c : BN / 2 + side * (COLS / 2) + c - COLS / 2) : side * COLS + c);
        };
        uint32_t d[2][16];
        tmem_ld_32x16(from + col(0), d[0]);
#pragma unroll
        for (int c = 0; c < COLS; c += 16) {
          const int now = (c / 16) & 1;
          tmem_ld_wait_for(d[now]);
          if (c + 16 < COLS) {
            tmem_ld_32x16(from + col(c + 16), d[now ^ 1]);
          } else {  // everything has left the buffer
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(tempty_bar(buf));
          }
          const float cc = GATED && c >= COLS / 2 ? c1 : c0;
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[c + i] = fmaf(cc, __uint_as_float(d[now][i]), acc[c + i]);
        }
        if (++buf == BUFS) {
          buf = 0;
          tphase ^= 1u;
        }
      }
      if (!ok) break;
      const int r_in8 = lane >> 2, piece = lane & 3;  // reading the staged rows: eight at a time, four lanes each
      if constexpr (GATED) {
        constexpr int OUT = COLS / 2;
        const int c0 = tl.n0 + side * OUT;
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < OUT; ++i) {
          const float g = acc[i];
          // (__expf is exact to 2 + |g| / 10 units in the last place, where the sums before it are to about 10)
          const float a = c0 + i < half_n ? g / (1.f + __expf(-g)) * acc[OUT + i] : 0.f;
          acc[i] = a;
          amax = f8::max_nan(amax, fabsf(a));
        }
        // The two warps of a row exchange theirs through the second halves of their staging, by turns of the tiles (a warp that
        // writes for a tile has seen all of them arrive for the one before, and so read what is overwritten).
        const uint32_t there = 2048 + (turn & 1) * 128 + lane * 4;
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(mine + there), "f"(amax) : "memory");
        mbar_arrive(amax_bar);
        ok = all_got(mbar_wait(amax_bar, turn & 1, abort_flag, p.status, ERR_WAIT_TMEM_FULL));
        if (!ok) break;
        float other;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(other) : "r"(staging + ((warp - 2) ^ 4) * 4096 + there) : "memory");
        const float sc = f8::scale_of(f8::max_nan(amax, other));
        // times the reciprocal: the products carry errors of their own that are larger than its
        const float inv = 1.f / sc;
        const int out_blocks = (half_n + 127) / 128;
        if (side == 0 && row < tl.row_end) p.s[static_cast<long long>(row) * out_blocks + tl.n0 / 128] = sc;
#pragma unroll
        for (int j = 0; j < OUT / 16; ++j) {
          uint32_t v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            v[i] = f8::pack_e4m3(acc[16 * j + 4 * i] * inv, acc[16 * j + 4 * i + 1] * inv, acc[16 * j + 4 * i + 2] * inv, acc[16 * j + 4 * i + 3] * inv);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(mine + lane * 64 + ((j ^ ((lane >> 1) & 3)) * 16)), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                       "r"(v[3])
                       : "memory");
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 8 * i + r_in8, to = tl.row0 + quad * 32 + r;
          uint4 v;
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                       : "r"(mine + r * 64 + ((piece ^ ((r >> 1) & 3)) * 16))
                       : "memory");
          if (to < tl.row_end && c0 + piece * 16 < half_n) *reinterpret_cast<uint4*>(p.q + static_cast<long long>(to) * half_n + c0 + piece * 16) = v;
        }
        __syncwarp();
      } else {
#pragma unroll
        for (int j = 0; j < COLS / 32; ++j) {
          const int c0 = tl.n0 + side * COLS + j * 32;
          if (c0 < p.N) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(mine + lane * 128 + ((i ^ (lane & 7)) * 16)), "f"(acc[32 * j + 4 * i]),
                           "f"(acc[32 * j + 4 * i + 1]), "f"(acc[32 * j + 4 * i + 2]), "f"(acc[32 * j + 4 * i + 3])
                           : "memory");
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = 8 * i + r_in8, to = tl.row0 + quad * 32 + r, c = c0 + piece * 8;
              float f[8];
#pragma unroll
              for (int h = 0; h < 2; ++h)
                asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                             : "=f"(f[4 * h]), "=f"(f[4 * h + 1]), "=f"(f[4 * h + 2]), "=f"(f[4 * h + 3])
                             : "r"(mine + r * 128 + (((2 * piece + h) ^ (r & 7)) * 16))
                             : "memory");
              if (to < tl.row_end && c < p.N) {
                __nv_bfloat16* dst = p.y + static_cast<long long>(to) * p.ldy + c;
                const __nv_bfloat16* res = p.residual ? p.residual + static_cast<long long>(to) * p.ldr + c : nullptr;
                if (p.vec_ok && c + 8 <= p.N) {
                  if (res) {
                    const uint4 raw = *reinterpret_cast<const uint4*>(res);
                    const __nv_bfloat162* b = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                      const float2 a = __bfloat1622float2(b[k]);
                      f[2 * k] += a.x;
                      f[2 * k + 1] += a.y;
                    }
                  }
                  *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
                } else {
#pragma unroll
                  for (int k = 0; k < 8; ++k)
                    if (c + k < p.N) dst[k] = __float2bfloat16(f[k] + (res ? __bfloat162float(res[k]) : 0.f));
                }
              }
            }
            __syncwarp();
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn g_encode = nullptr;
std::once_flag g_encode_once;
thread_local std::string g_err;

int fail(const std::string& m) {
  g_err = m;
  return -1;
}

// 8-bit matrix [rows, cols] with boxes of 128 columns, 128-byte swizzle; what lies outside reads as zero
int make_map(CUtensorMap* map, const void* ptr, long long rows, long long cols, long long pitch, int box_rows) {
  std::call_once(g_encode_once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<EncodeTiledFn>(fn);
  });
  if (!g_encode) return fail("cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(BK), static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[2] = {1u, 1u};
  const CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail("cuTensorMapEncodeTiled failed with code " + std::to_string(int(r)));
  return 0;
}

// Shared memory beyond the default, asked for once per kernel and device.
template <typename K>
int allow_smem(K kernel, int bytes, std::atomic<unsigned long long>& asked, int dev) {
  const unsigned long long bit = 1ull << (dev & 63);
  if (asked.load(std::memory_order_acquire) & bit) return 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
    cudaGetLastError();  // (reported here)
    return fail("cudaFuncSetAttribute(MaxDynamicSharedMemorySize) failed");
  }
  asked.fetch_or(bit, std::memory_order_acq_rel);
  return 0;
}

int device_and_sms(int* sms) {
  static std::atomic<int> known[64];
  int dev = 0;
  cudaGetDevice(&dev);
  int n = known[dev & 63].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    known[dev & 63].store(n, std::memory_order_relaxed);
  }
  *sms = n;
  return dev;
}

Args args_of(const Fp8Gemm& g) {
  Args a;
  memset(&a, 0, sizeof(a));
  a.M = g.M;
  a.N = g.N;
  a.K = g.K;
  a.halves = g.q ? 2 : 1;
  a.blocks_n = a.halves * ((g.N / a.halves + 127) / 128);
  a.blocks_k = (g.K + BK - 1) / BK;
  a.xs = g.xs;
  a.ws = g.ws;
  a.groups = g.groups;
  a.max_tiles = g.max_tiles;
  a.tile_group = g.tile_group;
  a.num_tiles = g.num_tiles;
  a.y = static_cast<__nv_bfloat16*>(g.y);
  a.ldy = g.ldy;
  a.residual = static_cast<const __nv_bfloat16*>(g.residual);
  a.ldr = g.ldr;
  a.vec_ok = (g.ldy % 8 == 0 && (reinterpret_cast<uintptr_t>(g.y) & 15) == 0 &&
              (!g.residual || (g.ldr % 8 == 0 && (reinterpret_cast<uintptr_t>(g.residual) & 15) == 0))) ? 1 : 0;
  a.q = g.q;
  a.s = g.s;
  a.status = g.status;
  return a;
}

template <int BN, bool GATED>
int launch(const Fp8Gemm& g, cudaStream_t stream) {
  constexpr int STAGES = BN == 256 ? 4 : 6;
  constexpr int SMEM = STAGES * (BM + BN) * BK + STAGING + 1024;
  CUtensorMap mx, mw;
  if (make_map(&mx, g.x, g.M, g.K, g.ldx, BM)) return -1;
  if (make_map(&mw, g.w, static_cast<long long>(g.groups) * g.N, g.K, g.K, 128)) return -1;
  int sms = 0;
  const int dev = device_and_sms(&sms);
  static std::atomic<unsigned long long> asked{0};
  auto kernel = fp8_gemm_kernel<BN, GATED, STAGES>;
  if (allow_smem(kernel, SMEM, asked, dev)) return -1;
  const Args a = args_of(g);
  const long long m_tiles = g.tile_group ? g.max_tiles : (g.M + BM - 1) / BM;
  const int cols = GATED ? BN / 2 : BN;
  const long long tiles = m_tiles * ((g.N / a.halves + cols - 1) / cols);
  if (tiles > 0x7fffffffll) return fail("too many tiles");
  kernel<<<static_cast<int>(tiles < sms ? tiles : sms), THREADS, SMEM, stream>>>(mx, mw, a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(std::string("fp8 gemm launch failed: ") + cudaGetErrorString(e));
  return 0;
}

}  // namespace

const char* fp8_last_error() { return g_err.c_str(); }

int fp8_gemm_launch(const Fp8Gemm& g, cudaStream_t stream) {
  if (g.M <= 0 || g.N <= 0) return 0;
  if (g.tile_group && g.max_tiles <= 0) return 0;
  if (g.q) return launch<256, true>(g, stream);
  const long long m_tiles = g.tile_group ? g.max_tiles : (g.M + BM - 1) / BM;
  return m_tiles * ((g.N + 255) / 256) >= 148 ? launch<256, false>(g, stream) : launch<128, false>(g, stream);
}

}  // namespace mb
