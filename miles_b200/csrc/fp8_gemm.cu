// Products of 8-bit rows with block-scaled 8-bit weights for sm_100a:
//
//   y[t, n] = (residual[t, n] +) sum over blocks b of 128 along K of  xs[t, b] ws[n / 128, b] sum over k in b of x[t, k] w[n, k]
//
// in E4M3 with fp32 scales of any value, so that no scale can ride in the tensor core's own (power-of-two) ones: a block's product is
// computed by four tcgen05.mma into a TMEM buffer of its own, and warps add it, scaled, to sums in registers (fp32) while the tensor core fills the
// other buffer. The rows are one batch, or sorted by expert (row tiles {matrix, first row, rows} as the router's sort leaves them). A gate-up
// weight's tile takes 128 gate rows and their 128 up rows, so that silu(gate) * up leaves as a whole block of 128 columns of 8-bit rows,
// scaled by their largest value, without passing through memory in between.
//
// A pair of CTAs (`cta_group::2`) computes 256 rows x 256 columns, each CTA its 128 rows. A block takes the tensor core 512 clocks alone (336 ns
// at the clock that the power allows then). Shared memory is as busy: 32 KB of operands arrive and 32 KB are read at 128 bytes a
// clock; products and copies together take 460 ns, with the loads from TMEM 500, with the additions 580 (a library's e4m3 product with one scale
// a matrix, which adds nothing up, 430). So nothing else may pass there: the scales of the rows, which 512 threads would
// fetch from 128 lines (225 -> 374 ns a block for the hand-over of buffers alone), are fetched by two warps, eight blocks at a time, which
// leave the products of both scales as the readers want them; and one instruction multiplies all 256 columns, since two of 128 read x
// twice (617 ns). An arrival at the other CTA's barrier is a relaxed one: releasing there costs 1200 to 1900 clocks.
//
//   warp 0      : TMA producer (128-byte swizzle)          warp 1 : TMEM allocator, tcgen05.mma issuer
//   warps 2, 3  : scales of the rows times the weights', eight blocks ahead
//   warps 4..19 : sums in registers, a row and 64 columns a thread, then rows through shared memory
//
// y leaves in boxes of 32 rows x 64 columns by asynchronous stores that nobody waits for until the warp's next box (their 32 KB more take a stage of
// operands; with stores by threads, from half of that: 87 -> 73 us at 32768 x 2048 x 768, 129 -> 118 at K = 1536, 146 -> 143 at 8192 x 2048 x
// 8192). An expert's last rows, with another's behind them in the box, and rows of y that do not begin or end at 16 bytes are stored by threads.
//
// Measured, us: 8192 x 24576 x 4096 gate-up 942 (1750 TFLOP/s), 8192 x 4096 x 4096 with residual 142 (160 in a long run, at the clock that its
// power leaves), experts of 65536 rows, 128 of 1536 x 2048 gate-up 341, 2048 x 768 199.
//
// Reference counterpart: the block-wise FP8 GEMMs of the serving engines that load its FP8 checkpoints (weight_block_size [128, 128]:
// miles/backends/megatron_utils/megatron_to_hf/processors/quantizer_fp8.py, miles/utils/fp8_kernel.py:24-79).
#include <cuda.h>
#include <string.h>

#include <mutex>
#include <type_traits>

#include "fp8_tile.cuh"
#include "pdl.cuh"

namespace mb {
namespace {

constexpr int BM = 128, BN = 256, BK = 128;  // rows of a CTA, columns of its pair's tile (W rows), columns of a block
constexpr int COLS = 64;                     // of a thread
constexpr int BUFS = 2;
constexpr int X_BYTES = BM * BK, W_BYTES = BN / 2 * BK;  // of a stage: this CTA's rows of x, and of W
constexpr int STAGE = X_BYTES + W_BYTES;
constexpr int EPI_WARPS = 16;
constexpr int THREADS = 128 + 32 * EPI_WARPS;  // the first warpgroup gives registers to the others, which sum up
constexpr int AHEAD = 8, SLOTS = 2;          // blocks of scales in a slot
constexpr int SLOT_BYTES = 2 * AHEAD * BM * 4;
// Stages, and what a warp has to stage its 32 rows: whole rows of y leave by asynchronous stores, which the next tile need not wait for.
template <bool GATED>
struct Room {
  static constexpr int STAGES = GATED ? 5 : 4, WARP = GATED ? 2048 : 4096;
  static constexpr int SMEM = STAGES * STAGE + EPI_WARPS * WARP + SLOTS * SLOT_BYTES + 1024;
};

struct Args {
  int M, N, K;
  int halves, blocks_n, blocks_k;  // of a matrix; blocks of its scales
  const float* xs;
  const float* ws;
  int groups, max_tiles;
  const int4* tiles;               // {matrix, first row, rows, 0}: at most 256 rows each
  const int* num_tiles;
  __nv_bfloat16* y;
  long long ldy;
  const __nv_bfloat16* residual;
  long long ldr;
  int vec_y, vec_r, vec_s;         // 16-byte accesses fit: of y and the residual, boxes
  uint8_t* q;
  float* s;
  int* status;
};

struct Tile {
  int row0, row_end, n0, group;  // rows of x; first column of y (or of silu(gate) * up)
};

__device__ __forceinline__ void umma_f8_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t"
      "}\n"
      :
      : "r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void st_shared(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 ld_shared(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

template <bool GATED>
__device__ __forceinline__ int column_tiles(const Args& p) {
  constexpr int W = GATED ? BN / 2 : BN;
  return (p.N / p.halves + W - 1) / W;
}
template <bool GATED>
__device__ __forceinline__ int tiles_of(const Args& p) {
  const int m = p.tiles ? min(max(*p.num_tiles, 0), p.max_tiles) : (p.M + 2 * BM - 1) / (2 * BM);
  return m * column_tiles<GATED>(p);
}
template <bool GATED>
__device__ __forceinline__ Tile tile_at(const Args& p, int t) {
  const int n_tiles = column_tiles<GATED>(p);
  Tile r;
  int mt = t / n_tiles, nt = t - mt * n_tiles;
  if (p.tiles) {
    const int4 e = p.tiles[mt];
    r.group = e.x;
    r.row0 = e.y;
    r.row_end = e.y + e.z;
  } else {
    // bands of four row tiles, their columns outermost: pairs that run together share tiles of W in L2
    constexpr int BAND = 4;
    const int m_tiles = (p.M + 2 * BM - 1) / (2 * BM);
    const int band = t / (BAND * n_tiles), first = band * BAND;
    const int rows = min(m_tiles - first, BAND), in_band = t - band * BAND * n_tiles;
    mt = first + in_band % rows;
    nt = in_band / rows;
    r.group = 0;
    r.row0 = mt * 2 * BM;
    r.row_end = min(p.M, r.row0 + 2 * BM);
  }
  r.n0 = nt * (GATED ? BN / 2 : BN);
  return r;
}

template <bool GATED>
__global__ void __launch_bounds__(THREADS, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_y,
                const __grid_constant__ CUtensorMap map_r, const Args p) {
  constexpr int STAGES = Room<GATED>::STAGES, WARP = Room<GATED>::WARP;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t staging = base + STAGES * STAGE;
  const uint32_t scales = staging + EPI_WARPS * WARP;
  __shared__ __align__(8) unsigned long long bars[2 * STAGES + 2 * BUFS + 2 * SLOTS + 1 + EPI_WARPS];
  __shared__ uint32_t tmem_slot_s;
  __shared__ int abort_s;
  volatile int* abort_flag = &abort_s;
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };                            // of the CTA of rank 0: both CTAs' copies have landed
  auto empty_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto tfull_bar = [&](int b) { return bar0 + 8u * (2 * STAGES + b); };
  auto tempty_bar = [&](int b) { return bar0 + 8u * (2 * STAGES + BUFS + b); };    // of the CTA of rank 0: both CTAs have read the buffer
  auto sfull_bar = [&](int s) { return bar0 + 8u * (2 * STAGES + 2 * BUFS + s); };
  auto sempty_bar = [&](int s) { return bar0 + 8u * (2 * STAGES + 2 * BUFS + SLOTS + s); };
  const uint32_t amax_bar = bar0 + 8u * (2 * STAGES + 2 * BUFS + 2 * SLOTS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int first_tile = blockIdx.x / 2, step = gridDim.x / 2;

  if (threadIdx.x == 0) {
    abort_s = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < BUFS; ++b) {
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), 2 * EPI_WARPS);
    }
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(sfull_bar(s), 2);
      mbar_init(sempty_bar(s), EPI_WARPS);
    }
    mbar_init(amax_bar, 32 * EPI_WARPS);
    for (int w = 0; w < EPI_WARPS; ++w) mbar_init(amax_bar + 8u + 8u * w, 1);
    fence_barrier_init();
    prefetch_tensormap(&map_x);
    prefetch_tensormap(&map_w);
  }
  if (warp == 1) tmem_alloc_pair(smem_u32(&tmem_slot_s), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_slot_s);
  cluster_sync_all();  // both CTAs' barriers and TMEM are there before either uses the other's
  pdl_enter();
  const int total = tiles_of<GATED>(p);
  const int half_n = p.N / p.halves;

  // 4 x 32 x 32 + 16 x 32 x 112 registers are the 640 x 96 of the launch
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
    if (warp == 0) {
      if (elect_one()) {
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int t = first_tile; ok && t < total; t += step) {
          const Tile tl = tile_at<GATED>(p, t);
          const int w0 = tl.group * p.N + tl.n0 + rank * (GATED ? 64 : 128);  // this CTA's rows of W
          for (int kb = 0; kb < p.blocks_k; ++kb) {
            if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, ERR_WAIT_EMPTY)) {
              ok = false;
              break;
            }
            if (rank == 0) mbar_expect_tx(full_bar(stage), 2 * STAGE);
            const uint32_t full = map_to_rank(full_bar(stage), 0), dst = base + stage * STAGE;
            tma_load_2d_pair(dst, &map_x, full, kb * BK, tl.row0 + rank * BM);
            tma_load_2d_pair(dst + X_BYTES, &map_w, full, kb * BK, w0);
            if (GATED) tma_load_2d_pair(dst + X_BYTES + W_BYTES / 2, &map_w, full, kb * BK, w0 + half_n);  // the up rows of its gate rows
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
        for (int s = 0; ok && s < STAGES; ++s) {  // the other CTA's commits have arrived before this one leaves
          ok = mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, ERR_WAIT_EMPTY);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
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
      // (elect.sync tells the compiler that one thread issues: under `lane == 0` a block takes 1040 clocks instead of 512)
      if (rank == 0 && elect_one()) {
        constexpr uint32_t idesc = f8::idesc_e4m3(2 * BM, BN);
        int stage = 0, buf = 0;
        uint32_t phase = 0, tphase = 0;
        bool ok = true;
        for (int t = first_tile; ok && t < total; t += step) {
          for (int kb = 0; ok && kb < p.blocks_k; ++kb) {
            ok = mbar_wait(full_bar(stage), phase, abort_flag, p.status, ERR_WAIT_FULL) &&
                 mbar_wait(tempty_bar(buf), tphase ^ 1u, abort_flag, p.status, ERR_WAIT_TMEM_EMPTY);
            if (!ok) break;
            tc_fence_after();
            const uint32_t x = base + stage * STAGE, w = x + X_BYTES;
#pragma unroll
            for (int k = 0; k < BK / 32; ++k)
              umma_f8_pair(tmem + buf * BN, make_smem_desc(x + k * 32, 16, 1024), make_smem_desc(w + k * 32, 16, 1024), idesc, k > 0 ? 1u : 0u);
            umma_commit_pair(tfull_bar(buf));
            umma_commit_pair(empty_bar(stage));
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
      }
      __syncwarp();
    } else {
      // [slot][half of the columns, or gate and up][block][row]: this warp's 64 rows
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = first_tile; ok && t < total; t += step) {
        const Tile tl = tile_at<GATED>(p, t);
        const int nb = tl.n0 / 128, row = tl.row0 + rank * BM + (warp - 2) * 64 + lane;
        const float* x0 = p.xs + static_cast<long long>(min(row, p.M - 1)) * p.blocks_k;
        const float* x1 = p.xs + static_cast<long long>(min(row + 32, p.M - 1)) * p.blocks_k;
        const float* ws0 = p.ws + (static_cast<long long>(tl.group) * p.blocks_n + nb) * p.blocks_k;
        const float* ws1 = ws0 + static_cast<long long>(GATED ? p.blocks_n / 2 : nb + 1 < p.blocks_n ? 1 : 0) * p.blocks_k;
        for (int kb = 0; ok && kb < p.blocks_k; kb += AHEAD) {
          ok = f8::all_got(mbar_wait(sempty_bar(slot), phase ^ 1u, abort_flag, p.status, ERR_WAIT_EMPTY));
          if (!ok) break;
          const int n = min(AHEAD, p.blocks_k - kb);
          // lanes 0..7 the first weights' scales of the blocks, 8..15 the second's
          const float w = lane < 2 * AHEAD && (lane & (AHEAD - 1)) < n ? (lane < AHEAD ? ws0 : ws1)[kb + (lane & (AHEAD - 1))] : 0.f;
          const uint32_t to = scales + slot * SLOT_BYTES + ((warp - 2) * 64 + lane) * 4;
#pragma unroll
          for (int i = 0; i < AHEAD; i += 4) {
            float a[4], b[4];
            if (p.vec_s) {
              const float4 u = i < n ? *reinterpret_cast<const float4*>(x0 + kb + i) : make_float4(0.f, 0.f, 0.f, 0.f);
              const float4 v = i < n ? *reinterpret_cast<const float4*>(x1 + kb + i) : make_float4(0.f, 0.f, 0.f, 0.f);
              a[0] = u.x, a[1] = u.y, a[2] = u.z, a[3] = u.w, b[0] = v.x, b[1] = v.y, b[2] = v.z, b[3] = v.w;
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                a[k] = i + k < n ? x0[kb + i + k] : 0.f;
                b[k] = i + k < n ? x1[kb + i + k] : 0.f;
              }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float w0 = __shfl_sync(0xffffffffu, w, i + k), w1 = __shfl_sync(0xffffffffu, w, AHEAD + i + k);
              const uint32_t at = to + (i + k) * (BM * 4);
              asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(a[k] * w0) : "memory");
              asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + 128), "f"(b[k] * w0) : "memory");
              asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + SLOT_BYTES / 2), "f"(a[k] * w1) : "memory");
              asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + SLOT_BYTES / 2 + 128), "f"(b[k] * w1) : "memory");
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(sfull_bar(slot));
          if (++slot == SLOTS) {
            slot = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
    // rows of the tile that this warp reaches in TMEM; its part of the columns: 64 of y, or 32 of the gates and 32 of their up columns
    const int quad = warp & 3, part = (warp - 4) >> 2, half = part >> 1;
    const uint32_t mine = staging + (warp - 4) * WARP;
    const uint32_t from0 = tmem + (GATED ? half * (BN / 2) + (part & 1) * 32 : part * COLS) + (static_cast<uint32_t>(quad * 32) << 16);
    constexpr int THEN = GATED ? BN / 4 : 32;  // from its first 32 columns to the others
    const uint32_t my_scales = scales + (GATED ? 0 : half * (SLOT_BYTES / 2)) + (quad * 32 + lane) * 4;
    // Between blocks as few instructions as can be: the additions alone take half of the clocks that the products leave. So a wait that
    // runs out is looked at once a tile (what is read meanwhile is thrown away, and every later wait ends at once), and a buffer is
    // handed back by one lane without a word from the others: the wait for their loads is the whole warp's.
    const uint32_t tempty0 = map_to_rank(tempty_bar(0), 0);
    const auto release = [&](int buf) {
      tc_fence_before();
      if (lane == 0) f8::arrive_relaxed(tempty0 + 8u * buf);
    };
    int buf = 0, slot = 0, tiles_done = 0;
    uint32_t tphase = 0, sphase = 0, rphase = 0;
    const uint32_t residual_bar = amax_bar + 8u + 8u * (warp - 4);
    bool ok = true;
    for (int t = first_tile; t < total; t += step, ++tiles_done) {
      const Tile tl = tile_at<GATED>(p, t);
      const int row0 = tl.row0 + rank * BM + quad * 32, n0 = tl.n0;  // this warp's rows
      const int rows = min(max(tl.row_end - row0, 0), 32);
      const bool ahead = !GATED && p.residual && p.vec_r && rows > 0 && n0 + part * COLS < p.N;
      if (ahead) {  // the residual's box arrives while the sums are formed
        fence_proxy_async();  // (what threads read here for the last tile)
        __syncwarp();
        if (lane == 0) {
          tma_store_wait_read<0>();
          mbar_expect_tx(residual_bar, WARP);
          tma_load_2d(mine, &map_r, residual_bar, n0 + part * COLS, row0);
        }
        __syncwarp();
      }
      float acc[COLS];
#pragma unroll
      for (int i = 0; i < COLS; ++i) acc[i] = 0.f;
#pragma unroll 1
      for (int kb = 0; kb < p.blocks_k; ++kb) {
        const int in_slot = kb & (AHEAD - 1);
        if (in_slot == 0) {
          ok = mbar_wait(sfull_bar(slot), sphase, abort_flag, p.status, ERR_WAIT_FULL) && ok;
          __syncwarp();
        }
        const uint32_t at = my_scales + slot * SLOT_BYTES + in_slot * (BM * 4);
        float c0, c1;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(c0) : "r"(at) : "memory");
        if constexpr (GATED) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(c1) : "r"(at + SLOT_BYTES / 2) : "memory");
        else c1 = c0;
        if (in_slot == AHEAD - 1 || kb + 1 == p.blocks_k) {
          __syncwarp();
          if (lane == 0) mbar_arrive(sempty_bar(slot));
          if (++slot == SLOTS) {
            slot = 0;
            sphase ^= 1u;
          }
        }
        ok = mbar_wait(tfull_bar(buf), tphase, abort_flag, p.status, ERR_WAIT_TMEM_FULL) && ok;
        __syncwarp();
        tc_fence_after();
        uint32_t d[32];
        tmem_ld_32x32(from0 + buf * BN, d);
        f8::tmem_ld_wait_for(d);
#pragma unroll
        for (int i = 0; i < 32; ++i) acc[i] = fmaf(c0, __uint_as_float(d[i]), acc[i]);
        tmem_ld_32x32(from0 + buf * BN + THEN, d);
        f8::tmem_ld_wait_for(d);
        release(buf);
        if (++buf == BUFS) {
          buf = 0;
          tphase ^= 1u;
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) acc[32 + i] = fmaf(c1, __uint_as_float(d[i]), acc[32 + i]);
      }
      ok = f8::all_got(ok);
      if (!ok) break;
      if constexpr (GATED) {
        constexpr int OUT = COLS / 2;
        const int c0 = n0 + part * OUT;
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < OUT; ++i) {
          const float a = c0 + i < half_n ? f8::silu(acc[i]) * acc[OUT + i] : 0.f;
          acc[i] = a;
          amax = f8::max_nan(amax, fabsf(a));
        }
        // The four warps of a row exchange theirs through the second halves of their staging, by turns of the tiles (a warp that
        // writes for a tile has seen all of them arrive for the one before, and so read what is overwritten).
        const uint32_t there = 1024 + (tiles_done & 1) * 128 + lane * 4;
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(mine + there), "f"(amax) : "memory");
        mbar_arrive(amax_bar);
        ok = f8::all_got(mbar_wait(amax_bar, tiles_done & 1, abort_flag, p.status, ERR_WAIT_TMEM_FULL));
        if (!ok) break;
#pragma unroll
        for (int k = 1; k < 4; ++k) {
          float other;
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(other) : "r"(staging + ((part ^ k) * 4 + quad) * WARP + there) : "memory");
          amax = f8::max_nan(amax, other);
        }
        const float s = f8::scale_of(amax);
        // times the reciprocal: the products carry errors of their own that are larger than its
        const float inv = 1.f / s;
        if (part == 0 && lane < rows) p.s[static_cast<long long>(row0 + lane) * ((half_n + 127) / 128) + n0 / 128] = s;
#pragma unroll
        for (int j = 0; j < OUT / 16; ++j) {
          uint32_t v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            v[i] = f8::pack_e4m3(acc[16 * j + 4 * i] * inv, acc[16 * j + 4 * i + 1] * inv, acc[16 * j + 4 * i + 2] * inv, acc[16 * j + 4 * i + 3] * inv);
          st_shared(mine + lane * 32 + ((j ^ ((lane >> 2) & 1)) * 16), make_uint4(v[0], v[1], v[2], v[3]));
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 2; ++i) {  // sixteen rows at a time, two lanes each
          const int r = 16 * i + (lane >> 1), piece = lane & 1;
          const uint4 v = ld_shared(mine + r * 32 + ((piece ^ ((r >> 2) & 1)) * 16));
          if (r < rows && c0 + piece * 16 < half_n) *reinterpret_cast<uint4*>(p.q + static_cast<long long>(row0 + r) * half_n + c0 + piece * 16) = v;
        }
        __syncwarp();
      } else {
        // rows of 128 bytes, 16-byte pieces in places that differ by row (the swizzle of the tensor maps)
        const auto place = [&](int r, int piece) { return mine + r * 128 + ((piece ^ (r & 7)) * 16); };
        const int c0 = n0 + part * COLS;
        if (ahead) {
          ok = f8::all_got(mbar_wait(residual_bar, rphase, abort_flag, p.status, ERR_WAIT_FULL));
          if (!ok) break;
          rphase ^= 1u;
        } else {  // what this warp staged last has been read
          if (lane == 0) tma_store_wait_read<0>();
          __syncwarp();
        }
        if (p.residual) {  // joins the sums before they are rounded
          if (!ahead) {
#pragma unroll 4
            for (int i = 0; i < 64; ++i) {
              const int r = i >> 1, c = (i & 1) * 32 + lane;
              unsigned short v = 0;
              if (r < rows && c0 + c < p.N) v = reinterpret_cast<const unsigned short*>(p.residual)[static_cast<long long>(row0 + r) * p.ldr + c0 + c];
              asm volatile("st.shared.u16 [%0], %1;" ::"r"(place(r, c >> 3) + (c & 7) * 2), "h"(v) : "memory");
            }
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint4 v = ld_shared(place(lane, i));
            const __nv_bfloat162* b = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 f = __bfloat1622float2(b[k]);
              acc[8 * i + 2 * k] += f.x;
              acc[8 * i + 2 * k + 1] += f.y;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float* f = acc + 8 * i;
          st_shared(place(lane, i), make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7])));
        }
        // All 32 rows are of this tile, or the rows of y end with it: the store leaves out what lies outside y.
        if (p.vec_y && (rows == 32 || row0 + rows == p.M)) {
          fence_proxy_async();
          __syncwarp();
          if (lane == 0 && rows > 0 && c0 < p.N) {
            tma_store_2d(&map_y, mine, c0, row0);
            tma_store_commit();
          }
        } else if (p.vec_y && c0 + COLS <= p.N) {  // the last rows of an expert's, with another's behind them
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = 4 * i + (lane >> 3), piece = lane & 7;
            if (r < rows) *reinterpret_cast<uint4*>(p.y + static_cast<long long>(row0 + r) * p.ldy + c0 + piece * 8) = ld_shared(place(r, piece));
          }
        } else {
          __syncwarp();
#pragma unroll 4
          for (int i = 0; i < 64; ++i) {
            const int r = i >> 1, c = (i & 1) * 32 + lane;
            unsigned short v;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(place(r, c >> 3) + (c & 7) * 2) : "memory");
            if (r < rows && c0 + c < p.N) reinterpret_cast<unsigned short*>(p.y)[static_cast<long long>(row0 + r) * p.ldy + c0 + c] = v;
          }
        }
        __syncwarp();
      }
    }
    if (!GATED && lane == 0) {  // shared memory outlives the stores, and where a wait has run out, the residual's box has a bounded time to land
      tma_store_wait<0>();
      if (!ok && p.residual) {
        const unsigned long long t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 2000000ull) {
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // neither CTA leaves while the other's products, copies or arrivals may reach it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// Row tiles of up to 256 rows from those of up to 128: a tile of whole 128 rows takes its successor along if that is the same expert's
// and begins where it ends. One block goes through the list, 1024 at a time: where a run of such tiles began tells whether a tile is
// the first of two.
__global__ void __launch_bounds__(1024)
pair_tiles_kernel(const int* __restrict__ tile_group, const int* __restrict__ num_tiles, int max_tiles, int groups, int M, int4* __restrict__ out,
                  int* __restrict__ count) {
  pdl_enter();
  __shared__ int run_s[32], taken_s[32];
  const int n = min(max(*num_tiles, 0), max_tiles), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const auto entry = [&](int i) {
    int4 e = reinterpret_cast<const int4*>(tile_group)[i];
    e.x = min(max(e.x, 0), groups - 1);
    e.y = min(max(e.y, 0), M);
    e.z = min(min(max(e.z, 0), BM), M - e.y);
    return e;
  };
  const auto follows = [](const int4& a, const int4& b) { return a.x == b.x && a.z == BM && b.y == a.y + BM; };
  int run_before = 0, taken_before = 0;
  for (int i0 = 0; i0 < n; i0 += 1024) {
    const int i = i0 + threadIdx.x;
    int4 e = make_int4(0, 0, 0, 0), next = e;
    bool starts = false, more = false;
    if (i < n) {
      e = entry(i);
      starts = i == 0 || !follows(entry(i - 1), e);
      if (i + 1 < n) {
        next = entry(i + 1);
        more = follows(e, next);
      }
    }
    int run = starts ? i : 0;  // the latest start so far
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run = max(run, v);
    }
    if (lane == 31) run_s[warp] = run;
    __syncthreads();
    run = max(run, run_before);
    for (int w = 0; w < warp; ++w) run = max(run, run_s[w]);
    const bool take = i < n && ((i - run) & 1) == 0;
    const unsigned ballot = __ballot_sync(0xffffffffu, take);
    if (lane == 0) taken_s[warp] = __popc(ballot);
    __syncthreads();
    int at = taken_before + __popc(ballot & ((1u << lane) - 1u));
    for (int w = 0; w < warp; ++w) at += taken_s[w];
    if (take) out[at] = make_int4(e.x, e.y, e.z + (more ? next.z : 0), 0);
    for (int w = 0; w < 32; ++w) {
      run_before = max(run_before, run_s[w]);
      taken_before += taken_s[w];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) *count = taken_before;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn g_encode = nullptr;
std::once_flag g_encode_once;
thread_local std::string g_err;

}  // namespace

int fp8_fail(const std::string& m) {
  g_err = m;
  return -1;
}

// 8-bit matrix [rows, cols] with boxes of 128 columns, 128-byte swizzle; what lies outside reads as zero
int fp8_make_map(CUtensorMap* map, const void* ptr, long long rows, long long cols, long long pitch, int box_rows) {
  std::call_once(g_encode_once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<EncodeTiledFn>(fn);
  });
  if (!g_encode) return fp8_fail("cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(BK), static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[2] = {1u, 1u};
  const CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fp8_fail("cuTensorMapEncodeTiled failed with code " + std::to_string(int(r)));
  return 0;
}

// bf16 matrix [rows, cols] that boxes of 32 rows x 64 columns are stored to or read from
static int fp8_make_bf16_map(CUtensorMap* map, const void* ptr, long long rows, long long cols, long long ld) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
  const cuuint32_t box[2] = {64u, 32u};
  const cuuint32_t estr[2] = {1u, 1u};
  const CUresult r = g_encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fp8_fail("cuTensorMapEncodeTiled failed with code " + std::to_string(int(r)));
  return 0;
}

int fp8_device(int* sms) {
  static std::atomic<int> known[64];
  int dev = 0;
  cudaGetDevice(&dev);
  int n = known[dev & 63].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess) {
      known[dev & 63].store(n, std::memory_order_relaxed);
    } else {  // (no device: what is asked then is only which kernel would run)
      cudaGetLastError();
      n = 148;
    }
  }
  *sms = n;
  return dev;
}

namespace {

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
  a.y = static_cast<__nv_bfloat16*>(g.y);
  a.ldy = g.ldy;
  a.residual = static_cast<const __nv_bfloat16*>(g.residual);
  a.ldr = g.ldr;
  // (an asynchronous store ends at the 16 bytes that hold the last column, so N is a multiple of 8 elements too)
  a.vec_y = !g.q && g.N % 8 == 0 && g.ldy % 8 == 0 && (reinterpret_cast<uintptr_t>(g.y) & 15) == 0;
  a.vec_r = g.N % 8 == 0 && g.ldr % 8 == 0 && (reinterpret_cast<uintptr_t>(g.residual) & 15) == 0;
  a.vec_s = a.blocks_k % 4 == 0 && (reinterpret_cast<uintptr_t>(g.xs) & 15) == 0;
  a.q = g.q;
  a.s = g.s;
  a.status = g.status;
  return a;
}

template <bool GATED>
int launch(const Fp8Gemm& g, cudaStream_t stream) {
  constexpr int SMEM = Room<GATED>::SMEM;
  CUtensorMap mx, mw, my, mr;
  if (fp8_make_map(&mx, g.x, g.M, g.K, g.ldx, BM)) return -1;
  if (fp8_make_map(&mw, g.w, static_cast<long long>(g.groups) * g.N, g.K, g.K, GATED ? 64 : 128)) return -1;
  int sms = 0;
  const int dev = fp8_device(&sms);
  static std::atomic<unsigned long long> asked{0};
  auto kernel = fp8_gemm_kernel<GATED>;
  if (fp8_allow_smem(kernel, SMEM, asked, dev)) return -1;
  Args a = args_of(g);
  memset(&my, 0, sizeof(my));
  memset(&mr, 0, sizeof(mr));
  if (a.vec_y && fp8_make_bf16_map(&my, g.y, g.M, g.N, g.ldy)) return -1;
  if (a.residual && a.vec_r && fp8_make_bf16_map(&mr, g.residual, g.M, g.N, g.ldr)) return -1;
  if (g.tile_group) {
    a.tiles = reinterpret_cast<const int4*>(g.workspace);
    a.num_tiles = static_cast<const int*>(g.workspace) + 4ll * g.max_tiles;
    const cudaError_t e = pdl_launch(pair_tiles_kernel, dim3(1), dim3(1024), 0, stream, g.tile_group, g.num_tiles, g.max_tiles, g.groups, g.M,
                                     static_cast<int4*>(g.workspace), static_cast<int*>(g.workspace) + 4ll * g.max_tiles);
    if (e != cudaSuccess) {
      cudaGetLastError();  // (reported here)
      return fp8_fail(std::string("pair_tiles launch failed: ") + cudaGetErrorString(e));
    }
  }
  const long long m_tiles = g.tile_group ? g.max_tiles : (g.M + 2 * BM - 1) / (2 * BM);
  const int cols = GATED ? BN / 2 : BN;
  const long long tiles = m_tiles * ((g.N / a.halves + cols - 1) / cols);
  if (tiles > 0x3fffffffll) return fp8_fail("too many tiles");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * (tiles < sms / 2 ? tiles : sms / 2)));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, mx, mw, my, mr, a);
  if (e != cudaSuccess) {
    cudaGetLastError();  // (reported here)
    return fp8_fail(std::string("fp8 gemm launch failed: ") + cudaGetErrorString(e));
  }
  return 0;
}

}  // namespace

const char* fp8_last_error() { return g_err.c_str(); }

long long fp8_gemm_workspace(const Fp8Gemm& g) { return g.tile_group && !fp8_is_skinny(g) ? 16ll * g.max_tiles + 16 : 0; }

int fp8_gemm_launch(const Fp8Gemm& g, cudaStream_t stream) {
  if (g.M <= 0 || g.N <= 0) return 0;
  if (g.tile_group && g.max_tiles <= 0) return 0;
  if (fp8_is_skinny(g)) return fp8_skinny_launch(g, stream);
  return g.q ? launch<true>(g, stream) : launch<false>(g, stream);
}

}  // namespace mb
