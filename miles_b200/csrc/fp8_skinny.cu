// Products of few 8-bit rows with block-scaled 8-bit weights: decode steps, experts of a few rows, short prompts. The formula is that of
// fp8_gemm.cu.
//
// They are bound by the bytes of W, and by how many of them are on their way from how many SMs. So 128 rows of W are the tensor core's M and
// the rows of x its N (16, 32, 64 or 128): no part of a tile is padding that has to be streamed. A block of 128 along K is one stage, one
// buffer of TMEM and four tcgen05.mma; warps add it to sums in registers, a row of W a thread, times the weights' scale and the scale
// of each column's row of x, which a warp lays out in shared memory a block ahead. The blocks of a tile are shared by a cluster of up to
// eight CTAs, whose sums meet in distributed shared memory in rank order, so results do not depend on timing. A gate-up weight's CTA
// streams 128 gate rows and their 128 up rows, which are a whole block of silu(gate) * up: a warp finds its largest value by shuffles.
//
// Measured, us (the bytes of W alone at 6.5 TB/s): one row 5120 x 2048 5.3 (1.6), 23 rows 2560 x 9728 9.3 (3.8), 64 rows 6144 x 4096 11.3 (3.9);
// 128 experts, 64 tokens by eight: gate-up 1536 x 2048 70 (61).
//
//   warp 0     : TMA producer (128-byte swizzle)          warp 1 : TMEM allocator, tcgen05.mma issuer
//   the others : four warps, or eight for 128 columns, TMEM -> sums in registers -> shared memory, cluster sum, store
#include <cuda.h>
#include <string.h>

#include "fp8_tile.cuh"
#include "pdl.cuh"

namespace mb {
namespace {

constexpr int BM = 128, BK = 128;
constexpr int W_BYTES = BM * BK;
constexpr int MAX_STAGES = 12;

struct Args {
  int M, N;
  int halves, blocks_n, blocks_k;  // of a matrix; blocks of its scales
  int per_rank, stages;            // blocks of each CTA of the cluster; stages of its ring
  const float* xs;
  const float* ws;
  int groups, max_tiles;
  const int* tile_group;
  const int* num_tiles;
  __nv_bfloat16* y;
  long long ldy;
  const __nv_bfloat16* residual;
  long long ldr;
  int vec_y, vec_r;                // 8-byte accesses fit
  uint8_t* q;
  float* s;
  int* status;
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
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float4 ld_rank_f4(uint32_t local_addr, uint32_t rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(map_to_rank(local_addr, rank)) : "memory");
  return v;
}

// TMEM columns of a CTA. Its shared memory is at least the same part of an SM's: then CTAs that fit an SM together have room in its TMEM
// together, whatever their kernels, and none of a cluster waits there for a CTA of a cluster that waits for it elsewhere.
template <int NT, bool GATED>
struct Shape {
  static constexpr int G = GATED ? 2 : 1;
  static constexpr int BUFS = NT * G <= 32 ? 4 : 2;
  static constexpr int TMEM = BUFS * NT * G;
  static constexpr int MIN_SMEM = TMEM * 228 * 2;  // TMEM / 512 of 228 KB
  static constexpr int EPI_WARPS = NT * G >= 128 ? 8 : 4;  // (128 rows of x, us a block: four 0.69, eight 0.61)
  static constexpr int COLS = NT * 4 / EPI_WARPS;     // rows of x that a warp sums up
  static constexpr int THREADS = 64 + 32 * EPI_WARPS;
  static constexpr int STAGE = G * W_BYTES + NT * BK;
  static constexpr int PART = NT * BM * 4;         // a CTA's sums of one matrix, over the ring
};

template <int NT, bool GATED>
__global__ void __launch_bounds__(Shape<NT, GATED>::THREADS, Shape<NT, GATED>::TMEM <= 128 ? 2 : 1)
fp8_skinny_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const Args p) {
  using S = Shape<NT, GATED>;
  constexpr int G = S::G, BUFS = S::BUFS, STAGE = S::STAGE, PART = S::PART, COLS = S::COLS, EPI_WARPS = S::EPI_WARPS;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  __shared__ __align__(8) unsigned long long bars[2 * MAX_STAGES + 2 * BUFS];
  __shared__ __align__(16) float scales_s[EPI_WARPS][2][G * COLS];  // of a warp's current block and the next
  __shared__ uint32_t tmem_slot_s;
  __shared__ int abort_s;
  volatile int* abort_flag = &abort_s;
  const uint32_t bar0 = smem_u32(bars);
  auto full_bar = [&](int s) { return bar0 + 8u * s; };
  auto empty_bar = [&](int s) { return bar0 + 8u * (MAX_STAGES + s); };
  auto tfull_bar = [&](int b) { return bar0 + 8u * (2 * MAX_STAGES + b); };
  auto tempty_bar = [&](int b) { return bar0 + 8u * (2 * MAX_STAGES + BUFS + b); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank(), ranks = cluster_size();
  const int n0 = blockIdx.y * BM, half_n = p.N / p.halves;
  const int kb0 = min(p.blocks_k, static_cast<int>(rank) * p.per_rank);
  const int blocks = min(p.blocks_k, kb0 + p.per_rank) - kb0;

  if (threadIdx.x == 0) {
    abort_s = 0;
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < BUFS; ++b) {
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), EPI_WARPS);
    }
    fence_barrier_init();
    prefetch_tensormap(&map_w);
    prefetch_tensormap(&map_x);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_slot_s), S::TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_slot_s);
  // one matrix for all rows: the first stages of it on their way into L2 while the predecessor finishes
  if (!p.tile_group && warp == 0 && lane == 0)
    for (int b = 0; b < min(blocks, p.stages); ++b) {
      tma_prefetch_2d(&map_w, (kb0 + b) * BK, n0);
      if (GATED) tma_prefetch_2d(&map_w, (kb0 + b) * BK, half_n + n0);
    }
  pdl_enter();

  int row0 = blockIdx.z * NT, rows = min(NT, p.M - row0), group = 0;
  if (p.tile_group) {
    rows = 0;
    if (static_cast<int>(blockIdx.z) < min(*p.num_tiles, p.max_tiles)) {
      const int4 e = reinterpret_cast<const int4*>(p.tile_group)[blockIdx.z];
      group = min(max(e.x, 0), p.groups - 1);
      row0 = min(max(e.y, 0), p.M);
      rows = min(min(max(e.z, 0), 128), p.M - row0);
    }
  }
  const int w0 = group * p.N + n0;

  int stage = 0, buf = 0;  // each role's own
  uint32_t phase = 0, tphase = 0;
  bool ok = true;
  for (int first = 0; first < rows; first += NT) {  // (a row tile of more than NT rows: the weights come from L2 again)
    const int t0 = row0 + first, count = min(NT, rows - first);
    if (warp == 0) {
      if (elect_one()) {
        for (int b = 0; ok && b < blocks; ++b) {
          ok = mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag, p.status, ERR_WAIT_EMPTY);
          if (!ok) break;
          mbar_expect_tx(full_bar(stage), STAGE);
          const uint32_t dst = base + stage * STAGE;
          tma_load_2d(dst, &map_w, full_bar(stage), (kb0 + b) * BK, w0);
          if (GATED) tma_load_2d(dst + W_BYTES, &map_w, full_bar(stage), (kb0 + b) * BK, w0 + half_n);
          tma_load_2d(dst + G * W_BYTES, &map_x, full_bar(stage), (kb0 + b) * BK, t0);
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) {  // copies in flight get a bounded time to land before shared memory is released
          const unsigned long long begun = globaltimer_ns();
          while (globaltimer_ns() - begun < 2000000ull) {
          }
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      if (elect_one()) {
        constexpr uint32_t idesc = f8::idesc_e4m3(BM, NT);
        for (int b = 0; ok && b < blocks; ++b) {
          ok = mbar_wait(full_bar(stage), phase, abort_flag, p.status, ERR_WAIT_FULL) &&
               mbar_wait(tempty_bar(buf), tphase ^ 1u, abort_flag, p.status, ERR_WAIT_TMEM_EMPTY);
          if (!ok) break;
          tc_fence_after();
          const uint32_t w = base + stage * STAGE, x = w + G * W_BYTES;
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int k = 0; k < BK / 32; ++k)
              umma_f8(tmem + (buf * G + g) * NT, make_smem_desc(w + g * W_BYTES + k * 32, 16, 1024), make_smem_desc(x + k * 32, 16, 1024), idesc, k > 0 ? 1u : 0u);
          umma_commit(empty_bar(stage));
          umma_commit(tfull_bar(buf));
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
          }
          if (++buf == BUFS) {
            buf = 0;
            tphase ^= 1u;
          }
        }
      }
      __syncwarp();
    } else {
      const int quad = warp & 3, c0 = (warp - 2) / 4 * COLS;  // rows of W that this warp reaches in TMEM; its rows of x
      constexpr int PER = COLS >= 32 ? COLS / 32 : 1;         // of which a lane fetches the scales of these
      const float* xs[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) xs[j] = p.xs + static_cast<long long>(min(t0 + c0 + min(lane + 32 * j, COLS - 1), p.M - 1)) * p.blocks_k + kb0;
      const float* ws0 = p.ws + (static_cast<long long>(group) * p.blocks_n + n0 / 128) * p.blocks_k + kb0;
      const float* ws1 = ws0 + (GATED ? static_cast<long long>(p.blocks_n / 2) * p.blocks_k : 0);
      float acc[G][COLS];
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < COLS; ++i) acc[g][i] = 0.f;
      float xn[PER], wn0 = 0.f, wn1 = 0.f;
#pragma unroll
      for (int j = 0; j < PER; ++j) xn[j] = 0.f;
      if (blocks > 0) {
#pragma unroll
        for (int j = 0; j < PER; ++j) xn[j] = xs[j][0];
        wn0 = ws0[0];
        if (GATED) wn1 = ws1[0];
      }
      const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
      for (int b = 0; b < blocks; ++b) {
        float* mine = scales_s[warp - 2][b & 1];
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (COLS >= 32 || lane < COLS) {
            mine[lane + 32 * j] = xn[j] * wn0;
            if (GATED) mine[COLS + lane + 32 * j] = xn[j] * wn1;
          }
        __syncwarp();
        if (b + 1 < blocks) {
#pragma unroll
          for (int j = 0; j < PER; ++j) xn[j] = xs[j][b + 1];
          wn0 = ws0[b + 1];
          if (GATED) wn1 = ws1[b + 1];
        }
        // (a wait that runs out shows in `ok` at the end; what is read meanwhile is thrown away, and every later wait ends at once)
        ok = mbar_wait(tfull_bar(buf), tphase, abort_flag, p.status, ERR_WAIT_TMEM_FULL) && ok;
        __syncwarp();
        tc_fence_after();
        constexpr int CH = COLS >= 32 ? 32 : 16;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int c = 0; c < COLS; c += CH) {
            uint32_t d[CH];
            if constexpr (CH == 32) {
              tmem_ld_32x32(tmem + (buf * G + g) * NT + lanes + c0 + c, d);
              f8::tmem_ld_wait_for(d);
            } else {
              tmem_ld_32x16(tmem + (buf * G + g) * NT + lanes + c0 + c, d);
              f8::tmem_ld_wait_for(d);
            }
#pragma unroll
            for (int i = 0; i < CH; i += 4) {
              const float4 s = *reinterpret_cast<const float4*>(mine + g * COLS + c + i);
              acc[g][c + i] = fmaf(s.x, __uint_as_float(d[i]), acc[g][c + i]);
              acc[g][c + i + 1] = fmaf(s.y, __uint_as_float(d[i + 1]), acc[g][c + i + 1]);
              acc[g][c + i + 2] = fmaf(s.z, __uint_as_float(d[i + 2]), acc[g][c + i + 2]);
              acc[g][c + i + 3] = fmaf(s.w, __uint_as_float(d[i + 3]), acc[g][c + i + 3]);
            }
          }
        tc_fence_before();
        if (lane == 0) mbar_arrive(tempty_bar(buf));  // (the wait for the loads was the whole warp's)
        if (++buf == BUFS) {
          buf = 0;
          tphase ^= 1u;
        }
      }
      // the sums of this CTA's blocks -> shared memory [matrix][row of x][row of W], over the ring: its last stage has been multiplied
      if (f8::all_got(ok)) {
        const uint32_t dst = base + c0 * (BM * 4) + (quad * 32 + lane) * 4;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int i = 0; i < COLS; ++i)
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(dst + g * PART + i * (BM * 4)), "f"(acc[g][i]) : "memory");
      }
    }
    // every thread of every CTA of the cluster arrives, whatever happened before
    __syncthreads();
    cluster_sync_all();
    if (warp >= 2) {
      const int n = n0 + lane * 4;
      for (int t = static_cast<int>(rank) + static_cast<int>(ranks) * (warp - 2); t < count; t += static_cast<int>(ranks) * EPI_WARPS) {
        float f[G][4];
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint32_t src = base + g * PART + t * (BM * 4) + lane * 16;
          float4 part[8];
#pragma unroll
          for (uint32_t r = 0; r < 8; ++r)
            if (r < ranks) part[r] = ld_rank_f4(src, r);
          f[g][0] = part[0].x, f[g][1] = part[0].y, f[g][2] = part[0].z, f[g][3] = part[0].w;
#pragma unroll
          for (uint32_t r = 1; r < 8; ++r)
            if (r < ranks) f[g][0] += part[r].x, f[g][1] += part[r].y, f[g][2] += part[r].z, f[g][3] += part[r].w;
        }
        const long long row = t0 + t;
        if constexpr (GATED) {
          float a[4], amax = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            a[i] = n + i < half_n ? f8::silu(f[0][i]) * f[1][i] : 0.f;
            amax = f8::max_nan(amax, fabsf(a[i]));
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) amax = f8::max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
          const float s = f8::scale_of(amax), inv = 1.f / s;
          if (n < half_n) *reinterpret_cast<uint32_t*>(p.q + row * half_n + n) = f8::pack_e4m3(a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv);
          if (lane == 0) p.s[row * ((half_n + 127) / 128) + n0 / 128] = s;
        } else {
          __nv_bfloat16* dst = p.y + row * p.ldy + n;
          const __nv_bfloat16* res = p.residual ? p.residual + row * p.ldr + n : nullptr;
          if (res) {
            if (p.vec_r && n + 4 <= p.N) {
              const uint2 raw = *reinterpret_cast<const uint2*>(res);
              const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.x));
              const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.y));
              f[0][0] += a.x, f[0][1] += a.y, f[0][2] += b.x, f[0][3] += b.y;
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (n + i < p.N) f[0][i] += __bfloat162float(res[i]);
            }
          }
          if (p.vec_y && n + 4 <= p.N) {
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(f[0][0], f[0][1]), pack_bf16(f[0][2], f[0][3]));
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (n + i < p.N) dst[i] = __float2bfloat16(f[0][i]);
          }
        }
      }
      fence_proxy_async();  // the next rows' copies write where these sums were read
    }
    __syncthreads();
    cluster_sync_all();  // no CTA goes on, or leaves, while another reads its sums
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, S::TMEM);
  }
}

// CTAs that share the blocks of a tile: while each keeps two and all that have rows are resident at once (by expert: at most a tile for
// every row, and no more than the list has room for). Clusters of eight do not all find room at one CTA an SM: 128 rows, 2048 x 4096 16.2 us
// against 10.7 for twice the rows in clusters of four.
int split_of(const Fp8Gemm& g, long long z, int n_tiles, int blocks_k, int sms, int per_sm) {
  const long long live = g.tile_group && g.M < z ? g.M : z;
  const int resident = sms * per_sm;
  int split = 1;
  while (split < (per_sm == 1 ? 4 : 8) && live * n_tiles * split * 2 <= resident && blocks_k >= split * 2 * 2) split *= 2;
  return split;
}

// Rows of x in a tile. Experts are not equally liked: half as many again as the average fit, four times as many where the average is four at most
// (gate-up experts of 64 tokens 69 us, with tiles of 32 rows 75).
int rows_of_tile(const Fp8Gemm& g) {
  if (!g.tile_group) return g.M <= 16 ? 16 : g.M <= 32 ? 32 : g.M <= 64 || g.q ? 64 : 128;
  const long long live = g.groups < g.M ? g.groups : g.M;
  if (g.M <= 4 * live) return 16;
  const long long rows = (static_cast<long long>(g.M) + g.M / 2) / live;
  return rows <= 32 ? 32 : rows <= 64 || g.q ? 64 : 128;
}

template <int NT, bool GATED>
int launch(const Fp8Gemm& g, cudaStream_t stream) {
  using S = Shape<NT, GATED>;
  CUtensorMap mx, mw;
  if (fp8_make_map(&mx, g.x, g.M, g.K, g.ldx, NT)) return -1;
  if (fp8_make_map(&mw, g.w, static_cast<long long>(g.groups) * g.N, g.K, g.K, BM)) return -1;
  int sms = 0;
  const int dev = fp8_device(&sms);
  static std::atomic<unsigned long long> asked{0};
  auto kernel = fp8_skinny_kernel<NT, GATED>;
  constexpr int MOST = S::TMEM <= 128 ? 108 * 1024 : 216 * 1024;  // two CTAs an SM, or one
  if (fp8_allow_smem(kernel, MOST, asked, dev)) return -1;
  Args a;
  memset(&a, 0, sizeof(a));
  a.M = g.M;
  a.N = g.N;
  a.halves = S::G;
  a.blocks_n = S::G * ((g.N / S::G + BM - 1) / BM);
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
  a.vec_y = g.ldy % 4 == 0 && (reinterpret_cast<uintptr_t>(g.y) & 7) == 0;
  a.vec_r = g.ldr % 4 == 0 && (reinterpret_cast<uintptr_t>(g.residual) & 7) == 0;
  a.q = g.q;
  a.s = g.s;
  a.status = g.status;
  const int n_tiles = (g.N / S::G + BM - 1) / BM;
  const long long z = g.tile_group ? g.max_tiles : (g.M + NT - 1) / NT;
  const int split = split_of(g, z, n_tiles, a.blocks_k, sms, S::TMEM <= 128 ? 2 : 1);
  a.per_rank = (a.blocks_k + split - 1) / split;
  int stages = (MOST - 1024) / S::STAGE;
  if (stages > MAX_STAGES) stages = MAX_STAGES;
  if (stages > a.per_rank) stages = a.per_rank;
  if (stages < 2) stages = 2;
  a.stages = stages;
  int smem = stages * S::STAGE;
  if (smem < S::G * S::PART) smem = S::G * S::PART;
  smem += 1024;
  if (smem < S::MIN_SMEM) smem = S::MIN_SMEM;
  if (n_tiles > 65535 || z > 65535) return fp8_fail("too many tiles");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(split, n_tiles, static_cast<unsigned>(z));
  cfg.blockDim = dim3(S::THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, mx, mw, a);
  if (e != cudaSuccess) {
    cudaGetLastError();  // (reported here)
    return fp8_fail(std::string("fp8 skinny gemm launch failed: ") + cudaGetErrorString(e));
  }
  return 0;
}

}  // namespace

// Few rows, or few tiles: by what either kernel costs, us. Pairs (fp8_gemm.cu) take 4.5 us and, for each round of their tiles over the SMs, 0.48 a
// block of 128 along K and 1.2 at its end (2.5 with SwiGLU; by expert 2 more to join row tiles). The CTAs here take 5.7 and, a round, 0.61 to
// 0.75 a block where one fits an SM; where two do, 3 and 3 a round, and 0.45 a block; or what the blocks of all of them need to arrive.
// Measured, us, pairs / here: 24576 x 4096 gate-up, 64 rows 40 / 30, 128 rows 41 / 56; 6144 x 4096, 128 rows 21 / 16, 512 22 / 52; 4096 x 12288, 256
// rows 50 / 36, 512 50 / 66; 128 experts, gate-up 1536 x 2048, 16 rows each 114 / 80, 64 117 / 144, 2048 x 768, 16 rows 68 / 58, 48 69 / 119.
bool fp8_is_skinny(const Fp8Gemm& g) {
  if (g.M <= 0) return true;
  int sms = 0;
  fp8_device(&sms);
  const int G = g.q ? 2 : 1, n = g.N / G, blocks_k = (g.K + BK - 1) / BK, nt = rows_of_tile(g);
  const long long live = g.M < g.groups ? g.M : g.groups;  // experts with rows
  if (g.tile_group && (g.M > live * 2 * nt / 3 || g.max_tiles > 65535)) return false;  // (more rows than such tiles hold)
  const long long pairs = (g.tile_group ? live + g.M / 256 : (g.M + 255) / 256) * ((n + 256 / G - 1) / (256 / G));
  const long long z = g.tile_group ? live : (g.M + nt - 1) / nt;
  const int n_tiles = (n + BM - 1) / BM, per_sm = nt * G < 128 ? 2 : 1, resident = sms * per_sm;
  if (z > 65535 || n_tiles > 65535) return false;
  const int split = split_of(g, z, n_tiles, blocks_k, sms, per_sm);
  const long long ctas = z * n_tiles * split;
  const double arrive = static_cast<double>(ctas < resident ? ctas : resident) * G * W_BYTES / 6.0e6;
  const double alone = nt * G < 128 ? 0.45 : G == 2 ? 0.75 : 0.61, block = arrive > alone ? arrive : alone;
  const double rounds = static_cast<double>((ctas + resident - 1) / resident), own = (blocks_k + split - 1) / split * block;
  const double here = per_sm == 1 ? rounds * (5.7 + own) : 3.0 + rounds * (3.0 + own);
  const double there = (g.tile_group ? 6.5 : 4.5) + static_cast<double>((2 * pairs + sms - 1) / sms) * (0.48 * blocks_k + (G == 2 ? 2.5 : 1.2));
  return here <= there;
}

int fp8_grouped_launches(long long rows, int groups, int N, int K, bool gated, int max_tiles) {
  if (rows <= 0 || max_tiles <= 0) return 0;
  static uint8_t some[16];  // (which kernel it is does not depend on what lies where)
  Fp8Gemm g{};
  g.M = static_cast<int>(rows);
  g.N = N;
  g.K = K;
  g.groups = groups;
  g.max_tiles = max_tiles;
  g.tile_group = reinterpret_cast<const int*>(some);
  if (gated) g.q = some;
  return fp8_is_skinny(g) ? 1 : 2;
}

int fp8_skinny_launch(const Fp8Gemm& g, cudaStream_t stream) {
  const int nt = rows_of_tile(g);
  if (g.q) return nt == 16 ? launch<16, true>(g, stream) : nt == 32 ? launch<32, true>(g, stream) : launch<64, true>(g, stream);
  if (nt == 16) return launch<16, false>(g, stream);
  if (nt == 32) return launch<32, false>(g, stream);
  return nt == 64 ? launch<64, false>(g, stream) : launch<128, false>(g, stream);
}

}  // namespace mb
