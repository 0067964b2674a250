// What the kernels of 8-bit products share.
#pragma once
#include <atomic>
#include <string>

#include "fp8_block.h"
#include "fp8_math.cuh"
#include "ptx.cuh"

namespace mb {

// ---- host side (fp8_gemm.cu)
int fp8_fail(const std::string& m);  // the message of a failed call; -1
// Tensor map of an 8-bit matrix [rows, cols] with boxes of 128 columns, 128-byte swizzle; what lies outside reads as zero.
int fp8_make_map(CUtensorMap* map, const void* ptr, long long rows, long long cols, long long pitch, int box_rows);
int fp8_device(int* sms);            // the current device and its SMs
int fp8_skinny_launch(const Fp8Gemm& g, cudaStream_t stream);  // fp8_skinny.cu
bool fp8_is_skinny(const Fp8Gemm& g);

// Shared memory beyond the default, asked for once per kernel and device.
template <typename K>
int fp8_allow_smem(K kernel, int bytes, std::atomic<unsigned long long>& asked, int dev) {
  const unsigned long long bit = 1ull << (dev & 63);
  if (asked.load(std::memory_order_acquire) & bit) return 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
    cudaGetLastError();  // (reported here)
    return fp8_fail("cudaFuncSetAttribute(MaxDynamicSharedMemorySize) failed");
  }
  asked.fetch_or(bit, std::memory_order_acq_rel);
  return 0;
}

// ---- device side
namespace f8 {

// Instruction descriptor of kind::f8f6f4: fp32 accumulators (bit 4), E4M3 operands (0 at bits 7 and 10), both K-major.
__host__ __device__ constexpr uint32_t idesc_e4m3(int m, int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// The wait of a load from TMEM names its registers, so that nothing that reads them moves ahead of it while the next load is under way.
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]),
                 "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29])
               :
               : "memory");
  asm volatile("" : "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
// Whether every thread of the warp came out of its wait: the loads from TMEM behind it are the whole warp's.
__device__ __forceinline__ bool all_got(bool got) { return __all_sync(0xffffffffu, got); }

// An arrival that publishes no memory: a TMEM buffer is handed back, whose loads are complete and ordered by the fence before. (With
// .release.cluster the second CTA's arrival waits 1200 to 1900 clocks for the thread's other accesses.)
__device__ __forceinline__ void arrive_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

}  // namespace f8
}  // namespace mb
