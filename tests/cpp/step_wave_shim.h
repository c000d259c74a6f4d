// Wave operations for the CPU stand-in of the HIP runtime (hip_cpu_shim):
// force-included where csrc/step_embedding.hip is compiled for the CPU. Every
// lane of a workgroup is a thread there, so an operation across a wave is a
// barrier of the workgroup, and a kernel may use one only where all its lanes
// arrive (which the kernels compiled this way do).
#ifndef STEP_WAVE_SHIM_H_
#define STEP_WAVE_SHIM_H_

#include <hip/hip_runtime.h>

#include <atomic>

// fewer and shorter waves' worth of threads, the same code
#define STEP_SORT_THREADS 128
#define STEP_DIGIT_BITS 5

namespace step_wave_shim {
inline std::atomic<uint64_t> g_mask[16];
inline uint32_t g_value[1024];
}  // namespace step_wave_shim

inline uint64_t __ballot(bool set) {
  const unsigned wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  __syncthreads();
  if (lane == 0) step_wave_shim::g_mask[wave] = 0;
  __syncthreads();
  if (set) step_wave_shim::g_mask[wave] |= 1ull << lane;
  __syncthreads();
  return step_wave_shim::g_mask[wave];
}
inline uint32_t __shfl(uint32_t x, int from) {
  __syncthreads();
  step_wave_shim::g_value[threadIdx.x] = x;
  __syncthreads();
  return step_wave_shim::g_value[threadIdx.x / 64 * 64 + from];
}
inline uint32_t __shfl_up(uint32_t x, int by) {
  const unsigned lane = threadIdx.x % 64;
  __syncthreads();
  step_wave_shim::g_value[threadIdx.x] = x;
  __syncthreads();
  return lane < static_cast<unsigned>(by) ? x : step_wave_shim::g_value[threadIdx.x - by];
}
inline int __popcll(uint64_t x) { return __builtin_popcountll(x); }
inline uint32_t atomicAdd(uint32_t* to, uint32_t x) { return __atomic_fetch_add(to, x, __ATOMIC_RELAXED); }

#endif  // STEP_WAVE_SHIM_H_
