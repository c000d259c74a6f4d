// Wave operations for the CPU stand-in of the HIP runtime (hip_cpu_shim):
// force-included where csrc/step_embedding.hip is compiled for the CPU. Every
// lane of a workgroup is a thread there, so an operation across a wave is a
// barrier of its 64 threads, and a kernel may use one only where all lanes of a
// wave arrive (which the kernels compiled this way do).
#ifndef STEP_WAVE_SHIM_H_
#define STEP_WAVE_SHIM_H_

#include <hip/hip_runtime.h>

#include <atomic>
#include <condition_variable>
#include <mutex>

// fewer and shorter waves' worth of threads, the same code
#define STEP_SORT_THREADS 128
#define STEP_DIGIT_BITS 5

namespace step_wave_shim {
struct Wave {
  std::mutex mu;
  std::condition_variable cv;
  unsigned count = 0;
  uint64_t phase = 0;
  std::atomic<uint64_t> mask{0};
  uint32_t value[64];
  void barrier() {
    std::unique_lock<std::mutex> lock(mu);
    const uint64_t here = phase;
    if (++count == 64) {
      count = 0;
      phase++;
      cv.notify_all();
    } else {
      cv.wait(lock, [&] { return phase != here; });
    }
  }
};
inline Wave g_wave[16];
inline Wave& wave() { return g_wave[threadIdx.x / 64]; }
}  // namespace step_wave_shim

inline uint64_t __ballot(bool set) {
  auto& w = step_wave_shim::wave();
  const unsigned lane = threadIdx.x % 64;
  w.barrier();
  if (lane == 0) w.mask = 0;
  w.barrier();
  if (set) w.mask |= 1ull << lane;
  w.barrier();
  return w.mask;
}
inline uint32_t __shfl(uint32_t x, int from) {
  auto& w = step_wave_shim::wave();
  w.barrier();
  w.value[threadIdx.x % 64] = x;
  w.barrier();
  return w.value[from];
}
inline uint32_t __shfl_up(uint32_t x, int by) {
  auto& w = step_wave_shim::wave();
  const unsigned lane = threadIdx.x % 64;
  w.barrier();
  w.value[lane] = x;
  w.barrier();
  return lane < static_cast<unsigned>(by) ? x : w.value[lane - by];
}
inline void step_wave_fence() { step_wave_shim::wave().barrier(); }
inline int __popcll(uint64_t x) { return __builtin_popcountll(x); }
inline uint32_t atomicAdd(uint32_t* to, uint32_t x) { return __atomic_fetch_add(to, x, __ATOMIC_RELAXED); }

#endif  // STEP_WAVE_SHIM_H_
