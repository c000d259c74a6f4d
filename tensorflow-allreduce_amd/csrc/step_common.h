// Shared by the sources of libstep_hip.so: status handling, element types and
// the wave operations the kernels use.
#ifndef STEP_COMMON_H_
#define STEP_COMMON_H_

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>
#include <string.h>

#include <type_traits>

#include "step_abi.h"

namespace step {

int hip_fail(hipError_t e);  // records the error for step_last_hip_error, returns STEP_ERR_HIP

// The status of the launches made so far by this thread.
inline int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? STEP_OK : hip_fail(e);
}

constexpr size_t kMostSize = 0x7fffffff;  // tokens, rows, columns: positions and keys are 32-bit

inline bool is_float(int dtype) { return dtype == STEP_F32 || dtype == STEP_BF16 || dtype == STEP_F16; }
inline size_t dtype_size(int dtype) { return dtype == STEP_F32 || dtype == STEP_I32 ? 4 : dtype == STEP_I64 ? 8 : 2; }
__host__ __device__ inline size_t round_up(size_t x, size_t to) { return (x + to - 1) / to * to; }

// ---- element types -------------------------------------------------------------
// The storage types of the three value types, and their conversions: to 32 bits
// exactly, back with one rounding to nearest even.
struct F32 { float v; };
struct BF16 { uint16_t v; };
struct F16 { uint16_t v; };

__device__ __forceinline__ float to_float(F32 x) { return x.v; }
__device__ __forceinline__ float to_float(BF16 x) { return __builtin_bit_cast(float, static_cast<uint32_t>(x.v) << 16); }
__device__ __forceinline__ float to_float(F16 x) { return static_cast<float>(__builtin_bit_cast(_Float16, x.v)); }

template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ F32 from_float<F32>(float x) { return {x}; }
template <> __device__ __forceinline__ BF16 from_float<BF16>(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
  return {__builtin_bit_cast(uint16_t, static_cast<__bf16>(x))};
#else
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  if ((u & 0x7fffffffu) > 0x7f800000u) return {static_cast<uint16_t>((u >> 16) | 0x40)};
  return {static_cast<uint16_t>((u + 0x7fff + ((u >> 16) & 1)) >> 16)};
#endif
}
template <> __device__ __forceinline__ F16 from_float<F16>(float x) {
  return {__builtin_bit_cast(uint16_t, static_cast<_Float16>(x))};
}

// A lane's 16 bytes of a row.
template <typename T> struct Vec {
  static constexpr int kCount = 16 / static_cast<int>(sizeof(T));
  T at[kCount];
};

}  // namespace step

#endif  // STEP_COMMON_H_
