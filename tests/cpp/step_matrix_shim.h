// Matrix-core and LDS operations for the CPU stand-in of the HIP runtime
// (hip_cpu_shim): force-included, behind step_wave_shim.h, where
// csrc/step_orthogonalize.hip is compiled for the CPU.
//
// A load from global memory into LDS that a kernel does not wait for lands as
// late as the kernel's own waits allow: it is put off until a wait leaves fewer
// loads under way, so a wait that is counted too high reads what was there
// before, and one that misses its barrier is a race.
#ifndef STEP_MATRIX_SHIM_H_
#define STEP_MATRIX_SHIM_H_

#include "step_wave_shim.h"

#include <deque>

// shorter rounds of a list, the same code
#define STEP_MOST_ITEMS 3
#define STEP_MOST_GROUPS 2
#define STEP_ROUND_ELEMENTS 60000

namespace step_matrix_shim {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));

// tiles of this side for every product, whatever they would cost (0: by cost)
inline unsigned g_side = 0;

struct Load {
  const void* from;
  void* to;
};
inline thread_local std::deque<Load> t_loads;

inline void load_to_lds(const void* from, void* base) {
  t_loads.push_back({from, static_cast<char*>(base) + threadIdx.x % 64 * 16});
}
inline void wait_loads(unsigned left) {
  while (t_loads.size() > left) {
    memcpy(t_loads.front().to, t_loads.front().from, 16);
    t_loads.pop_front();
  }
  __syncthreads();
}

// What each lane of a wave hands to the others: two buffers that take turns, so that one barrier an operation is enough (no
// lane is two operations ahead of another).
template <typename T> struct Exchange {
  T value[2][64];
};
template <typename T> inline Exchange<T> g_exchange[16];
template <typename T> inline thread_local unsigned t_turn = 0;
template <typename T> inline const T* exchange(const T& mine) {
  T* values = g_exchange<T>[threadIdx.x / 64].value[t_turn<T>++ % 2];
  values[threadIdx.x % 64] = mine;
  step_wave_shim::wave().barrier();
  return values;
}

struct Operands {
  half8 a, b;
};
// C + A B of 16 x 16 x 32: lane l holds row (column) l % 16 of A (B), the eight k from l / 16 * 8 on, and column l % 16, the
// four rows from l / 16 * 4 on, of C.
inline float4v mfma_16x16x32(half8 a, half8 b, float4v c) {
  const Operands* all = exchange(Operands{a, b});
  const unsigned lane = threadIdx.x % 64;
  for (unsigned e = 0; e < 4; e++)
    for (unsigned k = 0; k < 32; k++)
      c[e] += static_cast<float>(all[k / 8 * 16 + lane / 16 * 4 + e].a[k % 8]) * static_cast<float>(all[k / 8 * 16 + lane % 16].b[k % 8]);
  return c;
}

// Only what the kernels use: quads whose neighbours (0xb1) or halves (0x4e) change places.
inline int quad_perm(int x, int control) { return exchange(x)[threadIdx.x % 64 ^ (control == 0xb1 ? 1 : 2)]; }

// Byte k of the result is byte selector[k] of b (0 to 3) or a (4 to 7).
inline unsigned byte_perm(unsigned a, unsigned b, unsigned selector) {
  const uint64_t both = static_cast<uint64_t>(a) << 32 | b;
  unsigned r = 0;
  for (unsigned k = 0; k < 4; k++) r |= static_cast<unsigned>(both >> (selector >> 8 * k & 7) * 8 & 0xff) << 8 * k;
  return r;
}

}  // namespace step_matrix_shim

inline double __shfl_xor(double x, int by) { return step_matrix_shim::exchange(x)[threadIdx.x % 64 ^ static_cast<unsigned>(by)]; }

#define __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, cbsz, abid, blgp) step_matrix_shim::mfma_16x16x32(a, b, c)
#define __builtin_amdgcn_mov_dpp(x, control, rows, banks, bound) step_matrix_shim::quad_perm(static_cast<int>(x), control)
#define __builtin_amdgcn_perm(a, b, selector) step_matrix_shim::byte_perm(a, b, selector)
#define __builtin_amdgcn_readfirstlane(x) (x)  // of what all lanes of a wave have
#define __builtin_amdgcn_sched_group_barrier(kind, count, group) do {} while (0)

#endif  // STEP_MATRIX_SHIM_H_
