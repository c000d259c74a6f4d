// Orthogonalised update by Newton-Schulz products for MI355X (gfx950):
// include/step_abi.h.
//
// Mathematics. With U an m x n update (m <= n; a tall one is taken transposed),
//   X_0 = U / (|U|_F + eps)
//   X_k+1 = (a I + b A + c A A) X_k,   A = X_k X_k^T
// every singular value of X runs through the same odd polynomial and is brought
// near 1 while the singular vectors stay. Three products per step: A and its
// square are symmetric, so only the tiles on and below the diagonal are computed
// (and stored twice): m^2 n + m^3 + 2 m^2 n multiplications and additions each
// instead of 2 m^2 n + 2 m^3 + 2 m^2 n.
//
// Numbers. The products run on the matrix cores with fp16 operands and float32
// sums. fp16 and not bfloat16: the iterates are bounded by about 1.2, so a fixed
// power of two (kScaleX, kScaleA, kScaleB) keeps them inside fp16's range, and its
// three more bits make every rounding eight times smaller. What is rounded off X
// is kept: X = hi + lo / 2048 in two fp16 planes, and the linear term a X counts
// both. Without that, rounding noise in the directions that U hardly has grows by
// a factor of a = 3.4 per step (485 in five), until it is 14 % of the result for
// an update of rank one, and with it 0.05 to 0.3 % whatever the rank (norm of the
// difference over that of the result; up to 0.6 % where an update has fewer than
// eight rows, whose few roundings hit everything).
//   SPLIT = false (bfloat16 results, 16-bit weights): products of the hi planes.
//   (The last iterate but one does without: its rounding grows by a once.)
//   SPLIT = true (other results): hi hi + (hi lo + lo hi) / 2048, three products,
//   22 bits of every operand: about 1e-6 off.
//
// Layout. Everything is padded to multiples of 64 with zeros, which the products
// keep. All three products contract over the contiguous index of both operands:
// X is kept by rows and, as Y = X^T, by columns, and A and B are symmetric.
#include "step_common.h"

#include <math.h>

#include <algorithm>

namespace step {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));

// Stored values are the real ones times these. |X| <= 1.2 and |A| <= 1.5 for updates that the iteration brings
// together; there is room for iterates up to 64, 4 and 64 times as large as 1.
constexpr float kScaleX = 1024.f;
constexpr float kScaleA = 16384.f;
constexpr float kScaleB = 1024.f;
constexpr float kScaleLow = 2048.f;  // hi + lo / 2048: the next 11 bits, away from fp16's smallest numbers

constexpr int kPad = 64;           // and the depth of one stage of a product
// (a build for the CPU takes shorter rounds)
#ifndef STEP_MOST_ITEMS
#define STEP_MOST_ITEMS 64
#define STEP_MOST_GROUPS 32
#define STEP_ROUND_ELEMENTS (1ull << 26)
#endif
constexpr int kMostItems = STEP_MOST_ITEMS;    // batches of matrices of one round, by value in the kernels' arguments
constexpr int kMostGroups = STEP_MOST_GROUPS;  // and shapes among them
constexpr int kMostPieces = 1024;  // partial sums of squares per matrix
constexpr uint64_t kPiece = 8192;  // elements of one, at least

constexpr size_t kMostSide = 1u << 20;
constexpr size_t kMostElements = 1ull << 33;
constexpr int kMostSteps = 64;

// ---- where a matrix keeps its planes -------------------------------------------

struct Planes {
  uint64_t norm, x_hi, x_lo, y_hi, y_lo, a_hi, a_lo, b_hi, b_lo, b_rest, bytes;
  uint64_t y_hi_step, y_lo_step;  // Y has two buffers that take turns; its low plane needs one only if no product reads it
};

__host__ __device__ inline uint32_t pieces_of(uint64_t size) {
  return static_cast<uint32_t>(size / kPiece + 1 < kMostPieces ? size / kPiece + 1 : kMostPieces);
}

__host__ __device__ inline Planes planes_of(uint64_t m, uint64_t n, bool split) {
  Planes p = {};
  uint64_t at = 0;
  const uint64_t mn = m * n * 2, mm = m * m * 2;
  p.norm = at; at += round_up(pieces_of(m * n) * 8, 256);
  p.x_hi = at; at += mn;
  p.y_hi = at; at += 2 * mn;
  p.y_hi_step = mn;
  p.y_lo = at; at += split ? 2 * mn : mn;
  p.y_lo_step = split ? mn : 0;
  p.a_hi = at; at += mm;
  p.b_hi = at; at += mm;
  if (split) {
    p.x_lo = at; at += mn;
    p.a_lo = at; at += mm;
    p.b_lo = at; at += mm;
  } else {
    p.b_rest = at; at += m * 2;  // what B's diagonal lost when it was rounded
  }
  p.bytes = round_up(at, 256);
  return p;
}

// Matrices of one shape, one behind the other in the workspace.
struct Group {
  uint64_t base;
  uint32_t m, n;          // padded
  uint32_t first_tile;    // of the launch
  uint32_t tiles;         // of one matrix
  uint32_t count, first_matrix;  // its matrices of the round
};
struct Groups {
  Group at[kMostGroups];
  int count;
};

// `count` contiguous updates of the caller.
struct Segment {
  const void* grad;
  float* momentum;
  uint64_t base;
  uint32_t rows, cols;
  uint32_t first_tile;
  uint32_t tiles;         // of one matrix
};
struct Segments {
  Segment at[kMostItems];
  int count;
};

// And where their results go.
struct Target {
  void* out;
  uint32_t rows, cols;
  uint32_t first_tile;    // its first matrix of the round
  float rate;             // what the orthogonalised update is multiplied by (Muon)
};
struct Targets {
  Target at[kMostItems];
  int count;
  int type, muon;
  float keep;
};
struct Nothing {};

// The last entry that begins at or before `tile`.
template <typename S> __device__ __forceinline__ int find(const S& s, uint32_t tile) {
  int lo = 0, hi = s.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (s.at[mid].first_tile <= tile) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ void split_value(float x, _Float16* hi, _Float16* lo) {
  *hi = static_cast<_Float16>(x);
  *lo = static_cast<_Float16>((x - static_cast<float>(*hi)) * kScaleLow);
}

// ---- the update, its norm, and the first iterate ---------------------------------

struct MomentumRule {
  float momentum;  // mu
  int nesterov, use;
};

// `count` (at most four) elements from `p` on, which is aligned to an element only.
template <typename T> struct Four;
template <> struct Four<F32> { typedef uint32_t type __attribute__((ext_vector_type(4))); };
template <> struct Four<BF16> { typedef uint16_t type __attribute__((ext_vector_type(4))); };
template <> struct Four<F16> { typedef uint16_t type __attribute__((ext_vector_type(4))); };
template <typename T> struct FourOf {
  typedef typename Four<T>::type V;
  typedef V VU __attribute__((aligned(sizeof(T))));
  struct Array { T at[4]; };
};
template <typename T> __device__ __forceinline__ float4v load4(const T* p, uint64_t count) {
  typename FourOf<T>::Array a = {};
  if (count >= 4) {
    a = __builtin_bit_cast(typename FourOf<T>::Array, static_cast<typename FourOf<T>::V>(*reinterpret_cast<const typename FourOf<T>::VU*>(p)));
  } else {
    for (int k = 0; k < 3; k++)
      if (static_cast<uint64_t>(k) < count) a.at[k] = p[k];
  }
  return float4v{to_float(a.at[0]), to_float(a.at[1]), to_float(a.at[2]), to_float(a.at[3])};
}
template <typename T> __device__ __forceinline__ void store4(T* p, float4v v, uint64_t count) {
  typename FourOf<T>::Array a;
  for (int k = 0; k < 4; k++) a.at[k] = from_float<T>(v[k]);
  if (count >= 4) {
    *reinterpret_cast<typename FourOf<T>::VU*>(p) = __builtin_bit_cast(typename FourOf<T>::V, a);
  } else {
    for (int k = 0; k < 3; k++)
      if (static_cast<uint64_t>(k) < count) p[k] = a.at[k];
  }
}

// Four elements of the update: the gradient, or what the momentum (this step's, written by the norm kernel) makes of it.
template <typename T>
__device__ __forceinline__ float4v update_at(const Segment& s, uint64_t at, uint64_t count, const MomentumRule& rule) {
  const float4v g = load4(static_cast<const T*>(s.grad) + at, count);
  if (!rule.use) return g;
  const float4v m = load4(reinterpret_cast<const F32*>(s.momentum) + at, count);
  return rule.nesterov ? g + rule.momentum * m : m;
}

// One workgroup per piece of a matrix: momentum = mu momentum + grad, and the piece's sum of squares of the update, in 64
// bits: gradients of 1e-20 have a norm too. Bound by HBM: 50 million bf16 gradients with their momentum 108 us, 0.5 GB at
// 4.7 TB/s.
template <typename T>
__global__ void __launch_bounds__(256) norm_kernel(Segments segments, MomentumRule rule, char* ws, int split) {
  __shared__ double sums[4];
  const Segment& s = segments.at[find(segments, blockIdx.x)];
  const uint32_t matrix = (blockIdx.x - s.first_tile) / s.tiles, piece = (blockIdx.x - s.first_tile) % s.tiles;
  const uint64_t size = static_cast<uint64_t>(s.rows) * s.cols, base = matrix * size;
  const uint64_t length = (size + s.tiles - 1) / s.tiles;
  const uint64_t begin = piece * length, end = begin + length < size ? begin + length : size;
  double sum = 0;
#pragma unroll 4
  for (uint64_t i = begin + threadIdx.x * 4; i < end; i += 1024) {
    float4v u = load4(static_cast<const T*>(s.grad) + base + i, end - i);
    if (rule.use) {
      const float4v m = rule.momentum * load4(reinterpret_cast<const F32*>(s.momentum) + base + i, end - i) + u;
      store4(reinterpret_cast<F32*>(s.momentum) + base + i, m, end - i);
      u = rule.nesterov ? u + rule.momentum * m : m;
    }
    for (int k = 0; k < 4; k++)
      if (i + k < end) sum += static_cast<double>(u[k]) * u[k];
  }
  for (int step = 32; step; step /= 2) sum += __shfl_xor(sum, step);
  if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    const bool tall = s.rows > s.cols;
    const Planes p = planes_of(round_up(tall ? s.cols : s.rows, kPad), round_up(tall ? s.rows : s.cols, kPad), split);
    reinterpret_cast<double*>(ws + s.base + matrix * p.bytes + p.norm)[piece] = sums[0] + sums[1] + sums[2] + sums[3];
  }
}

// One workgroup per 64 x 64 tile of U, through LDS: X_0 by rows and by columns. Bound by HBM: of those 50 million 0.6 GB in 136 us,
// 4.4 TB/s.
template <typename T, bool SPLIT>
__global__ void __launch_bounds__(256) first_kernel(Segments segments, MomentumRule rule, float eps, char* ws) {
  __shared__ float tile[64][65];
  __shared__ double sums[4];
  const Segment& s = segments.at[find(segments, blockIdx.x)];
  const uint32_t matrix = (blockIdx.x - s.first_tile) / s.tiles, t = (blockIdx.x - s.first_tile) % s.tiles;
  const bool tall = s.rows > s.cols;
  const uint32_t m = static_cast<uint32_t>(round_up(tall ? s.cols : s.rows, kPad));
  const uint32_t n = static_cast<uint32_t>(round_up(tall ? s.rows : s.cols, kPad));
  const Planes p = planes_of(m, n, SPLIT);
  char* at = ws + s.base + matrix * p.bytes;
  const uint64_t size = static_cast<uint64_t>(s.rows) * s.cols;
  const uint32_t across = (tall ? m : n) / 64, r0 = t / across * 64, c0 = t % across * 64;
  const uint32_t row = threadIdx.x / 16, col = threadIdx.x % 16 * 4;
  float4v u[4];
#pragma unroll
  for (int k = 0; k < 4; k++) {
    const uint32_t r = r0 + row + k * 16, c = c0 + col;
    u[k] = r < s.rows && c < s.cols ? update_at<T>(s, matrix * size + static_cast<uint64_t>(r) * s.cols + c, s.cols - c, rule) : float4v{0, 0, 0, 0};
  }
  const uint32_t pieces = pieces_of(size);
  double sum = 0;
  for (uint32_t k = threadIdx.x; k < pieces; k += 256) sum += reinterpret_cast<const double*>(at + p.norm)[k];
  for (int step = 32; step; step /= 2) sum += __shfl_xor(sum, step);
  if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = sum;
  __syncthreads();
  const double scale = kScaleX / (sqrt(sums[0] + sums[1] + sums[2] + sums[3]) + static_cast<double>(eps));
#pragma unroll
  for (int k = 0; k < 4; k++)
    for (int e = 0; e < 4; e++) tile[row + k * 16][col + e] = static_cast<float>(u[k][e] * scale);
  __syncthreads();
  // U's rows are X's rows if it is wide, Y's if it is tall
  _Float16* x_hi = reinterpret_cast<_Float16*>(at + p.x_hi);
  _Float16* x_lo = SPLIT ? reinterpret_cast<_Float16*>(at + p.x_lo) : nullptr;
  _Float16* y_hi = reinterpret_cast<_Float16*>(at + p.y_hi);
  _Float16* y_lo = reinterpret_cast<_Float16*>(at + p.y_lo);
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const uint32_t i = threadIdx.x / 8 + k * 32, j = threadIdx.x % 8 * 8;
    for (int by_col = 0; by_col < 2; by_col++) {
      half8 hi, lo;
      for (int e = 0; e < 8; e++) {
        _Float16 h, l;
        split_value(by_col ? tile[j + e][i] : tile[i][j + e], &h, &l);
        hi[e] = h;
        lo[e] = l;
      }
      const bool to_y = tall != (by_col != 0);
      const uint64_t to = static_cast<uint64_t>((by_col ? c0 : r0) + i) * (to_y ? m : n) + (by_col ? r0 : c0) + j;
      if (to_y) {
        *reinterpret_cast<half8*>(y_hi + to) = hi;
        *reinterpret_cast<half8*>(y_lo + to) = lo;
      } else {
        *reinterpret_cast<half8*>(x_hi + to) = hi;
        if (SPLIT) *reinterpret_cast<half8*>(x_lo + to) = lo;
      }
    }
  }
}

// ---- products -----------------------------------------------------------------------

// A = X X^T; B = a I + b A + c A A; the next X = B X and its Y; the last X, to the caller. The linear term is on B's
// diagonal, so that the products add it: no pass reads X for it, but the low plane where they do not. In fp16 that
// diagonal, 1024 * 3.4 and more, is off by up to 2^-12 of itself, which every later step stretches: where there is no low
// plane of B, what was rounded off its diagonal is kept apart (b_rest) and multiplied as a diagonal matrix, one more product
// of 16 x 16 x 32 for each of a wave's pieces. Without it, updates of rank one are 0.24 % off at any size (2-norm); with it
// 0.06 % at 128 rows and 0.02 % at 1000.
enum Kind { GRAM, SQUARE, APPLY, LAST };

// Moves 16 bytes per lane from global memory into LDS at base + 16 * lane, without registers in between.
__device__ __forceinline__ void load_to_lds(const void* from, void* base) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_global_load_lds(reinterpret_cast<const __attribute__((address_space(1))) uint32_t*>(reinterpret_cast<uintptr_t>(from)),
                                   reinterpret_cast<__attribute__((address_space(3))) uint32_t*>(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(base))),
                                   16, 0, 0);
#elif defined(STEP_MATRIX_SHIM_H_)
  step_matrix_shim::load_to_lds(from, base);
#endif
}

// Which row of a wave's part of a tile lane r of 16 reads for piece x. In pairs, so that the four rows of a result that a
// lane holds of piece 2 k and the four of piece 2 k + 1 are eight in a row: 16 bytes of what is stored by columns.
template <bool PAIRS> __device__ __forceinline__ uint32_t row_of_piece(uint32_t x, uint32_t r) {
  return PAIRS ? x / 2 * 32 + r / 4 * 8 + x % 2 * 4 + r % 4 : x * 16 + r;
}
// A row of a stage is 64 halves: 8 chunks of 16 bytes, whose order depends on the row so that the 16 lanes that read one
// chunk index of a piece's rows touch different banks (no conflicts measured).
template <bool PAIRS> __device__ __forceinline__ uint32_t chunk_place(uint32_t row, uint32_t chunk) {
  return chunk ^ (PAIRS ? (row >> 1 & 1) | (row >> 3 & 3) << 1 : row >> 1 & 7);
}

// Asks the compiler to mix the LDS reads and global loads of a half step among its products instead of putting them first.
template <int READS, int PRODUCTS, int LOADS> __device__ __forceinline__ void interleave() {
  constexpr int EACH = PRODUCTS / (READS + LOADS) > 0 ? PRODUCTS / (READS + LOADS) : 1;
#pragma unroll
  for (int k = 0; k < READS + LOADS; k++) {
    __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
    if (k % 2 == 0 && k / 2 < LOADS) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
    else __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
  }
}

template <int N> __device__ __forceinline__ void wait_loads() {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
#elif defined(STEP_MATRIX_SHIM_H_)
  step_matrix_shim::wait_loads(N);
#endif
}

// Four lanes side by side hold four rows of one column each; afterwards four columns of one row each.
__device__ __forceinline__ half4 transpose4(half4 v) {
  typedef uint32_t pair __attribute__((ext_vector_type(2)));
  pair r = __builtin_bit_cast(pair, v);
  const uint32_t lane = threadIdx.x;
  // with the lane next to it: 2 x 2 blocks
  const uint32_t o0 = __builtin_amdgcn_mov_dpp(r.x, 0xb1, 0xf, 0xf, true), o1 = __builtin_amdgcn_mov_dpp(r.y, 0xb1, 0xf, 0xf, true);
  // even: (mine[0], theirs[0]); odd: (theirs[1], mine[1])
  const uint32_t even0 = __builtin_amdgcn_perm(o0, r.x, 0x05040100), even1 = __builtin_amdgcn_perm(o1, r.y, 0x05040100);
  const uint32_t odd0 = __builtin_amdgcn_perm(r.x, o0, 0x07060302), odd1 = __builtin_amdgcn_perm(r.y, o1, 0x07060302);
  r.x = lane & 1 ? odd0 : even0;
  r.y = lane & 1 ? odd1 : even1;
  // with the lane two further on: the blocks off the diagonal change places
  const uint32_t p0 = __builtin_amdgcn_mov_dpp(r.x, 0x4e, 0xf, 0xf, true), p1 = __builtin_amdgcn_mov_dpp(r.y, 0x4e, 0xf, 0xf, true);
  pair out;
  out.x = lane & 2 ? p1 : r.x;
  out.y = lane & 2 ? r.y : p0;
  return __builtin_bit_cast(half4, out);
}

__device__ __forceinline__ float4v transpose4(float4v v) {
  const uint32_t lane = threadIdx.x;
  auto next = [](float x) { return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0xb1, 0xf, 0xf, true)); };
  auto after_next = [](float x) { return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x4e, 0xf, 0xf, true)); };
  const float s0 = next(lane & 1 ? v[0] : v[1]), s1 = next(lane & 1 ? v[2] : v[3]);
  if (lane & 1) { v[0] = s0; v[2] = s1; }
  else { v[1] = s0; v[3] = s1; }
  const float t0 = after_next(lane & 2 ? v[0] : v[2]), t1 = after_next(lane & 2 ? v[1] : v[3]);
  if (lane & 2) { v[0] = t0; v[1] = t1; }
  else { v[2] = t0; v[3] = t1; }
  return v;
}

// Tile t of the triangle of a square of `down` x `down` tiles, on and below the diagonal, in blocks of 4 x 4 tiles: what
// runs at the same time shares rows.
__device__ __forceinline__ void triangle_tile(uint32_t t, uint32_t down, uint32_t* ti, uint32_t* tj) {
  uint32_t block = static_cast<uint32_t>((sqrtf(8.f * t + 1.f) - 1.f) * 0.125f);
  while (block && 2 * block * (4 * block + 1) > t) block--;
  while (2 * (block + 1) * (4 * block + 5) <= t) block++;
  t -= 2 * block * (4 * block + 1);                      // 4 block (4 block + 1) / 2 tiles above
  const uint32_t high = down - 4 * block < 4 ? down - 4 * block : 4;
  const uint32_t across = t / (high * 4);
  if (across < block) {
    t -= across * high * 4;
    *ti = 4 * block + t % high;
    *tj = 4 * across + t / high;
  } else {
    t -= block * high * 4;
    uint32_t i = 0;
    while ((i + 1) * (i + 2) / 2 <= t) i++;
    *ti = 4 * block + i;
    *tj = 4 * block + t - i * (i + 1) / 2;
  }
}

// Tile t of down x across, in strips of eight rows of tiles.
__device__ __forceinline__ void square_tile(uint32_t t, uint32_t down, uint32_t across, uint32_t* ti, uint32_t* tj) {
  const uint32_t strip = t / (8 * across), high = down - 8 * strip < 8 ? down - 8 * strip : 8;
  t -= strip * 8 * across;
  *ti = strip * 8 + t % high;
  *tj = t / high;
}

// One product of a step for all matrices of a launch. A workgroup makes a SIDE x SIDE tile with KS groups of WM x WN waves,
// which take the stages of 64 halves of depth in turn and add their sums up in LDS at the end (tiles of 64: a matrix
// has few, and its depth is what takes the time). Stages go from global memory into LDS without registers, STAGES deep;
// the reads of a half step are mixed among the products of the half before.
// Reached: the Gram matrix of 4096 x 16384 260 us (1057 TFLOP/s of its triangle), B X of the same 531 to 561 us (980 to
// 1035); 8192^3 by the library 1254. Behind the main loop every result is split, transposed and stored
// twice (8 to 16 bytes per element), with one workgroup on a compute unit and nothing to hide it behind: that bounds B X
// where the contraction is short (m <= 1024, half of its time or more). Storing past the caches makes it slower (64-byte
// pieces of lines, which the L2 joins), as does a contraction cut among workgroups that add up behind the last.
template <int SIDE, int WM, int WN, int KS, int STAGES, Kind KIND, bool SPLIT>
__global__ void __launch_bounds__(KS * WM * WN * 64, 2)
    product_kernel(Groups groups, std::conditional_t<KIND == LAST, Targets, Nothing> targets, char* ws, int from, int low_in,
                   int low_out, float a, float b, float c) {
  constexpr bool FROM_Y = KIND == APPLY || KIND == LAST;
  constexpr int PLANES = SPLIT ? 2 : 1;
  constexpr int THREADS = WM * WN * 64;                     // of a group
  constexpr int FM = SIDE / WM / 16, FN = SIDE / WN / 16;   // 16 x 16 pieces of a wave
  constexpr int SUB = PLANES * 2 * SIDE * 64;               // halves of one group's stage: hi rows of both operands, lo rows
  constexpr int LOADS = PLANES * 2 * SIDE * 8 / THREADS;    // 16-byte chunks per lane and stage
  constexpr int PER_OPERAND = SIDE * 8 / THREADS;
  static_assert(SIDE * 8 % THREADS == 0, "a load belongs to one operand");
  static_assert(KS == 1 || (KS == 2 && FN % 2 == 0), "");
  constexpr int EN = FN / KS;                               // pieces across that a wave finishes
  constexpr bool PAIR_P = FM % 2 == 0, PAIR_Q = EN % 2 == 0;  // rows, columns of pieces are taken in pairs
  constexpr int DOWN = PAIR_P ? 2 : 1, ACROSS = PAIR_Q ? 2 : 1;
  constexpr int STAGED = STAGES * KS * SUB, SUMS = KS == 1 ? 0 : KS * SIDE * SIDE * 2;
  __shared__ _Float16 lds[STAGED > SUMS ? STAGED : SUMS];

  // Workgroups are dealt to the eight chiplets in turn: give each chiplet, and its cache, an eighth of every group's tiles
  // that are neighbours.
  const Group& g = groups.at[find(groups, blockIdx.x)];
  const uint32_t m = g.m, n = g.n, in_group = blockIdx.x - g.first_tile, of_group = g.tiles * g.count;
  const uint32_t share = of_group / 8, spare = of_group % 8, chiplet = in_group % 8;
  const uint32_t number = chiplet * share + (chiplet < spare ? chiplet : spare) + in_group / 8;
  const uint32_t matrix = number / g.tiles, tile = number % g.tiles;
  const Planes p = planes_of(m, n, SPLIT);
  char* at = ws + g.base + matrix * p.bytes;
  uint32_t ti, tj;
  if (FROM_Y) square_tile(tile, (m + SIDE - 1) / SIDE, (n + SIDE - 1) / SIDE, &ti, &tj);
  else triangle_tile(tile, (m + SIDE - 1) / SIDE, &ti, &tj);
  const uint32_t i0 = ti * SIDE, j0 = tj * SIDE, rows_q = FROM_Y ? n : m;
  const uint32_t depth = KIND == GRAM ? n : m, last = depth / 64;

  const uint32_t lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t mine = wave / (WM * WN), place = wave % (WM * WN);  // the wave's group, and its place there
  const uint32_t wi = place / WN * (SIDE / WM), wj = place % WN * (SIDE / WN);

  // What this lane loads: a chunk of each of PER_OPERAND rows of either operand, as bytes from the tile's first row (at
  // most 256 rows of 2^20 columns); rows behind the matrix repeat its last one.
  uint32_t offset[2 * PER_OPERAND];
#pragma unroll
  for (int k = 0; k < 2 * PER_OPERAND; k++) {
    const uint32_t chunk = k * THREADS + threadIdx.x % THREADS, row = chunk / 8;
    const bool second = k >= PER_OPERAND;
    const uint32_t r = second ? row - SIDE : row, end = second ? rows_q - j0 - 1 : m - i0 - 1;
    offset[k] = ((r < end ? r : end) * (depth / 8) + (second ? chunk_place<PAIR_Q>(r, chunk % 8) : chunk_place<PAIR_P>(r, chunk % 8))) * 16;
  }
  const uint64_t row_p = static_cast<uint64_t>(i0) * depth * 2, row_q = static_cast<uint64_t>(j0) * depth * 2;
  const uint64_t y_hi = p.y_hi + from * p.y_hi_step, y_lo = p.y_lo + from * p.y_lo_step;
  const char* operand[4] = {at + row_p + (KIND == GRAM ? p.x_hi : KIND == SQUARE ? p.a_hi : p.b_hi),
                            at + row_q + (KIND == GRAM ? p.x_hi : KIND == SQUARE ? p.a_hi : y_hi),
                            at + row_p + (KIND == GRAM ? p.x_lo : KIND == SQUARE ? p.a_lo : p.b_lo),
                            at + row_q + (KIND == GRAM ? p.x_lo : KIND == SQUARE ? p.a_lo : y_lo)};
  // the stages that begin at `step`, one for each group (behind the end: the last one again, which nobody multiplies)
  auto issue = [&](uint32_t step, uint32_t buffer) {
    step = KS == 1 || step + mine < last ? step + mine : last - 1;
    _Float16* to = lds + (buffer * KS + mine) * SUB + place * 64 * 8;
#pragma unroll
    for (int k = 0; k < LOADS; k++)
      load_to_lds(operand[k / PER_OPERAND] + step * 128ull + offset[k % (2 * PER_OPERAND)], to + k * THREADS * 8);
  };

  float4v acc[FM][FN] = {}, low[SPLIT ? FM : 1][SPLIT ? FN : 1] = {};
  // Fragments are read a half stage ahead of the products that use them, so that LDS and the matrix cores work at the
  // same time also where a SIMD has one wave.
  half8 fp[2][PLANES][FM], fq[2][PLANES][FN];
  auto read = [&](uint32_t buffer, int s) {
    const _Float16* stage = lds + (buffer * KS + mine) * SUB;
    const uint32_t chunk = s * 4 + lane / 16;
#pragma unroll
    for (int h = 0; h < PLANES; h++) {
#pragma unroll
      for (int x = 0; x < FM; x++) {
        const uint32_t row = wi + row_of_piece<PAIR_P>(x, lane % 16);
        fp[s][h][x] = *reinterpret_cast<const half8*>(stage + (h * 2 * SIDE + row) * 64 + chunk_place<PAIR_P>(row, chunk) * 8);
      }
#pragma unroll
      for (int y = 0; y < FN; y++) {
        const uint32_t row = wj + row_of_piece<PAIR_Q>(y, lane % 16);
        fq[s][h][y] = *reinterpret_cast<const half8*>(stage + (h * 2 * SIDE + SIDE + row) * 64 + chunk_place<PAIR_Q>(row, chunk) * 8);
      }
    }
  };
  auto multiply = [&](int s) {
#pragma unroll
    for (int x = 0; x < FM; x++)
#pragma unroll
      for (int y = 0; y < FN; y++) {
        acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp[s][0][x], fq[s][0][y], acc[x][y], 0, 0, 0);
        if constexpr (SPLIT) {
          low[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp[s][0][x], fq[s][1][y], low[x][y], 0, 0, 0);
          low[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp[s][1][x], fq[s][0][y], low[x][y], 0, 0, 0);
        }
      }
  };
  // What B's diagonal lost, as diagonal matrices of 32 rows (a pair of pieces), times those rows of X, from LDS while their
  // stage is there. (Muon of 24 matrices of width 1024: 1683 us without, 1713 so, 1760 with those rows fetched once more
  // behind the last stage.)
  constexpr bool REST = FROM_Y && !SPLIT;
  static_assert(!REST || PAIR_P, "");
  __shared__ uint16_t rest[REST ? SIDE : 1];
  uint32_t one_rest = 0;
  if (REST && threadIdx.x < SIDE) one_rest = reinterpret_cast<const uint16_t*>(at + p.b_rest)[i0 + threadIdx.x < m ? i0 + threadIdx.x : m - 1];
  auto add_rest = [&](uint32_t stage, uint32_t buffer) {
    if constexpr (REST) {
#pragma unroll
      for (int x = 0; x < FM; x++) {
        const uint32_t half = (i0 + wi) / 32 + x / 2;
        if (half / 2 != stage) continue;
        uint32_t lane = threadIdx.x % 64;
#if defined(__HIP_DEVICE_COMPILE__)
        asm volatile("" : "+v"(lane));  // the diagonals are made here: kept through the loop, they cost tiles of 256 their registers
#endif
        // the lane's row of the piece is on the diagonal in one of the eight places that the lane holds of it, or in none
        const uint32_t chunk = half % 2 * 4 + lane / 16, place = lane % 4;
        uint32_t on = rest[wi + row_of_piece<true>(x, lane % 16)];
        on = lane / 16 == lane % 16 / 4 ? place % 2 ? on << 16 : on : 0;
        typedef uint32_t raw4 __attribute__((ext_vector_type(4)));
        raw4 d = {0, 0, 0, 0};
        d[x % 2 * 2] = place < 2 ? on : 0;
        d[x % 2 * 2 + 1] = place < 2 ? 0 : on;
#pragma unroll
        for (int y = 0; y < FN; y++) {
          const uint32_t row = wj + row_of_piece<PAIR_Q>(y, lane % 16);
          const half8 q = *reinterpret_cast<const half8*>(lds + (buffer * KS + mine) * SUB + (SIDE + row) * 64 + chunk_place<PAIR_Q>(row, chunk) * 8);
          acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, d), q, acc[x][y], 0, 0, 0);
        }
      }
    }
  };
  constexpr int READS = PLANES * (FM + FN), PRODUCTS = FM * FN * (SPLIT ? 3 : 1);
#pragma unroll
  for (int k = 0; k < STAGES; k++)
    if (static_cast<uint32_t>(k * KS) < last) issue(k * KS, k);
  if (REST && threadIdx.x < SIDE) rest[threadIdx.x] = static_cast<uint16_t>(one_rest);
  // the first stage has landed when at most the later ones' loads are under way
  if ((STAGES - 1) * KS < last) wait_loads<(STAGES - 1) * LOADS>();
  else wait_loads<0>();
  read(0, 0);
  uint32_t step = 0, buffer = 0;
  auto after = [](uint32_t buffer) { return buffer + 1 == STAGES ? 0 : buffer + 1; };
  for (; step + STAGES * KS < last; step += KS, buffer = after(buffer)) {
    add_rest(step + mine, buffer);
    read(buffer, 1);
    multiply(0);
    interleave<READS, PRODUCTS, 0>();
    // behind the barrier the next stage has landed, and every wave has read all of this one, which the loads overwrite
    wait_loads<(STAGES - 2) * LOADS>();
    issue(step + STAGES * KS, buffer);
    read(after(buffer), 0);
    multiply(1);
    interleave<READS, PRODUCTS, LOADS>();
  }
  for (; step < last; step += KS, buffer = after(buffer)) {
    const bool busy = KS == 1 || step + mine < last;
    if (busy) add_rest(step + mine, buffer);
    read(buffer, 1);
    if (busy) multiply(0);
    wait_loads<0>();
    if (step + KS < last) read(after(buffer), 0);
    if (busy) multiply(1);
  }
  if constexpr (SPLIT) {
#pragma unroll
    for (int x = 0; x < FM; x++)
#pragma unroll
      for (int y = 0; y < FN; y++) acc[x][y] += low[x][y] * (1.f / kScaleLow);
  }
  // the groups' sums, in their order; each goes on with its share of the pieces of a place in the tile
  const uint32_t ey = mine * EN;
  float4v sum[FM][EN];
  if constexpr (KS == 1) {
#pragma unroll
    for (int x = 0; x < FM; x++)
#pragma unroll
      for (int y = 0; y < EN; y++) sum[x][y] = acc[x][y];
  } else {
    constexpr int GROUP = WM * WN * FM * FN * 64;
    float4v* sums = reinterpret_cast<float4v*>(lds) + place * (FM * FN * 64) + lane;
    wait_loads<0>();
#pragma unroll
    for (int x = 0; x < FM; x++)
#pragma unroll
      for (int y = 0; y < FN; y++) sums[mine * GROUP + (x * FN + y) * 64] = acc[x][y];
    __syncthreads();
#pragma unroll
    for (int x = 0; x < FM; x++)
#pragma unroll
      for (int y = 0; y < EN; y++) {
        sum[x][y] = sums[(x * FN + y + ey) * 64];
#pragma unroll
        for (int k = 1; k < KS; k++) sum[x][y] += sums[k * GROUP + (x * FN + y + ey) * 64];
      }
  }

  // A lane holds rows 4 (lane / 16) + 0..3 and column lane % 16 of every 16 x 16 piece: of a pair of them 16 bytes of what
  // is stored by columns. Exchanged among four lanes it is 16 bytes of what is stored by rows. Addresses: the wave's
  // corner, the same for all its lanes, then 32 bits for a lane's place in it.
  const uint64_t old_hi_at = p.a_hi, old_lo_at = FROM_Y ? y_lo : p.a_lo;
  const uint64_t col_hi_at = KIND == APPLY ? p.y_hi + (from ^ 1) * p.y_hi_step : KIND == GRAM ? p.a_hi : p.b_hi;
  const uint64_t col_lo_at = KIND == APPLY ? p.y_lo + (from ^ 1) * p.y_lo_step : KIND == GRAM ? p.a_lo : p.b_lo;
  const uint64_t row_hi_at = KIND == APPLY ? p.x_hi : col_hi_at, row_lo_at = KIND == APPLY ? p.x_lo : col_lo_at;
  const uint32_t row_length = FROM_Y ? n : m;
  const uint64_t corner_i = i0 + wi, corner_j = j0 + wj + ey * 16;
  const uint64_t col_corner = (corner_j * m + corner_i) * 2, row_corner = (corner_i * row_length + corner_j) * 2;
  // a lane's first row and column by columns; its row and first column by rows
  const uint32_t col_i = lane / 16 * (4 * DOWN), col_j = row_of_piece<PAIR_Q>(0, lane % 16);
  const uint32_t row_i = lane / 16 * (4 * DOWN) + lane % 4, row_j = lane % 16 / 4 * (4 * ACROSS);
  const uint32_t col_lane = (col_j * m + col_i) * 2, row_lane = (row_i * row_length + row_j) * 2;
  // What the result is made from is fetched some rows of pieces ahead of its use: the stores may not pass the loads.
  constexpr int SETS = FM / DOWN, AHEAD = SETS < 3 ? SETS : 3;
  const bool with_hi = KIND == SQUARE, with_low = KIND == SQUARE ? SPLIT : !SPLIT && FROM_Y && low_in;
  typedef std::conditional_t<PAIR_P, half8, half4> Down;
  typedef std::conditional_t<PAIR_Q, half8, half4> Across;
  Down old_hi[AHEAD][EN], old_lo[AHEAD][EN];
  auto fetch = [&](int set) {
    if (KIND == GRAM || corner_i + set * 16 * DOWN >= m) return;
#pragma unroll
    for (int y = 0; y < EN; y++) {
      if (corner_j + y / ACROSS * 16 * ACROSS >= rows_q) break;
      const char* from_col = at + col_corner + (static_cast<uint64_t>(y / ACROSS * 16 * ACROSS + y % ACROSS * 4) * m + set * 16 * DOWN) * 2;
      if (with_hi) old_hi[set % AHEAD][y] = *reinterpret_cast<const Down*>(from_col + old_hi_at + col_lane);
      if (with_low) old_lo[set % AHEAD][y] = *reinterpret_cast<const Down*>(from_col + old_lo_at + col_lane);
    }
  };
  Target t = {};
  bool tall = false, muon = false;
  float keep = 0.f;
  if constexpr (KIND == LAST) {
    const uint32_t of_round = g.first_matrix + matrix;
    t = targets.at[find(targets, of_round)];
    const uint64_t skip = static_cast<uint64_t>(of_round - t.first_tile) * t.rows * t.cols;
    t.out = static_cast<char*>(t.out) + skip * (targets.type == STEP_F32 ? 4 : 2);
    tall = t.rows > t.cols;
    muon = targets.muon;
    keep = targets.keep;
  }
  auto finish = [&](auto type) {
    typedef decltype(type) T;
#pragma unroll
    for (int set = 0; set < AHEAD - 1; set++) fetch(set);
#pragma unroll
    for (int set = 0; set < SETS; set++) {
      if (set + AHEAD - 1 < SETS) fetch(set + AHEAD - 1);
      if (corner_i + set * 16 * DOWN >= m) break;
#pragma unroll
      for (int y0 = 0; y0 < EN; y0 += ACROSS) {
        if (corner_j + y0 * 16 >= rows_q) break;
        Across row_hi[DOWN], row_lo[DOWN];
#pragma unroll
        for (int dy = 0; dy < ACROSS; dy++) {
          const int y = y0 + dy;
          Down hi, lo;
#pragma unroll
          for (int dx = 0; dx < DOWN; dx++) {
            float4v v = sum[set * DOWN + dx][y];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              if (KIND == GRAM) {
                v[e] *= kScaleA / (kScaleX * kScaleX);
              } else if (KIND == SQUARE) {
                float old = static_cast<float>(old_hi[set % AHEAD][y][dx * 4 + e]);
                if (with_low) old += static_cast<float>(old_lo[set % AHEAD][y][dx * 4 + e]) * (1.f / kScaleLow);
                v[e] = b * (kScaleB / kScaleA) * old + c * (kScaleB / kScaleA / kScaleA) * v[e];
                if (corner_i + set * 16 * DOWN + col_i + dx * 4 + e == corner_j + y0 * 16 + dy * 4 + col_j) v[e] += a * kScaleB;
              } else {
                v[e] *= 1.f / kScaleB;
                if (with_low) v[e] += a * (1.f / kScaleLow) * static_cast<float>(old_lo[set % AHEAD][y][dx * 4 + e]);
              }
            }
            if (KIND == SQUARE && !SPLIT && ti == tj) {
              const uint32_t i = wi + set * 16 * DOWN + col_i + dx * 4, j = wj + ey * 16 + y0 * 16 + dy * 4 + col_j, e = j - i;
              if (e < 4) {
                const float on = e == 0 ? v[0] : e == 1 ? v[1] : e == 2 ? v[2] : v[3];
                reinterpret_cast<_Float16*>(at + p.b_rest)[j0 + j] = static_cast<_Float16>(on - static_cast<float>(static_cast<_Float16>(on)));
              }
            }
            if constexpr (KIND == LAST) {
              v = v * (1.f / kScaleX);
              if (!tall) v = transpose4(v);
              const uint64_t i = corner_i + set * 16 * DOWN + dx * 4 + (tall ? col_i : row_i);
              const uint64_t j = corner_j + y0 * 16 + dy * 4 + (tall ? col_j : row_j);
              const uint64_t r = tall ? j : i, col = tall ? i : j;
              if (r < t.rows && col < t.cols) {
                T* to = static_cast<T*>(t.out) + r * t.cols + col;
                if (muon) v = keep * load4(to, t.cols - col) - t.rate * v;
                store4(to, v, t.cols - col);
              }
            } else {
              half4 h, l;
#pragma unroll
              for (int e = 0; e < 4; e++) {
                _Float16 one, rest;
                split_value(v[e], &one, &rest);
                h[e] = hi[dx * 4 + e] = one;
                l[e] = lo[dx * 4 + e] = rest;
              }
              const half4 th = transpose4(h);
#pragma unroll
              for (int e = 0; e < 4; e++) row_hi[dx][dy * 4 + e] = th[e];
              if (SPLIT) {
                const half4 tl = transpose4(l);
#pragma unroll
                for (int e = 0; e < 4; e++) row_lo[dx][dy * 4 + e] = tl[e];
              }
            }
          }
          if constexpr (KIND != LAST) {
            if (KIND == APPLY || ti != tj) {               // Y; the mirror image of a tile off the diagonal
              char* to_col = at + col_corner + (static_cast<uint64_t>(y0 * 16 + dy * 4) * m + set * 16 * DOWN) * 2;
              *reinterpret_cast<Down*>(to_col + col_hi_at + col_lane) = hi;
              if (SPLIT ? true : KIND == APPLY && low_out) *reinterpret_cast<Down*>(to_col + col_lo_at + col_lane) = lo;
            }
          }
        }
        if constexpr (KIND != LAST) {
#pragma unroll
          for (int dx = 0; dx < DOWN; dx++) {
            char* to_row = at + row_corner + (static_cast<uint64_t>(set * 16 * DOWN + dx * 4) * row_length + y0 * 16) * 2;
            *reinterpret_cast<Across*>(to_row + row_hi_at + row_lane) = row_hi[dx];
            if (SPLIT) *reinterpret_cast<Across*>(to_row + row_lo_at + row_lane) = row_lo[dx];
          }
        }
      }
    }
  };
  if constexpr (KIND == LAST) {
    if (targets.type == STEP_F32) finish(F32());
    else if (targets.type == STEP_BF16) finish(BF16());
    else finish(F16());
  } else {
    finish(F32());
  }
}

// ---- small matrices -----------------------------------------------------------------

// Matrices of at most 64 x 256 (or the transposed) are a workgroup each, from the momentum to the result in one launch:
// both forms of X, A and B stay in LDS, every operand split. What bounds them is the chain of barriers and LDS reads of a
// step (about 4 us), where the launches of the products above take 15: 48 of 64 x 128 21 us, by the products 78.
constexpr uint32_t kSmallRows = 64, kSmallCols = 256, kSmallThreads = 512;

struct SmallItem {
  const void* grad;
  float* momentum;
  void* out;
  uint32_t first_tile;  // its first matrix of the launch
  uint16_t rows, cols;
  float rate;
};
struct SmallItems {
  SmallItem at[kMostItems];
  int count;
  int out_type, muon, steps;
  float keep, eps;
};
struct Coefficients {
  float at[3 * kMostSteps];
};

// Halves of a row of `length` (a multiple of 64) in LDS, its chunks of 16 bytes ordered by the row.
__device__ __forceinline__ uint32_t small_place(uint32_t row, uint32_t col, uint32_t length) {
  const uint32_t chunk = col / 8 ^ (length == 64 ? row >> 1 & 7 : row & 7);
  return row * length + chunk * 8 + col % 8;
}

template <typename T, int N>
__global__ void __launch_bounds__(kSmallThreads) small_kernel(SmallItems items, Coefficients coefficients, MomentumRule rule) {
  __shared__ _Float16 x_hi[64 * N], x_lo[64 * N], y_hi[64 * N], y_lo[64 * N], s_hi[64 * 64], s_lo[64 * 64];
  __shared__ double sums[kSmallThreads / 64];
  const SmallItem& item = items.at[find(items, blockIdx.x)];
  const uint32_t rows = item.rows, cols = item.cols;
  const bool tall = rows > cols;
  const uint64_t base = static_cast<uint64_t>(blockIdx.x - item.first_tile) * rows * cols;
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const uint32_t strip = wave % 4 * 16, half = wave / 4 * 2;  // a wave's rows of A and B, and the first of its two pieces there

  // the update, four elements of a row at a time, padded with zeros
  constexpr int MOST = 64 * N / 4 / kSmallThreads;
  const uint32_t per_row = (tall ? 64 : N) / 4;
  float4v u[MOST];
  double sum = 0;
#pragma unroll
  for (int k = 0; k < MOST; k++) {
    const uint32_t v = k * kSmallThreads + threadIdx.x, r = v / per_row, c = v % per_row * 4;
    u[k] = float4v{0, 0, 0, 0};
    if (r >= rows || c >= cols) continue;
    const uint64_t at = base + r * cols + c;
    u[k] = load4(static_cast<const T*>(item.grad) + at, cols - c);
    if (rule.use) {
      F32* momentum = reinterpret_cast<F32*>(item.momentum) + at;
      const float4v m = rule.momentum * load4(momentum, cols - c) + u[k];
      store4(momentum, m, cols - c);
      u[k] = rule.nesterov ? u[k] + rule.momentum * m : m;
    }
    for (int e = 0; e < 4; e++) {
      if (c + e >= cols) u[k][e] = 0.f;
      sum += static_cast<double>(u[k][e]) * u[k][e];
    }
  }
  for (int step = 32; step; step /= 2) sum += __shfl_xor(sum, step);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  sum = 0;
  for (int k = 0; k < static_cast<int>(kSmallThreads) / 64; k++) sum += sums[k];
  const double scale = kScaleX / (sqrt(sum) + static_cast<double>(items.eps));
#pragma unroll
  for (int k = 0; k < MOST; k++) {
    const uint32_t v = k * kSmallThreads + threadIdx.x, r = v / per_row, c = v % per_row * 4;
    for (int e = 0; e < 4; e++) {
      _Float16 hi, lo;
      split_value(static_cast<float>(u[k][e] * scale), &hi, &lo);
      const uint32_t i = tall ? c + e : r, j = tall ? r : c + e;
      x_hi[small_place(i, j, N)] = hi;
      x_lo[small_place(i, j, N)] = lo;
      y_hi[small_place(j, i, 64)] = hi;
      y_lo[small_place(j, i, 64)] = lo;
    }
  }

  auto fragment = [&](const _Float16* from, uint32_t row, uint32_t k, uint32_t length) {
    return *reinterpret_cast<const half8*>(from + small_place(row, k * 32 + lane / 16 * 8, length));
  };
  auto product = [](float4v& acc, float4v& low, half8 ph, half8 pl, half8 qh, half8 ql) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, qh, acc, 0, 0, 0);
    low = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, ql, low, 0, 0, 0);
    low = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, qh, low, 0, 0, 0);
  };
  // pieces of A and B, stored transposed, which they equal
  auto put_square = [&](const float4v (&v)[2]) {
#pragma unroll
    for (int y = 0; y < 2; y++) {
      half4 hi, lo;
      for (int e = 0; e < 4; e++) {
        _Float16 h, l;
        split_value(v[y][e], &h, &l);
        hi[e] = h;
        lo[e] = l;
      }
      const uint32_t to = small_place((half + y) * 16 + lane % 16, strip + lane / 16 * 4, 64);
      *reinterpret_cast<half4*>(s_hi + to) = hi;
      *reinterpret_cast<half4*>(s_lo + to) = lo;
    }
  };
  constexpr int WAVES = kSmallThreads / 64, PN = N / 16 / WAVES;  // pieces across of a wave's columns of X
  float4v next[4][PN];
  for (int step = 0;; step++) {
    const float a = coefficients.at[3 * step], b = coefficients.at[3 * step + 1], c = coefficients.at[3 * step + 2];
    __syncthreads();
    float4v acc[2] = {}, low[2] = {}, gram[2];
#pragma unroll 2
    for (uint32_t k = 0; k < N / 32; k++) {
      const half8 ph = fragment(x_hi, strip + lane % 16, k, N), pl = fragment(x_lo, strip + lane % 16, k, N);
#pragma unroll
      for (int y = 0; y < 2; y++)
        product(acc[y], low[y], ph, pl, fragment(x_hi, (half + y) * 16 + lane % 16, k, N), fragment(x_lo, (half + y) * 16 + lane % 16, k, N));
    }
#pragma unroll
    for (int y = 0; y < 2; y++) gram[y] = (acc[y] + low[y] * (1.f / kScaleLow)) * (kScaleA / (kScaleX * kScaleX));
    put_square(gram);
    __syncthreads();
#pragma unroll
    for (int y = 0; y < 2; y++) acc[y] = low[y] = float4v{0, 0, 0, 0};
#pragma unroll
    for (uint32_t k = 0; k < 2; k++) {
      const half8 ph = fragment(s_hi, strip + lane % 16, k, 64), pl = fragment(s_lo, strip + lane % 16, k, 64);
#pragma unroll
      for (int y = 0; y < 2; y++)
        product(acc[y], low[y], ph, pl, fragment(s_hi, (half + y) * 16 + lane % 16, k, 64), fragment(s_lo, (half + y) * 16 + lane % 16, k, 64));
    }
#pragma unroll
    for (int y = 0; y < 2; y++) {
      gram[y] = b * (kScaleB / kScaleA) * gram[y] + c * (kScaleB / kScaleA / kScaleA) * (acc[y] + low[y] * (1.f / kScaleLow));
      for (int e = 0; e < 4; e++)
        if (strip + lane / 16 * 4 + e == (half + y) * 16 + lane % 16) gram[y][e] += a * kScaleB;
    }
    __syncthreads();  // every wave has read A
    put_square(gram);
    __syncthreads();
    float4v next_low[4][PN];
#pragma unroll
    for (int x = 0; x < 4; x++)
#pragma unroll
      for (int y = 0; y < PN; y++) next[x][y] = next_low[x][y] = float4v{0, 0, 0, 0};
#pragma unroll
    for (uint32_t k = 0; k < 2; k++) {
      half8 qh[PN], ql[PN];
#pragma unroll
      for (int y = 0; y < PN; y++) {
        qh[y] = fragment(y_hi, wave * (N / WAVES) + y * 16 + lane % 16, k, 64);
        ql[y] = fragment(y_lo, wave * (N / WAVES) + y * 16 + lane % 16, k, 64);
      }
#pragma unroll
      for (int x = 0; x < 4; x++) {
        const half8 ph = fragment(s_hi, x * 16 + lane % 16, k, 64), pl = fragment(s_lo, x * 16 + lane % 16, k, 64);
#pragma unroll
        for (int y = 0; y < PN; y++) product(next[x][y], next_low[x][y], ph, pl, qh[y], ql[y]);
      }
    }
#pragma unroll
    for (int x = 0; x < 4; x++)
#pragma unroll
      for (int y = 0; y < PN; y++) next[x][y] = (next[x][y] + next_low[x][y] * (1.f / kScaleLow)) * (1.f / kScaleB);
    if (step + 1 == items.steps) break;
    // a wave reads and writes rows of Y of its own; X was last read two barriers ago
#pragma unroll
    for (int x = 0; x < 4; x++)
#pragma unroll
      for (int y = 0; y < PN; y++) {
        half4 hi, lo;
        for (int e = 0; e < 4; e++) {
          _Float16 h, l;
          split_value(next[x][y][e], &h, &l);
          hi[e] = h;
          lo[e] = l;
        }
        const uint32_t j = wave * (N / WAVES) + y * 16;
        const uint32_t by_col = small_place(j + lane % 16, x * 16 + lane / 16 * 4, 64);
        const uint32_t by_row = small_place(x * 16 + lane / 16 * 4 + lane % 4, j + lane % 16 / 4 * 4, N);
        *reinterpret_cast<half4*>(y_hi + by_col) = hi;
        *reinterpret_cast<half4*>(y_lo + by_col) = lo;
        *reinterpret_cast<half4*>(x_hi + by_row) = transpose4(hi);
        *reinterpret_cast<half4*>(x_lo + by_row) = transpose4(lo);
      }
  }
  auto finish = [&](auto type) {
    typedef decltype(type) O;
#pragma unroll
    for (int x = 0; x < 4; x++)
#pragma unroll
      for (int y = 0; y < PN; y++) {
        float4v v = next[x][y] * (1.f / kScaleX);
        if (!tall) v = transpose4(v);
        const uint32_t i = x * 16 + lane / 16 * 4 + (tall ? 0 : lane % 4);
        const uint32_t j = wave * (N / WAVES) + y * 16 + (tall ? lane % 16 : lane % 16 / 4 * 4);
        const uint32_t r = tall ? j : i, col = tall ? i : j;
        if (r >= rows || col >= cols) continue;
        O* to = static_cast<O*>(item.out) + base + r * cols + col;
        if (items.muon) v = items.keep * load4(to, cols - col) - item.rate * v;
        store4(to, v, cols - col);
      }
  };
  if (items.out_type == STEP_F32) finish(F32());
  else if (items.out_type == STEP_BF16) finish(BF16());
  else finish(F16());
}

// ---- host side -----------------------------------------------------------------------

// Elements of one round, beyond which more matrices fill the GPU no better and only ask for more workspace.
constexpr uint64_t kRoundElements = STEP_ROUND_ELEMENTS;

bool is_small(const step_matrix& x) { return std::min(x.rows, x.cols) <= kSmallRows && std::max(x.rows, x.cols) <= kSmallCols; }

// Whether small matrices go with the larger ones of their list: with split products, as exact as on their own, they ride
// along in launches that are made anyway (of the ResNet-50 set's 54 matrices 8 are small, and on their own they would take
// 98 us beside the 1370 of the whole step). Products of single operands are for the larger ones only, or what a small
// matrix gets would depend on its neighbours.
bool rides_along(const step_matrix* list, size_t length, int precise) {
  for (size_t k = 0; k < length && precise; k++)
    if (!is_small(list[k])) return true;
  return false;
}

struct Item {
  size_t matrix, first, count;  // matrices [first, first + count) of the caller's batch `matrix`
  uint32_t m, n;
};

// Cuts the caller's list (its small matrices only if asked to) into rounds, their items in the order of their padded
// shapes; visit(items, their number) for each.
template <typename Visit>
int for_rounds(const step_matrix* list, size_t length, bool with_small, const Visit& visit) {
  Item items[kMostItems];
  int used = 0, shapes = 0;
  uint64_t elements = 0;
  auto flush = [&]() {
    if (!used) return static_cast<int>(STEP_OK);
    std::stable_sort(items, items + used, [](const Item& x, const Item& y) { return x.m != y.m ? x.m > y.m : x.n > y.n; });
    const int rc = visit(static_cast<const Item*>(items), used);
    used = shapes = 0;
    elements = 0;
    return rc;
  };
  for (size_t k = 0; k < length; k++) {
    const size_t rows = list[k].rows, cols = list[k].cols;
    if (rows == 0 || cols == 0 || (!with_small && is_small(list[k]))) continue;
    const uint32_t m = static_cast<uint32_t>(round_up(std::min(rows, cols), kPad));
    const uint32_t n = static_cast<uint32_t>(round_up(std::max(rows, cols), kPad));
    const uint64_t one = static_cast<uint64_t>(m) * n;
    size_t first = 0;
    while (first < list[k].count) {
      bool known = false;
      for (int j = 0; j < used && !known; j++) known = items[j].m == m && items[j].n == n;
      const uint64_t room = elements < kRoundElements ? (kRoundElements - elements) / one : 0;
      if (used == kMostItems || (!known && shapes == kMostGroups) || (room == 0 && used)) {
        const int rc = flush();
        if (rc != STEP_OK) return rc;
        continue;
      }
      const size_t take = static_cast<size_t>(std::min<uint64_t>(list[k].count - first, std::max<uint64_t>(room, 1)));
      items[used++] = {k, first, take, m, n};
      shapes += known ? 0 : 1;
      elements += take * one;
      first += take;
    }
  }
  return flush();
}

// The workspace of one round: its matrices, one behind the other.
struct Layout {
  Groups groups;
  uint64_t base[kMostItems];
  uint64_t bytes;
};

Layout layout_for(const Item* items, int count, bool split) {
  Layout l;
  l.groups.count = 0;
  l.bytes = 0;
  uint32_t number = 0;
  for (int k = 0; k < count; k++) {
    const Item& item = items[k];
    l.base[k] = l.bytes;
    const int g = l.groups.count - 1;
    if (g >= 0 && l.groups.at[g].m == item.m && l.groups.at[g].n == item.n) {
      l.groups.at[g].count += static_cast<uint32_t>(item.count);
    } else {
      l.groups.at[l.groups.count++] = {l.bytes, item.m, item.n, 0, 0, static_cast<uint32_t>(item.count), number};
    }
    number += static_cast<uint32_t>(item.count);
    l.bytes += planes_of(item.m, item.n, split).bytes * item.count;
  }
  return l;
}

int check_list(const step_matrix* list, size_t length, int dtype, int out_dtype, bool muon) {
  if (length && !list) return STEP_ERR_ARGUMENT;
  if (!is_float(dtype) || !is_float(out_dtype)) return STEP_ERR_DTYPE;
  for (size_t k = 0; k < length; k++) {
    const step_matrix& x = list[k];
    if (x.rows > kMostSide || x.cols > kMostSide || x.count > kMostSize) return STEP_ERR_LIMIT;
    if (x.rows * x.cols > kMostElements) return STEP_ERR_LIMIT;
    if (x.rows && x.cols && x.count && (!x.grad || !x.out || (muon && !x.momentum))) return STEP_ERR_ARGUMENT;
  }
  return STEP_OK;
}

template <typename Go> void by_type(int dtype, const Go& go) {
  if (dtype == STEP_F32) go(F32());
  else if (dtype == STEP_BF16) go(BF16());
  else go(F16());
}

// What a workgroup of a tile size takes: microseconds per stage of its depth and for what comes behind, where
// `per_cu` workgroups share a compute unit.
struct Cost {
  double stage, end;
  uint32_t per_cu;
};
constexpr uint32_t kUnits = 256;  // compute units
// Iterates of more elements (8 bytes of each are moved behind a product) do not stay in the 256 MB cache in front of HBM.
constexpr uint64_t kNearElements = 1ull << 25;

// The tiles of side `side` of a product of every group, the deepest first, and about how long the launch takes.
template <Kind KIND> double cut(Groups& groups, uint32_t side, const Cost& cost, uint32_t* tiles) {
  double work = 0, longest = 0;
  *tiles = 0;
  std::stable_sort(groups.at, groups.at + groups.count, [](const Group& x, const Group& y) { return KIND == GRAM ? x.n > y.n : x.m > y.m; });
  for (int k = 0; k < groups.count; k++) {
    Group& g = groups.at[k];
    const uint32_t down = (g.m + side - 1) / side, across = (g.n + side - 1) / side;
    g.tiles = KIND == APPLY || KIND == LAST ? down * across : down * (down + 1) / 2;
    g.first_tile = *tiles;
    *tiles += g.tiles * g.count;
    const double one = (KIND == GRAM ? g.n : g.m) / 64 * cost.stage + cost.end;
    work += one * g.tiles * g.count;
    longest = std::max(longest, one);
  }
  const uint32_t at_once = kUnits * cost.per_cu;
  if (groups.count > 1) return std::max(longest / cost.per_cu, work / at_once);  // unlike tiles fill each other's gaps
  // alike ones go round by round; a workgroup that has a unit to itself is faster
  const uint32_t left = *tiles % at_once;
  return longest * (*tiles / at_once + (left == 0 ? 0 : left <= kUnits ? 1.0 / cost.per_cu : 1.0));
}

template <int SIDE, int WM, int WN, int KS, int STAGES, Kind KIND, bool SPLIT, typename Extra>
void launch_product(const Groups& groups, uint32_t tiles, const Extra& targets, char* ws, int from, int low_in, int low_out,
                    const float* coefficients, hipStream_t stream) {
  hipLaunchKernelGGL((product_kernel<SIDE, WM, WN, KS, STAGES, KIND, SPLIT>), dim3(tiles), dim3(KS * WM * WN * 64), 0, stream,
                     groups, targets, ws, from, low_in, low_out, coefficients[0], coefficients[1], coefficients[2]);
}

// The tile size by what the launch would take with each. Large tiles read less per product but leave compute units idle
// where there are few; the costs are those measured for one 1024 x 4096, 16 of 1024 x 1024, 4096 x 4096, 4096 x 16384 and
// 8192 x 8192. The Gram matrix of 4096 x 16384 has 136 tiles of 256 (326 us), 253 of 192 (256 us) or 528 of 128 (355 us), that of
// 1024 x 2752 has 36 of 128 (33 us) or 136 of 64 (17 us).
template <Kind KIND, bool SPLIT> uint32_t side_for(Groups groups) {
  constexpr bool SQUARES = KIND == APPLY || KIND == LAST;
  uint32_t tiles;
#if defined(STEP_MATRIX_SHIM_H_)
  if (step_matrix_shim::g_side) return SPLIT ? std::min(step_matrix_shim::g_side, 128u) : SQUARES && step_matrix_shim::g_side == 192 ? 256 : step_matrix_shim::g_side;
#endif
  if (SPLIT) {
    const double large = cut<KIND>(groups, 128, Cost{1.17, KIND == LAST ? 8. : KIND == APPLY ? 12. : 6., 1}, &tiles);
    const double small = cut<KIND>(groups, 64, Cost{0.48, KIND == APPLY ? 4. : 2.4, 1}, &tiles);
    return large < small ? 128 : 64;
  }
  uint64_t elements = 0;
  for (int k = 0; k < groups.count; k++) elements += static_cast<uint64_t>(groups.at[k].m) * groups.at[k].n * groups.at[k].count;
  const bool far = elements > kNearElements;
  const double t256 = cut<KIND>(groups, 256, Cost{SQUARES ? 1.5 : 1.3, KIND == LAST ? (far ? 26. : 22.) : KIND == APPLY ? (far ? 35. : 28.) : 10., 1}, &tiles);
  const double t192 = SQUARES ? 1e30 : cut<KIND>(groups, 192, Cost{0.98, 5., 1}, &tiles);
  const double t128 = cut<KIND>(groups, 128, Cost{0.98, KIND == LAST ? (far ? 14. : 8.) : KIND == APPLY ? (far ? 20. : 10.) : 4., 2}, &tiles);
  const double t64 = cut<KIND>(groups, 64, Cost{0.17, 3.5, 1}, &tiles);
  if (t64 <= std::min(std::min(t256, t192), t128)) return 64;
  if (t128 <= std::min(t256, t192)) return 128;
  return t256 <= t192 ? 256 : 192;
}

template <Kind KIND, bool SPLIT, typename Extra>
void product(const Layout& l, const Extra& targets, char* ws, int from, int low_in, int low_out, const float* coefficients,
             hipStream_t stream) {
  Groups groups = l.groups;
  const uint32_t side = side_for<KIND, SPLIT>(groups);
  uint32_t tiles;
  cut<KIND>(groups, side, Cost{0, 0, 1}, &tiles);
#define STEP_PRODUCT(...) launch_product<__VA_ARGS__, KIND, SPLIT>(groups, tiles, targets, ws, from, low_in, low_out, coefficients, stream)
  if constexpr (SPLIT) {
    if (side == 128) STEP_PRODUCT(128, 2, 4, 1, 2);
    else STEP_PRODUCT(64, 2, 2, 2, 2);
  } else {
    if (side == 64) STEP_PRODUCT(64, 2, 2, 2, 4);
    else if (side == 128) STEP_PRODUCT(128, 2, 2, 1, 2);
    else if (side == 256) STEP_PRODUCT(256, 2, 4, 1, 2);
    else if constexpr (KIND == GRAM || KIND == SQUARE) STEP_PRODUCT(192, 2, 4, 1, 3);
  }
#undef STEP_PRODUCT
}

struct Rule {
  MomentumRule momentum;
  float eps, keep;
  int muon, steps;
  const float* coefficients;
};

template <bool SPLIT>
int run_round(const step_matrix* list, const Item* items, int count, int dtype, int out_dtype, const Rule& rule, char* ws,
              hipStream_t stream) {
  const Layout l = layout_for(items, count, SPLIT);
  Segments by_piece, by_tile;
  Targets targets;
  by_piece.count = by_tile.count = targets.count = count;
  targets.type = out_dtype;
  targets.muon = rule.muon;
  targets.keep = rule.keep;
  uint32_t pieces = 0, tiles = 0, number = 0;
  for (int k = 0; k < count; k++) {
    const Item& item = items[k];
    const step_matrix& x = list[item.matrix];
    const uint64_t size = static_cast<uint64_t>(x.rows) * x.cols, skip = item.first * size;
    const uint32_t rows = static_cast<uint32_t>(x.rows), cols = static_cast<uint32_t>(x.cols), many = static_cast<uint32_t>(item.count);
    const char* grad = static_cast<const char*>(x.grad) + skip * dtype_size(dtype);
    float* momentum = rule.momentum.use ? x.momentum + skip : nullptr;
    const uint32_t of_pieces = pieces_of(size), of_tiles = static_cast<uint32_t>(static_cast<uint64_t>(item.m / 64) * (item.n / 64));
    by_piece.at[k] = {grad, momentum, l.base[k], rows, cols, pieces, of_pieces};
    by_tile.at[k] = {grad, momentum, l.base[k], rows, cols, tiles, of_tiles};
    targets.at[k] = {static_cast<char*>(x.out) + skip * dtype_size(out_dtype), rows, cols, number, x.rate};
    pieces += of_pieces * many;
    tiles += of_tiles * many;
    number += many;
  }
  by_type(dtype, [&](auto type) {
    typedef decltype(type) T;
    hipLaunchKernelGGL((norm_kernel<T>), dim3(pieces), dim3(256), 0, stream, by_piece, rule.momentum, ws, SPLIT ? 1 : 0);
    hipLaunchKernelGGL((first_kernel<T, SPLIT>), dim3(tiles), dim3(256), 0, stream, by_tile, rule.momentum, rule.eps, ws);
  });
  for (int step = 0; step < rule.steps; step++) {
    const float* c = rule.coefficients + 3 * step;
    const int from = step % 2, left = rule.steps - 1 - step;
    product<GRAM, SPLIT>(l, Nothing(), ws, from, 0, 0, c, stream);
    product<SQUARE, SPLIT>(l, Nothing(), ws, from, 0, 0, c, stream);
    // the low plane of the last iterate but one is left out (the only one of a single step is there already)
    if (left) product<APPLY, SPLIT>(l, Nothing(), ws, from, 1, left > 1, c, stream);
    else product<LAST, SPLIT>(l, targets, ws, from, step == 0, 0, c, stream);
  }
  return launched();
}

constexpr uint32_t kMostGrid = 1u << 22;  // workgroups of a launch, whose lanes have to stay below 2^32

// A list's small matrices, those of up to 64 x 128 apart: two workgroups of them fit a compute unit's LDS.
int run_small(const step_matrix* list, size_t length, int dtype, int out_dtype, const Rule& rule, hipStream_t stream) {
  bool any = false;
  Coefficients coefficients;
  memcpy(coefficients.at, rule.coefficients, sizeof(float) * 3 * rule.steps);
  for (const uint32_t across : {128u, 256u}) {
    SmallItems items;
    items.out_type = out_dtype;
    items.muon = rule.muon;
    items.steps = rule.steps;
    items.keep = rule.keep;
    items.eps = rule.eps;
    items.count = 0;
    uint32_t matrices = 0;
    auto flush = [&]() {
      if (!items.count) return;
      by_type(dtype, [&](auto type) {
        typedef decltype(type) T;
        if (across == 128) hipLaunchKernelGGL((small_kernel<T, 128>), dim3(matrices), dim3(kSmallThreads), 0, stream, items, coefficients, rule.momentum);
        else hipLaunchKernelGGL((small_kernel<T, 256>), dim3(matrices), dim3(kSmallThreads), 0, stream, items, coefficients, rule.momentum);
      });
      any = true;
      items.count = 0;
      matrices = 0;
    };
    for (size_t k = 0; k < length; k++) {
      const step_matrix& x = list[k];
      if (!is_small(x) || x.rows == 0 || x.cols == 0 || x.count == 0 || (std::max(x.rows, x.cols) <= 128) != (across == 128)) continue;
      for (size_t first = 0, take; first < x.count; first += take) {
        if (items.count == kMostItems || matrices == kMostGrid) flush();
        take = std::min<size_t>(x.count - first, kMostGrid - matrices);
        const size_t skip = first * x.rows * x.cols;
        items.at[items.count++] = {static_cast<const char*>(x.grad) + skip * dtype_size(dtype), x.momentum ? x.momentum + skip : nullptr,
                                   static_cast<char*>(x.out) + skip * dtype_size(out_dtype), matrices,
                                   static_cast<uint16_t>(x.rows), static_cast<uint16_t>(x.cols), x.rate};
        matrices += static_cast<uint32_t>(take);
      }
    }
    flush();
  }
  return any ? launched() : static_cast<int>(STEP_OK);
}

int run(const step_matrix* list, size_t length, int dtype, int out_dtype, int precise, const Rule& rule, void* workspace,
        size_t workspace_bytes, hipStream_t stream) {
  if (rule.steps < 1 || rule.steps > kMostSteps || !rule.coefficients) return STEP_ERR_ARGUMENT;
  const size_t need = step_orthogonalize_workspace(list, length, precise);
  if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256)) return STEP_ERR_ARGUMENT;
  const bool with_small = rides_along(list, length, precise);
  if (!with_small) {
    const int rc = run_small(list, length, dtype, out_dtype, rule, stream);
    if (rc != STEP_OK) return rc;
  }
  char* ws = static_cast<char*>(workspace);
  return for_rounds(list, length, with_small, [&](const Item* items, int count) {
    return precise ? run_round<true>(list, items, count, dtype, out_dtype, rule, ws, stream)
                   : run_round<false>(list, items, count, dtype, out_dtype, rule, ws, stream);
  });
}

}  // namespace
}  // namespace step

using namespace step;

extern "C" {

size_t step_orthogonalize_workspace(const step_matrix* list, size_t length, int precise) {
  uint64_t most = 0;
  if (length && !list) return 0;
  for_rounds(list, length, rides_along(list, length, precise), [&](const Item* items, int count) {
    most = std::max(most, layout_for(items, count, precise != 0).bytes);
    return static_cast<int>(STEP_OK);
  });
  return most;
}

int step_orthogonalize_side(const step_matrix* list, size_t length, int precise, int product) {
  int side = 0;
  if (length && !list) return 0;
  for_rounds(list, length, rides_along(list, length, precise), [&](const Item* items, int count) {
    const Groups groups = layout_for(items, count, precise != 0).groups;
    auto of = [&](auto split) {
      constexpr bool SPLIT = decltype(split)::value;
      return product == GRAM ? side_for<GRAM, SPLIT>(groups) : product == SQUARE ? side_for<SQUARE, SPLIT>(groups)
           : product == APPLY ? side_for<APPLY, SPLIT>(groups) : product == LAST ? side_for<LAST, SPLIT>(groups) : 0;
    };
    if (side == 0) side = static_cast<int>(precise ? of(std::true_type()) : of(std::false_type()));
    return static_cast<int>(STEP_OK);
  });
  return side;
}

int step_orthogonalize(const step_matrix* list, size_t length, int dtype, int out_dtype, int precise, int steps,
                       const float* coefficients, float eps, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_list(list, length, dtype, out_dtype, false);
  if (rc != STEP_OK) return rc;
  const Rule rule = {{0.f, 0, 0}, eps, 0.f, 0, steps, coefficients};
  return run(list, length, dtype, out_dtype, precise, rule, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

int step_muon(const step_matrix* list, size_t length, int dtype, int precise, int steps, const float* coefficients,
              float eps, float momentum, int nesterov, float keep, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_list(list, length, dtype, dtype, true);
  if (rc != STEP_OK) return rc;
  const Rule rule = {{momentum, nesterov, 1}, eps, keep, 1, steps, coefficients};
  return run(list, length, dtype, dtype, precise, rule, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

}  // extern "C"
