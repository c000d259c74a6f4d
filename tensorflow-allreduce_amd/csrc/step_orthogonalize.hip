// Orthogonalised update by Newton-Schulz products for MI355X (gfx950):
// include/step_abi.h.
//
// Mathematics. With U an m x n update (m <= n; a tall one is taken transposed),
//   X_0 = U / (|U|_F + eps)
//   X_k+1 = a X_k + (b A + c A A) X_k,   A = X_k X_k^T
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
// is kept: X = hi + lo / 2048 in two fp16 planes, and the linear term a X uses
// both. Without that, rounding noise in the directions that U hardly has grows by
// a factor of a = 3.4 per step (485 in five), until it is 14 % of the result for
// an update of rank one, and with it 0.03 to 0.2 % whatever the rank.
//   SPLIT = false (16-bit results): products of the hi planes.
//   SPLIT = true (float32 results): hi hi + (hi lo + lo hi) / 2048, three products,
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

constexpr int kPad = 64;             // and the depth of one stage of a product
constexpr int kMostSegments = 48;    // of one launch, by value in the kernel's arguments
constexpr int kNormBlocks = 256;     // partial sums of squares per matrix

constexpr size_t kMostSide = 1u << 20;
constexpr size_t kMostElements = 1ull << 33;
constexpr int kMostSteps = 64;

// ---- where a matrix keeps its planes -------------------------------------------

struct Planes {
  uint64_t x_hi, x_lo, y_hi, y_lo, a_hi, a_lo, b_hi, b_lo, norm, bytes;
  uint64_t y_hi_step, y_lo_step;  // Y has two buffers that take turns; its low plane needs one only if no product reads it
};

__host__ __device__ inline Planes planes_of(uint64_t m, uint64_t n, bool split) {
  Planes p = {};
  uint64_t at = 0;
  const uint64_t mn = m * n * 2, mm = m * m * 2;
  p.norm = at; at += kNormBlocks * 8;
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
  }
  p.bytes = (at + 255) / 256 * 256;
  return p;
}

// `count` matrices of one shape, one behind the other in the workspace.
struct Group {
  uint64_t base;
  uint32_t m, n;        // padded
  uint32_t first_tile;  // of the launch
  uint32_t tiles;       // of one matrix
};
struct Groups {
  Group at[kMostSegments];
  int count;
};

// `count` contiguous matrices of the caller.
struct Segment {
  const void* grad;
  float* momentum;
  void* out;
  uint64_t base;
  uint32_t rows, cols;
  uint32_t first_tile;
  uint32_t tiles;       // of one matrix
  float rate;           // what the orthogonalised update is multiplied by (Muon)
  int tall;
};
struct Segments {
  Segment at[kMostSegments];
  int count;
};

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

template <typename T>
__device__ __forceinline__ float update_at(const Segment& s, uint64_t at, const MomentumRule& rule) {
  const float g = to_float(static_cast<const T*>(s.grad)[at]);
  if (!rule.use) return g;
  const float m = s.momentum[at];  // this step's, written by the norm kernel
  return rule.nesterov ? g + rule.momentum * m : m;
}

// One block per piece of a matrix: momentum = mu momentum + grad, and the piece's sum of squares of the update. In 64
// bits: gradients of 1e-20 have a norm too.
template <typename T>
__global__ void __launch_bounds__(256) norm_kernel(Segments segments, MomentumRule rule, char* ws, int split) {
  __shared__ double sums[4];
  const Segment& s = segments.at[find(segments, blockIdx.x)];
  const uint32_t matrix = (blockIdx.x - s.first_tile) / s.tiles, piece = (blockIdx.x - s.first_tile) % s.tiles;
  const uint64_t size = static_cast<uint64_t>(s.rows) * s.cols, base = matrix * size;
  const uint64_t length = (size + s.tiles - 1) / s.tiles;
  const uint64_t end = (piece + 1) * length < size ? (piece + 1) * length : size;
  double sum = 0;
  for (uint64_t i = piece * length + threadIdx.x; i < end; i += 256) {
    if (rule.use) {
      const float g = to_float(static_cast<const T*>(s.grad)[base + i]);
      s.momentum[base + i] = rule.momentum * s.momentum[base + i] + g;
    }
    const double u = update_at<T>(s, base + i, rule);
    sum += u * u;
  }
  for (int step = 32; step; step /= 2) sum += __shfl_xor(sum, step);
  if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint64_t m = round_up(s.tall ? s.cols : s.rows, kPad), n = round_up(s.tall ? s.rows : s.cols, kPad);
    const Planes p = planes_of(m, n, split);
    reinterpret_cast<double*>(ws + s.base + matrix * p.bytes + p.norm)[piece] = sums[0] + sums[1] + sums[2] + sums[3];
  }
}

// One block per 64 x 64 tile of U: X_0 by rows and by columns.
template <typename T, bool SPLIT>
__global__ void __launch_bounds__(256) first_kernel(Segments segments, MomentumRule rule, float eps, char* ws) {
  __shared__ float tile[64][65];
  __shared__ double sums[4];
  const Segment& s = segments.at[find(segments, blockIdx.x)];
  const uint32_t matrix = (blockIdx.x - s.first_tile) / s.tiles, t = (blockIdx.x - s.first_tile) % s.tiles;
  const uint32_t m = static_cast<uint32_t>(round_up(s.tall ? s.cols : s.rows, kPad));
  const uint32_t n = static_cast<uint32_t>(round_up(s.tall ? s.rows : s.cols, kPad));
  const Planes p = planes_of(m, n, SPLIT);
  char* at = ws + s.base + matrix * p.bytes;
  const uint64_t size = static_cast<uint64_t>(s.rows) * s.cols;
  const uint32_t pieces = static_cast<uint32_t>(size / 4096 + 1 < kNormBlocks ? size / 4096 + 1 : kNormBlocks);
  double sum = threadIdx.x < pieces ? reinterpret_cast<const double*>(at + p.norm)[threadIdx.x] : 0;
  for (int step = 32; step; step /= 2) sum += __shfl_xor(sum, step);
  if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = sum;
  __syncthreads();
  const double scale = kScaleX / (sqrt(sums[0] + sums[1] + sums[2] + sums[3]) + static_cast<double>(eps));
  // the tile of U
  const uint32_t across = static_cast<uint32_t>(round_up(s.cols, 64)) / 64;
  const uint32_t r0 = t / across * 64, c0 = t % across * 64;
  for (uint32_t k = threadIdx.x; k < 64 * 64; k += 256) {
    const uint32_t r = r0 + k / 64, c = c0 + k % 64;
    float u = 0.f;
    if (r < s.rows && c < s.cols) u = static_cast<float>(update_at<T>(s, matrix * size + static_cast<uint64_t>(r) * s.cols + c, rule) * scale);
    tile[k / 64][k % 64] = u;
  }
  __syncthreads();
  // by_rows: the planes whose rows are U's rows; X if U is wide, Y if it is tall
  _Float16* x_hi = reinterpret_cast<_Float16*>(at + p.x_hi);
  _Float16* x_lo = SPLIT ? reinterpret_cast<_Float16*>(at + p.x_lo) : nullptr;
  _Float16* y_hi = reinterpret_cast<_Float16*>(at + p.y_hi);
  _Float16* y_lo = reinterpret_cast<_Float16*>(at + p.y_lo);
  for (uint32_t k = threadIdx.x; k < 64 * 64; k += 256) {
    const uint32_t i = k / 64, j = k % 64;
    _Float16 hi, lo;
    split_value(tile[i][j], &hi, &lo);
    const uint64_t by_row = static_cast<uint64_t>(r0 + i) * (s.tall ? m : n) + c0 + j;
    if (s.tall) { y_hi[by_row] = hi; y_lo[by_row] = lo; }
    else { x_hi[by_row] = hi; if (SPLIT) x_lo[by_row] = lo; }
    split_value(tile[j][i], &hi, &lo);
    const uint64_t by_col = static_cast<uint64_t>(c0 + i) * (s.tall ? n : m) + r0 + j;
    if (s.tall) { x_hi[by_col] = hi; if (SPLIT) x_lo[by_col] = lo; }
    else { y_hi[by_col] = hi; y_lo[by_col] = lo; }
  }
}

// ---- products -----------------------------------------------------------------------

enum Kind { GRAM, SQUARE, APPLY };

// Moves 16 bytes per lane from global memory into LDS at base + 16 * lane, without registers in between.
__device__ __forceinline__ void load_to_lds(const void* from, void* base) {
  __builtin_amdgcn_global_load_lds(reinterpret_cast<const __attribute__((address_space(1))) uint32_t*>(reinterpret_cast<uintptr_t>(from)),
                                   reinterpret_cast<__attribute__((address_space(3))) uint32_t*>(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(base))),
                                   16, 0, 0);
}

// A row of a stage is 64 halves: 8 chunks of 16 bytes, whose order depends on the row so that the 16 lanes that read one
// chunk index of 16 rows touch different banks.
__device__ __forceinline__ uint32_t chunk_place(uint32_t row, uint32_t chunk) { return chunk ^ ((row >> 1) & 7); }

template <int TM, int TN, int WM, int WN, Kind KIND, bool SPLIT>
__global__ void __launch_bounds__(WM * WN * 64) product_kernel(Groups groups, char* ws, int from, float a, float b, float c) {
  constexpr int THREADS = WM * WN * 64;
  constexpr int FM = TM / WM / 16, FN = TN / WN / 16;
  constexpr int LOADS = (TM + TN) * 8 / THREADS;     // 16-byte chunks per lane and stage
  constexpr int STAGE = (TM + TN) * 64;              // halves
  __shared__ _Float16 lds[2 * STAGE];

  const Group& g = groups.at[find(groups, blockIdx.x)];
  const uint32_t m = g.m, n = g.n;
  const uint32_t matrix = (blockIdx.x - g.first_tile) / g.tiles, tile = (blockIdx.x - g.first_tile) % g.tiles;
  const Planes p = planes_of(m, n, SPLIT);
  char* at = ws + g.base + matrix * p.bytes;

  uint32_t ti, tj;
  if (KIND == APPLY) {
    const uint32_t down = (m + TM - 1) / TM;
    ti = tile % down;
    tj = tile / down;
  } else {                                           // tile i (i + 1) / 2 + j, j <= i
    ti = static_cast<uint32_t>((sqrtf(8.f * tile + 1.f) - 1.f) * 0.5f);
    while (ti * (ti + 1) / 2 > tile) ti--;
    while ((ti + 1) * (ti + 2) / 2 <= tile) ti++;
    tj = tile - ti * (ti + 1) / 2;
  }
  const uint32_t i0 = ti * TM, j0 = tj * TN;
  const uint32_t depth = KIND == GRAM ? n : m;       // both operands' row length
  const uint32_t rows_p = m, rows_q = KIND == APPLY ? n : m;
  const uint64_t y_hi_at = p.y_hi + from * p.y_hi_step, y_lo_at = p.y_lo + from * p.y_lo_step;
  const uint64_t y_hi_to = p.y_hi + (from ^ 1) * p.y_hi_step, y_lo_to = p.y_lo + (from ^ 1) * p.y_lo_step;
  const char* p_hi = at + (KIND == GRAM ? p.x_hi : KIND == SQUARE ? p.a_hi : p.b_hi);
  const char* p_lo = at + (KIND == GRAM ? p.x_lo : KIND == SQUARE ? p.a_lo : p.b_lo);
  const char* q_hi = KIND == APPLY ? at + y_hi_at : p_hi;
  const char* q_lo = KIND == APPLY ? at + y_lo_at : p_lo;

  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  // what this lane loads: one chunk of each of LOADS rows; rows behind the matrix repeat its last one
  uint32_t offset[LOADS];
  for (int k = 0; k < LOADS; k++) {
    const uint32_t chunk = k * THREADS + threadIdx.x, row = chunk / 8;
    const bool second = row >= TM;
    uint32_t r = second ? j0 + row - TM : i0 + row;
    const uint32_t last = (second ? rows_q : rows_p) - 1;
    r = r < last ? r : last;
    offset[k] = chunk_place(row, chunk % 8) * 16;
    // rows times their length may pass 32 bits: kept in units of 16 bytes
    offset[k] = r * (depth / 8) + offset[k] / 16;
  }
  const uint32_t steps = depth / 64;
  const uint32_t total = SPLIT ? 3 * steps : steps;
  auto issue = [&](uint32_t step) {
    const uint32_t part = SPLIT ? step / steps : 2, k0 = SPLIT ? step % steps : step;
    const char* from_p = part == 1 ? p_lo : p_hi;    // hi lo, lo hi, hi hi
    const char* from_q = part == 0 ? q_lo : q_hi;
    _Float16* to = lds + (step & 1) * STAGE + wave * 64 * 8;
    for (int k = 0; k < LOADS; k++) {
      const bool second = k * THREADS / 8 >= TM;
      load_to_lds((second ? from_q : from_p) + (static_cast<uint64_t>(offset[k]) + k0 * 8) * 16, to + k * THREADS * 8);
    }
  };
  static_assert(TM * 8 % THREADS == 0, "a load belongs to one operand");

  const uint32_t wi = wave / WN * (TM / WM), wj = wave % WN * (TN / WN);
  float4v acc[FM][FN] = {};
  issue(0);
  for (uint32_t step = 0; step < total; step++) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (step + 1 < total) issue(step + 1);
    if (SPLIT && step == 2 * steps) {
      for (int x = 0; x < FM; x++)
        for (int y = 0; y < FN; y++) acc[x][y] *= 1.f / kScaleLow;
    }
    const _Float16* stage = lds + (step & 1) * STAGE;
    for (int s = 0; s < 2; s++) {
      half8 fp[FM], fq[FN];
      const uint32_t chunk = s * 4 + lane / 16;
      for (int x = 0; x < FM; x++) {
        const uint32_t row = wi + x * 16 + lane % 16;
        fp[x] = *reinterpret_cast<const half8*>(stage + row * 64 + chunk_place(row, chunk) * 8);
      }
      for (int y = 0; y < FN; y++) {
        const uint32_t row = TM + wj + y * 16 + lane % 16;
        fq[y] = *reinterpret_cast<const half8*>(stage + row * 64 + chunk_place(row, chunk) * 8);
      }
      for (int x = 0; x < FM; x++)
        for (int y = 0; y < FN; y++) acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp[x], fq[y], acc[x][y], 0, 0, 0);
    }
  }

  // a lane holds rows 4 (lane / 16) + 0..3 and column lane % 16 of every 16 x 16 piece
  for (int x = 0; x < FM; x++) {
    const uint32_t i = i0 + wi + x * 16 + lane / 16 * 4;
    if (i >= m) continue;
    for (int y = 0; y < FN; y++) {
      const uint32_t j = j0 + wj + y * 16 + lane % 16;
      if (j >= rows_q) continue;
      half4 hi, lo;
      if (KIND == APPLY) {
        const uint64_t by_col = static_cast<uint64_t>(j) * m + i;
        const half4 old_hi = *reinterpret_cast<const half4*>(at + y_hi_at + by_col * 2);
        const half4 old_lo = *reinterpret_cast<const half4*>(at + y_lo_at + by_col * 2);
        for (int e = 0; e < 4; e++) {
          const float v = a * (static_cast<float>(old_hi[e]) + static_cast<float>(old_lo[e]) * (1.f / kScaleLow)) + acc[x][y][e] * (1.f / kScaleB);
          _Float16 h, l;
          split_value(v, &h, &l);
          hi[e] = h;
          lo[e] = l;
        }
        *reinterpret_cast<half4*>(at + y_hi_to + by_col * 2) = hi;
        *reinterpret_cast<half4*>(at + y_lo_to + by_col * 2) = lo;
        for (int e = 0; e < 4; e++) {
          const uint64_t by_row = static_cast<uint64_t>(i + e) * n + j;
          reinterpret_cast<_Float16*>(at + p.x_hi)[by_row] = hi[e];
          if (SPLIT) reinterpret_cast<_Float16*>(at + p.x_lo)[by_row] = lo[e];
        }
      } else {
        const uint64_t to_hi = KIND == GRAM ? p.a_hi : p.b_hi, to_lo = KIND == GRAM ? p.a_lo : p.b_lo;
        const uint64_t by_col = static_cast<uint64_t>(j) * m + i;
        half4 a_hi = {}, a_lo = {};
        if (KIND == SQUARE) {
          a_hi = *reinterpret_cast<const half4*>(at + p.a_hi + by_col * 2);
          if (SPLIT) a_lo = *reinterpret_cast<const half4*>(at + p.a_lo + by_col * 2);
        }
        for (int e = 0; e < 4; e++) {
          float v;
          if (KIND == GRAM) {
            v = acc[x][y][e] * (kScaleA / (kScaleX * kScaleX));
          } else {
            const float old = static_cast<float>(a_hi[e]) + (SPLIT ? static_cast<float>(a_lo[e]) * (1.f / kScaleLow) : 0.f);
            v = b * (kScaleB / kScaleA) * old + c * (kScaleB / kScaleA / kScaleA) * acc[x][y][e];
          }
          _Float16 h, l;
          split_value(v, &h, &l);
          hi[e] = h;
          lo[e] = l;
        }
        // the tile and, off the diagonal, its mirror image
        for (int e = 0; e < 4; e++) {
          const uint64_t by_row = static_cast<uint64_t>(i + e) * m + j;
          reinterpret_cast<_Float16*>(at + to_hi)[by_row] = hi[e];
          if (SPLIT) reinterpret_cast<_Float16*>(at + to_lo)[by_row] = lo[e];
        }
        if (ti != tj) {
          *reinterpret_cast<half4*>(at + to_hi + by_col * 2) = hi;
          if (SPLIT) *reinterpret_cast<half4*>(at + to_lo + by_col * 2) = lo;
        }
      }
    }
  }
}

// ---- the result -----------------------------------------------------------------------

// One block per 64 x 64 tile of the result: out = X (orthogonalize) or out = keep out - rate X (Muon).
template <typename T, bool SPLIT>
__global__ void __launch_bounds__(256) last_kernel(Segments segments, int from, int muon, float keep, const char* ws) {
  __shared__ float tile[64][65];
  const Segment& s = segments.at[find(segments, blockIdx.x)];
  const uint32_t matrix = (blockIdx.x - s.first_tile) / s.tiles, t = (blockIdx.x - s.first_tile) % s.tiles;
  const uint32_t m = static_cast<uint32_t>(round_up(s.tall ? s.cols : s.rows, kPad));
  const uint32_t n = static_cast<uint32_t>(round_up(s.tall ? s.rows : s.cols, kPad));
  const Planes p = planes_of(m, n, SPLIT);
  const char* at = ws + s.base + matrix * p.bytes;
  const _Float16* y_hi = reinterpret_cast<const _Float16*>(at + p.y_hi + from * p.y_hi_step);
  const _Float16* y_lo = reinterpret_cast<const _Float16*>(at + p.y_lo + from * p.y_lo_step);
  const uint32_t across = static_cast<uint32_t>(round_up(s.cols, 64)) / 64;
  const uint32_t r0 = t / across * 64, c0 = t % across * 64;
  // Y's rows are the result's rows if it is tall, else its columns
  for (uint32_t k = threadIdx.x; k < 64 * 64; k += 256) {
    const uint32_t i = k / 64, j = k % 64;
    const uint64_t from_at = static_cast<uint64_t>((s.tall ? r0 : c0) + i) * m + (s.tall ? c0 : r0) + j;
    const float v = (static_cast<float>(y_hi[from_at]) + static_cast<float>(y_lo[from_at]) * (1.f / kScaleLow)) * (1.f / kScaleX);
    if (s.tall) tile[i][j] = v;
    else tile[j][i] = v;
  }
  __syncthreads();
  const uint64_t size = static_cast<uint64_t>(s.rows) * s.cols;
  T* out = static_cast<T*>(s.out) + matrix * size;
  for (uint32_t k = threadIdx.x; k < 64 * 64; k += 256) {
    const uint32_t r = r0 + k / 64, c = c0 + k % 64;
    if (r >= s.rows || c >= s.cols) continue;
    const uint64_t to = static_cast<uint64_t>(r) * s.cols + c;
    const float v = tile[k / 64][k % 64];
    out[to] = from_float<T>(muon ? keep * to_float(out[to]) - s.rate * v : v);
  }
}

// ---- host side -----------------------------------------------------------------------

// What one run through the phases takes: segments in the order of their padded shapes, the groups they make.
struct Chunk {
  Segments segments;
  Groups groups;
  uint64_t bytes;
};

// Matrices of one chunk, beyond which more of them fill the GPU no better and only ask for more workspace.
constexpr uint64_t kChunkElements = 1ull << 26;

struct Item {
  size_t matrix, first, count;  // matrices [first, first + count) of the caller's batch `matrix`
  uint32_t m, n;
};

// Cuts the caller's list into chunks; visit(items, number of items) for each. No memory: items by value.
template <typename Visit>
int for_chunks(const step_matrix* list, size_t length, const Visit& visit) {
  Item items[kMostSegments];
  int used = 0;
  uint64_t elements = 0;
  auto flush = [&]() {
    if (!used) return static_cast<int>(STEP_OK);
    std::stable_sort(items, items + used, [](const Item& x, const Item& y) { return x.m != y.m ? x.m < y.m : x.n < y.n; });
    const int rc = visit(items, used);
    used = 0;
    elements = 0;
    return rc;
  };
  for (size_t k = 0; k < length; k++) {
    const size_t rows = list[k].rows, cols = list[k].cols;
    const uint32_t m = static_cast<uint32_t>(round_up(std::min(rows, cols), kPad));
    const uint32_t n = static_cast<uint32_t>(round_up(std::max(rows, cols), kPad));
    if (rows == 0 || cols == 0) continue;
    const uint64_t one = static_cast<uint64_t>(m) * n;
    size_t first = 0;
    while (first < list[k].count) {
      const uint64_t room = elements < kChunkElements ? (kChunkElements - elements) / one : 0;
      if (used == kMostSegments || (room == 0 && used)) {
        const int rc = flush();
        if (rc != STEP_OK) return rc;
        continue;
      }
      const size_t take = static_cast<size_t>(std::min<uint64_t>(list[k].count - first, std::max<uint64_t>(room, 1)));
      items[used++] = {k, first, take, m, n};
      elements += take * one;
      first += take;
    }
  }
  return flush();
}

uint64_t chunk_bytes(const Item* items, int count, bool split) {
  uint64_t bytes = 0;
  for (int k = 0; k < count; k++) bytes += planes_of(items[k].m, items[k].n, split).bytes * items[k].count;
  return bytes;
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

// By type: the update's T picks the kernels that read it, the result's the one that writes it.
template <typename Go> void by_type(int dtype, const Go& go) {
  if (dtype == STEP_F32) go(F32());
  else if (dtype == STEP_BF16) go(BF16());
  else go(F16());
}

template <int TM, int TN, int WM, int WN, Kind KIND, bool SPLIT>
void launch_product(Groups groups, const uint32_t* counts, char* ws, int from, float a, float b, float c, hipStream_t stream) {
  uint32_t tiles = 0;
  for (int k = 0; k < groups.count; k++) {
    Group& g = groups.at[k];
    const uint32_t down = (g.m + TM - 1) / TM, across = (g.n + TN - 1) / TN;
    g.tiles = KIND == APPLY ? down * across : down * (down + 1) / 2;
    g.first_tile = tiles;
    tiles += g.tiles * counts[k];
  }
  hipLaunchKernelGGL((product_kernel<TM, TN, WM, WN, KIND, SPLIT>), dim3(tiles), dim3(WM * WN * 64), 0, stream, groups, ws, from, a, b, c);
}

template <Kind KIND, bool SPLIT>
void product(const Groups& groups, const uint32_t* counts, char* ws, int from, const float* coefficients, hipStream_t stream) {
  launch_product<128, 128, 2, 2, KIND, SPLIT>(groups, counts, ws, from, coefficients[0], coefficients[1], coefficients[2], stream);
}

struct Rule {
  MomentumRule momentum;
  float eps, keep;
  int muon, steps;
  const float* coefficients;
};

template <bool SPLIT>
int run_chunk(const step_matrix* list, const Item* items, int count, int dtype, int out_dtype, const Rule& rule, char* ws,
              hipStream_t stream) {
  Segments segments;
  Groups groups;
  uint32_t counts[kMostSegments];
  segments.count = count;
  groups.count = 0;
  uint64_t at = 0;
  for (int k = 0; k < count; k++) {
    const Item& item = items[k];
    const step_matrix& x = list[item.matrix];
    const uint64_t size = static_cast<uint64_t>(x.rows) * x.cols, skip = item.first * size;
    Segment& s = segments.at[k];
    s.grad = static_cast<const char*>(x.grad) + skip * dtype_size(dtype);
    s.momentum = x.momentum ? x.momentum + skip : nullptr;
    s.out = static_cast<char*>(x.out) + skip * dtype_size(out_dtype);
    s.base = at;
    s.rows = static_cast<uint32_t>(x.rows);
    s.cols = static_cast<uint32_t>(x.cols);
    s.rate = x.rate;
    s.tall = x.rows > x.cols;
    if (groups.count && groups.at[groups.count - 1].m == item.m && groups.at[groups.count - 1].n == item.n) {
      counts[groups.count - 1] += static_cast<uint32_t>(item.count);
    } else {
      groups.at[groups.count] = {at, item.m, item.n, 0, 0};
      counts[groups.count++] = static_cast<uint32_t>(item.count);
    }
    at += planes_of(item.m, item.n, SPLIT).bytes * item.count;
  }
  uint32_t pieces = 0, tiles = 0;
  Segments by_piece = segments;
  for (int k = 0; k < count; k++) {
    Segment& s = segments.at[k];
    const uint64_t size = static_cast<uint64_t>(s.rows) * s.cols;
    Segment& q = by_piece.at[k];
    q.tiles = static_cast<uint32_t>(std::min<uint64_t>(size / 4096 + 1, kNormBlocks));
    q.first_tile = pieces;
    pieces += q.tiles * static_cast<uint32_t>(items[k].count);
    s.tiles = static_cast<uint32_t>(round_up(s.rows, 64) / 64 * (round_up(s.cols, 64) / 64));
    s.first_tile = tiles;
    tiles += s.tiles * static_cast<uint32_t>(items[k].count);
  }
  by_type(dtype, [&](auto type) {
    typedef decltype(type) T;
    hipLaunchKernelGGL((norm_kernel<T>), dim3(pieces), dim3(256), 0, stream, by_piece, rule.momentum, ws, SPLIT ? 1 : 0);
    hipLaunchKernelGGL((first_kernel<T, SPLIT>), dim3(tiles), dim3(256), 0, stream, segments, rule.momentum, rule.eps, ws);
  });
  int from = 0;
  for (int step = 0; step < rule.steps; step++) {
    const float* c = rule.coefficients + 3 * step;
    product<GRAM, SPLIT>(groups, counts, ws, from, c, stream);
    product<SQUARE, SPLIT>(groups, counts, ws, from, c, stream);
    product<APPLY, SPLIT>(groups, counts, ws, from, c, stream);
    from ^= 1;
  }
  by_type(out_dtype, [&](auto type) {
    typedef decltype(type) T;
    hipLaunchKernelGGL((last_kernel<T, SPLIT>), dim3(tiles), dim3(256), 0, stream, segments, from, rule.muon, rule.keep, static_cast<const char*>(ws));
  });
  return launched();
}

int run(const step_matrix* list, size_t length, int dtype, int out_dtype, int precise, const Rule& rule, void* workspace,
        size_t workspace_bytes, hipStream_t stream) {
  if (rule.steps < 0 || rule.steps > kMostSteps || (rule.steps && !rule.coefficients)) return STEP_ERR_ARGUMENT;
  const size_t need = step_orthogonalize_workspace(list, length, precise);
  if (need == 0) return STEP_OK;
  if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256) return STEP_ERR_ARGUMENT;
  char* ws = static_cast<char*>(workspace);
  return for_chunks(list, length, [&](const Item* items, int count) {
    return precise ? run_chunk<true>(list, items, count, dtype, out_dtype, rule, ws, stream)
                   : run_chunk<false>(list, items, count, dtype, out_dtype, rule, ws, stream);
  });
}

}  // namespace
}  // namespace step

using namespace step;

extern "C" {

size_t step_orthogonalize_workspace(const step_matrix* list, size_t length, int precise) {
  uint64_t most = 0;
  if (length && !list) return 0;
  for_chunks(list, length, [&](const Item* items, int count) {
    most = std::max(most, chunk_bytes(items, count, precise != 0));
    return static_cast<int>(STEP_OK);
  });
  return most;
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
