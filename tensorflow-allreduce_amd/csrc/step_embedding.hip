// Embedding lookup, its gradient by sorted tokens, and the sum of gathered
// sparse rows for MI355X (gfx950): include/step_abi.h.
//
// Mathematics. With ids i_t (t < T) and a table W of V rows of D columns:
//   lookup     O[t, :]  = round(s * W[i_t, :])
//   gradient   dW[v, :] = round(s * sum over {t : i_t = v}, in order of t, of G[t, :])
// One multiplication (addition) per element read: bound by HBM bandwidth, the
// small calls by their launches.
//
// The gradient is gathered, not scattered: atomic additions into dW would
// serialise on the common tokens, need a float32 image of the whole table and
// change the result from call to call. Instead the positions are sorted by id
// (a stable least-significant-digit radix sort of (id, t) pairs, ids first cut
// to the bits that `rows` needs), which makes the rows of one id a run of
// ascending t, and every row of dW is summed by the lanes that store it:
// one read of G, one write of dW, in the table's own type.
//   * up to kOneGroup tokens one workgroup sorts them in LDS: one launch;
//   * more tokens take two launches per digit (count, then scatter; the scatter
//     adds up the counts of all tiles itself instead of a scan in between);
//   * the sorted order is cut into windows of 8 places; the lanes of a window sum
//     and store the runs that begin in it, in batches of 8 rows in flight;
//   * a run longer than a piece (a common token: thousands of rows) is cut at
//     multiples of the piece's length; each part is summed by a workgroup of its
//     own into 32 bits, and a second launch adds the parts in order;
//   * the same launch clears dW's empty rows, found without clearing a table
//     first: begin[v] is trusted only if the sorted ids say that a run of v begins
//     there.
#include "step_common.h"

namespace step {
namespace {

thread_local int g_last_hip_error = 0;

// A key is an id cut to 32 bits; every id outside [0, rows) becomes `rows`, sorts
// behind all rows and is dropped there.
__device__ __forceinline__ uint32_t key_of(const void* ids, int id_type, uint32_t t, uint32_t rows) {
  if (id_type == STEP_I32) {
    const uint32_t k = static_cast<const uint32_t*>(ids)[t];  // negative: large
    return k < rows ? k : rows;
  }
  const uint64_t k = static_cast<const uint64_t*>(ids)[t];
  return k < rows ? static_cast<uint32_t>(k) : rows;
}

// ---- lookup ---------------------------------------------------------------------

// Lanes of one row of a launch: `lanes` of them, each 16 bytes wide, side by side;
// a row wider than a workgroup is cut into `chunks` column ranges (grid y).
struct RowShape {
  uint32_t lanes, rows_per_group, chunks;
};

RowShape row_shape(size_t vectors) {
  RowShape s;
  s.chunks = static_cast<uint32_t>((vectors + 255) / 256);
  const size_t per_chunk = (vectors + s.chunks - 1) / s.chunks;
  if (per_chunk <= 32) {  // else whole waves
    s.lanes = 1;
    while (s.lanes < per_chunk) s.lanes *= 2;
  } else {
    s.lanes = static_cast<uint32_t>(round_up(per_chunk, 64));
  }
  s.rows_per_group = 256 / s.lanes;
  return s;
}

template <typename T> struct RawOf { typedef uint32_t type __attribute__((ext_vector_type(4))); };

template <typename T> struct Access {
  // rows of odd widths break 16-byte alignment: element-aligned 16-byte accesses
  typedef typename RawOf<T>::type Raw;
  typedef Raw RawU __attribute__((aligned(sizeof(T))));
  static constexpr uint32_t kCount = Vec<T>::kCount;

  // The first of the columns of a row's vector v. The last vector of a row whose width is no multiple of a vector's ends
  // with the row, so that it is loaded as a whole too; it stores only what the one before it does not.
  static __device__ __forceinline__ uint32_t column(uint32_t v, uint32_t width) {
    return v * kCount + kCount <= width || width < kCount ? v * kCount : width - kCount;
  }
  // `width` < kCount: a row narrower than a vector
  static __device__ __forceinline__ Vec<T> load(const T* p, uint32_t width) {
    Vec<T> v;
    if (width >= kCount) {
      v = __builtin_bit_cast(Vec<T>, static_cast<Raw>(*reinterpret_cast<const RawU*>(p)));
    } else {
      v = __builtin_bit_cast(Vec<T>, Raw{0, 0, 0, 0});
      for (uint32_t k = 0; k < kCount; k++)
        if (k < width) v.at[k] = p[k];
    }
    return v;
  }
  // Vector `vector` of the row that begins at `row`. PASSING: see leaves_caches(). (No argument: the compiler makes one
  // unmarked store of the two sides of a branch.)
  template <bool PASSING> static __device__ __forceinline__ void store(T* row, Vec<T> v, uint32_t vector, uint32_t width) {
    T* p = row + column(vector, width);
    if (vector * kCount + kCount <= width) {
      if (PASSING) __builtin_nontemporal_store(__builtin_bit_cast(Raw, v), reinterpret_cast<RawU*>(p));
      else *reinterpret_cast<RawU*>(p) = __builtin_bit_cast(Raw, v);
    } else {
      const uint32_t skip = vector * kCount - column(vector, width);
      for (uint32_t k = 0; k < kCount; k++)
        if (k >= skip && k < width) p[k] = v.at[k];
    }
  }
};

// Whether a result is larger than the caches (256 MiB behind the L2s), so that no reader finds it there: its stores then
// pass them by, and what is still to be read stays. A lookup of 131072 x 4096 bf16 rows 332 us without, 311 with; the
// gradient of 100000 such rows from 65536 tokens 343 and 329 alone, 776 and 752 with an optimizer that reads it. Smaller
// results lose: the gradient of 32000 such rows 100 and 93 alone, but 235 and 241 with its reader.
bool leaves_caches(size_t rows, size_t width, size_t bytes) { return rows * width * bytes > size_t(256) << 20; }

// Bound by HBM where the call is long (131072 rows of 4096 bf16 columns: 311 us, 6.9 TB/s of rows read and written, some
// of them from caches), by the launch where it is short (16 rows: 4 us of kernel, 8 us a call).
constexpr int kLookupRows = 4;  // rows a lane loads before it stores the first

template <typename T, bool PASSING>
__global__ void lookup_kernel(const void* ids, int id_type, uint32_t tokens, const T* weight, uint32_t rows,
                              uint32_t width, uint64_t weight_stride, float scale, T* out, uint32_t lanes,
                              uint32_t rows_per_group) {
  constexpr int N = Vec<T>::kCount;
  const uint32_t slot = threadIdx.x / lanes;
  const uint32_t vector = blockIdx.y * lanes + threadIdx.x % lanes;
  if (slot >= rows_per_group || vector * N >= width) return;
  const uint32_t column = Access<T>::column(vector, width);
  const uint64_t first = static_cast<uint64_t>(blockIdx.x) * rows_per_group * kLookupRows + slot;
  uint32_t key[kLookupRows];
  Vec<T> v[kLookupRows];
  for (int k = 0; k < kLookupRows; k++) {
    const uint64_t t = first + k * rows_per_group;
    key[k] = t < tokens ? key_of(ids, id_type, static_cast<uint32_t>(t), rows) : rows;
  }
  for (int k = 0; k < kLookupRows; k++)
    if (key[k] < rows) v[k] = Access<T>::load(weight + key[k] * weight_stride + column, width);
  for (int k = 0; k < kLookupRows; k++) {
    const uint64_t t = first + k * rows_per_group;
    if (t >= tokens) return;
    for (int e = 0; e < N; e++)
      v[k].at[e] = from_float<T>(key[k] < rows ? scale * to_float(v[k].at[e]) : 0.f);
    Access<T>::template store<PASSING>(out + t * width, v[k], vector, width);
  }
}

// ---- sort -------------------------------------------------------------------------

// (a build for the CPU, where every lane is a thread, takes smaller ones)
#ifndef STEP_SORT_THREADS
#define STEP_SORT_THREADS 1024
#define STEP_DIGIT_BITS 9
#endif
constexpr int kMostDigitBits = STEP_DIGIT_BITS;
constexpr int kBins = 1 << kMostDigitBits;
constexpr uint32_t kSortThreads = STEP_SORT_THREADS;
constexpr uint32_t kWaves = kSortThreads / 64;
static_assert(kSortThreads >= static_cast<uint32_t>(kBins), "one lane per digit");
// Tokens one workgroup sorts in LDS. Numbering the runs takes two launches more where several workgroups sort: 10007 tokens
// of 64 columns as slices 65 us in one workgroup and 73 in several, as a gradient 39 either way (8192: 33 in one).
constexpr uint32_t kOneGroup = 8 * kSortThreads, kOneGroupNumbered = 12 * kSortThreads;
constexpr int kTileKeys = 4;                              // keys per lane of a tile of the several-workgroup sort
constexpr uint32_t kTile = kSortThreads * kTileKeys;
// above that many tiles each pass would spend its time reading counts; tiles get longer instead
constexpr uint32_t kMostTiles = 256;

struct Digits {
  int bits, passes;
};

// Digits of at most 9 bits: a table of fewer than 2^18 rows takes two passes (the key `rows` needs bits too).
Digits digits_for(size_t rows) {
  int bits = 1;
  while (bits < 32 && (rows >> bits) != 0) bits++;
  Digits d;
  d.passes = (bits + kMostDigitBits - 1) / kMostDigitBits;
  d.bits = (bits + d.passes - 1) / d.passes;
  return d;
}

struct RankScratch {
  uint16_t count[kWaves][kBins];  // per wave: keys of each digit seen so far, then those in earlier waves (< 2^14)
  uint32_t total[kBins];
  uint32_t wave_sum[kWaves];
};

// The ranks of a round: the number of lanes of this wave before mine with my digit, and their mask. Every lane of the
// workgroup takes part in every round.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, int bits) {
  uint64_t peers = ~0ull;
  for (int b = 0; b < bits; b++) {
    const uint64_t set = __ballot((digit >> b) & 1);
    peers &= (digit >> b) & 1 ? set : ~set;
  }
  return peers;
}

__device__ __forceinline__ void wave_fence() {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#elif defined(STEP_WAVE_SHIM_H_)
  step_wave_fence();
#endif
}

// Counts the digits of `K` keys per lane, wave by wave in order, and leaves in rank[k] the key's place among those of
// its digit in its wave, in s.count[w][d] how many of digit d stand in waves before w, in s.total[d] the workgroup's
// count of digit d. A key at or behind `limit` (in the order of the waves' keys) takes no part.
template <int K>
__device__ __forceinline__ void rank_keys(RankScratch& s, const uint32_t (&key)[K], uint32_t (&rank)[K], uint32_t first,
                                          uint32_t limit, int shift, int bits) {
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const uint32_t bins = 1u << bits;
  for (uint32_t d = threadIdx.x; d < kWaves * kBins; d += kSortThreads) s.count[d / kBins][d % kBins] = 0;
  __syncthreads();
  for (int k = 0; k < K; k++) {
    const uint32_t digit = (key[k] >> shift) & (bins - 1);
    const bool here = first + k * 64 + lane < limit;
    const uint64_t peers = same_digit(digit, bits) & __ballot(here);
    const uint64_t before = peers & ((1ull << lane) - 1);
    const uint32_t seen = s.count[wave][digit];
    wave_fence();
    rank[k] = seen + static_cast<uint32_t>(__popcll(before));
    if (here && before == 0) s.count[wave][digit] = static_cast<uint16_t>(seen + __popcll(peers));
    wave_fence();
  }
  __syncthreads();
  for (uint32_t d = threadIdx.x; d < bins; d += kSortThreads) {
    uint32_t sum = 0;
    for (uint32_t w = 0; w < kWaves; w++) {
      const uint32_t c = s.count[w][d];
      s.count[w][d] = static_cast<uint16_t>(sum);
      sum += c;
    }
    s.total[d] = sum;
  }
  __syncthreads();
}

// Exclusive prefix sum of x over the workgroup; s.wave_sum is scratch. Every lane takes part.
__device__ __forceinline__ uint32_t group_scan(RankScratch& s, uint32_t x, uint32_t* sum) {
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  uint32_t up_to = x;
  for (int step = 1; step < 64; step *= 2) {
    const uint32_t other = __shfl_up(up_to, step);
    if (lane >= static_cast<uint32_t>(step)) up_to += other;
  }
  if (lane == 63) s.wave_sum[wave] = up_to;
  __syncthreads();
  uint32_t before = 0, all = 0;
  for (uint32_t w = 0; w < kWaves; w++) {
    if (w < wave) before += s.wave_sum[w];
    all += s.wave_sum[w];
  }
  __syncthreads();
  *sum = all;
  return before + up_to - x;
}

// What the sort leaves in the workspace. `order[i]` is the token at place i of the sorted order and `row_of[i]` its row
// of the output: the id itself (gradient), or the number of its run (sum_slices); ids outside the table stand last,
// with row_of = rows. Run r covers the places begin[r] .. end[r] - 1 (sum_slices: end[r] is begin[r + 1]).
struct Sorted {
  uint32_t* order;
  uint32_t* row_of;
  uint32_t* begin;
  uint32_t* end;
};

// Everything of the sort in one workgroup's LDS, and the runs. Bound by the chain of ballots and LDS accesses of a round of
// 64 keys per wave: 1024 tokens 7 us, 2048 11, 4096 15, 8192 23, 12288 30 (two passes). Above, several workgroups: 8193 tokens 32 us
// in five launches (count 3, scatter 11 per pass, runs 4), 65536 tokens 36.
template <int K>
__global__ void __launch_bounds__(kSortThreads) sort_one_kernel(const void* ids, int id_type, uint32_t tokens,
                                                                uint32_t rows, int bits, int passes, Sorted to,
                                                                int number_runs, void* out_ids, int64_t* out_count) {
  __shared__ RankScratch s;
  __shared__ uint32_t keys[K * kSortThreads];
  __shared__ uint16_t from[K * kSortThreads];
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const uint32_t first = wave * 64 * K;
  uint32_t key[K], token[K], rank[K];
  for (int k = 0; k < K; k++) {
    const uint32_t t = first + k * 64 + lane;
    token[k] = t;
    key[k] = t < tokens ? key_of(ids, id_type, t, rows) : rows;
  }
  for (int pass = 0; pass < passes; pass++) {
    const int shift = pass * bits;
    rank_keys<K>(s, key, rank, first, tokens, shift, bits);
    uint32_t all;
    const uint32_t d = threadIdx.x;
    const uint32_t before = group_scan(s, d < (1u << bits) ? s.total[d] : 0, &all);
    if (d < (1u << bits)) s.total[d] = before;
    __syncthreads();
    for (int k = 0; k < K; k++) {
      if (first + k * 64 + lane >= tokens) continue;
      const uint32_t digit = (key[k] >> shift) & ((1u << bits) - 1);
      const uint32_t at = s.total[digit] + s.count[wave][digit] + rank[k];
      keys[at] = key[k];
      from[at] = static_cast<uint16_t>(token[k]);
    }
    __syncthreads();
    for (int k = 0; k < K; k++) {
      const uint32_t t = first + k * 64 + lane;
      if (t >= tokens) continue;
      key[k] = keys[t];
      token[k] = from[t];
    }
    // the next pass writes keys[] behind barriers of its own
  }
  for (int k = 0; k < K; k++) {
    const uint32_t i = first + k * 64 + lane;
    // a run begins at i (and ends at i + 1) if the neighbouring key differs
    const bool begins = i < tokens && key[k] < rows && (i == 0 || keys[i - 1] != key[k]);
    const bool ends = i < tokens && key[k] < rows && (i + 1 == tokens || keys[i + 1] != key[k]);
    rank[k] = (begins ? 1u : 0u) | (ends ? 2u : 0u);
  }
  if (!number_runs) {
    for (int k = 0; k < K; k++) {
      const uint32_t i = first + k * 64 + lane;
      if (i >= tokens) continue;
      to.order[i] = token[k];
      to.row_of[i] = key[k];
      if (rank[k] & 1) to.begin[key[k]] = i;
      if (rank[k] & 2) to.end[key[k]] = i + 1;
    }
    return;
  }
  // the number of a run: how many begin before it, counted over waves, then rounds, then lanes
  uint32_t all;
  uint32_t in_wave = 0;
  for (int k = 0; k < K; k++) in_wave += static_cast<uint32_t>(__popcll(__ballot(rank[k] & 1)));
  uint32_t number = group_scan(s, lane == 0 ? in_wave : 0, &all);
  number = __shfl(number, 0);
  for (int k = 0; k < K; k++) {
    const uint32_t i = first + k * 64 + lane;
    const uint64_t starts = __ballot(rank[k] & 1);
    const uint32_t up_to = number + static_cast<uint32_t>(__popcll(starts & ((2ull << lane) - 1)));
    number += static_cast<uint32_t>(__popcll(starts));
    if (i >= tokens) continue;
    to.order[i] = token[k];
    const bool in_table = key[k] < rows;
    to.row_of[i] = in_table ? up_to - 1 : rows;
    if (rank[k] & 1) {
      to.begin[up_to - 1] = i;
      if (id_type == STEP_I32) static_cast<int32_t*>(out_ids)[up_to - 1] = static_cast<int32_t>(key[k]);
      else static_cast<int64_t*>(out_ids)[up_to - 1] = key[k];
    }
    if ((rank[k] & 2) && (i + 1 == tokens || keys[i + 1] >= rows)) to.begin[all] = i + 1;  // the last run's end
  }
  if (threadIdx.x == 0) *out_count = all;
}

// Several workgroups: the counts of a tile's digits, counts[tile * bins + digit].
__global__ void __launch_bounds__(kSortThreads) count_kernel(const void* ids, int id_type, const uint32_t* in_keys,
                                                             uint32_t tokens, uint32_t rows, uint32_t tile_length,
                                                             int shift, int bits, uint32_t* counts) {
  __shared__ uint32_t count[kBins];
  const uint32_t bins = 1u << bits;
  if (threadIdx.x < bins) count[threadIdx.x] = 0;
  __syncthreads();
  const uint64_t first = static_cast<uint64_t>(blockIdx.x) * tile_length;
  for (uint32_t j = threadIdx.x; j < tile_length; j += kSortThreads) {
    const uint64_t t = first + j;
    if (t >= tokens) break;
    const uint32_t key = in_keys ? in_keys[t] : key_of(ids, id_type, static_cast<uint32_t>(t), rows);
    atomicAdd(&count[(key >> shift) & (bins - 1)], 1u);
  }
  __syncthreads();
  if (threadIdx.x < bins) counts[static_cast<uint64_t>(blockIdx.x) * bins + threadIdx.x] = count[threadIdx.x];
}

// The scatter of a digit's pass. A digit's keys of this tile go behind all smaller digits' keys and those of the same
// digit in earlier tiles.
__global__ void __launch_bounds__(kSortThreads) scatter_kernel(const void* ids, int id_type, const uint32_t* in_keys,
                                                               const uint32_t* in_order, uint32_t tokens, uint32_t rows,
                                                               uint32_t tile_length, int shift, int bits,
                                                               const uint32_t* counts, uint32_t* out_keys,
                                                               uint32_t* out_order) {
  __shared__ RankScratch s;
  __shared__ uint32_t base[kBins];
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const uint32_t bins = 1u << bits;
  uint32_t in_earlier = 0, in_all = 0;
  if (threadIdx.x < bins) {
#pragma unroll 8
    for (uint32_t b = 0; b < gridDim.x; b++) {
      const uint32_t c = counts[static_cast<uint64_t>(b) * bins + threadIdx.x];
      if (b < blockIdx.x) in_earlier += c;
      in_all += c;
    }
  }
  uint32_t all;
  const uint32_t smaller = group_scan(s, in_all, &all);
  if (threadIdx.x < bins) base[threadIdx.x] = smaller + in_earlier;
  __syncthreads();
  const uint64_t tile = static_cast<uint64_t>(blockIdx.x) * tile_length;
  for (uint32_t part = 0; part < tile_length; part += kTile) {
    const uint64_t at0 = tile + part;
    const uint32_t here = at0 >= tokens ? 0 : tokens - at0 < kTile ? static_cast<uint32_t>(tokens - at0) : kTile;
    const uint32_t first = wave * 64 * kTileKeys;
    uint32_t key[kTileKeys], token[kTileKeys], rank[kTileKeys];
    for (int k = 0; k < kTileKeys; k++) {
      const uint32_t j = first + k * 64 + lane;
      key[k] = rows;
      token[k] = 0;
      if (j < here) {
        const uint32_t t = static_cast<uint32_t>(at0 + j);
        key[k] = in_keys ? in_keys[t] : key_of(ids, id_type, t, rows);
        token[k] = in_order ? in_order[t] : t;
      }
    }
    rank_keys<kTileKeys>(s, key, rank, first, here, shift, bits);
    for (int k = 0; k < kTileKeys; k++) {
      if (first + k * 64 + lane >= here) continue;
      const uint32_t digit = (key[k] >> shift) & (bins - 1);
      const uint32_t at = base[digit] + s.count[wave][digit] + rank[k];
      out_keys[at] = key[k];
      out_order[at] = token[k];
    }
    __syncthreads();
    if (threadIdx.x < bins) base[threadIdx.x] += s.total[threadIdx.x];
    __syncthreads();
  }
}

// The runs of the sorted keys: where each key's begins and ends (gradient).
__global__ void __launch_bounds__(kSortThreads) runs_kernel(const uint32_t* keys, uint32_t tokens, uint32_t rows,
                                                            Sorted to) {
  const uint64_t i = static_cast<uint64_t>(blockIdx.x) * kSortThreads + threadIdx.x;
  if (i >= tokens) return;
  const uint32_t key = keys[i];
  if (key >= rows) return;
  if (i == 0 || keys[i - 1] != key) to.begin[key] = static_cast<uint32_t>(i);
  if (i + 1 == tokens || keys[i + 1] != key) to.end[key] = static_cast<uint32_t>(i + 1);
}

__device__ __forceinline__ bool begins_run(const uint32_t* keys, uint64_t i, uint32_t tokens, uint32_t rows) {
  if (i >= tokens) return false;
  const uint32_t key = keys[i];
  return key < rows && (i == 0 || keys[i - 1] != key);
}

// Runs by number (sum_slices): one launch counts those that begin in each tile, the next numbers them.
__global__ void __launch_bounds__(kSortThreads) count_runs_kernel(const uint32_t* keys, uint32_t tokens, uint32_t rows,
                                                                  uint32_t tile_length, uint32_t* counts) {
  __shared__ RankScratch s;
  const uint64_t first = static_cast<uint64_t>(blockIdx.x) * tile_length;
  uint32_t mine = 0;
  for (uint32_t j = threadIdx.x; j < tile_length; j += kSortThreads) mine += begins_run(keys, first + j, tokens, rows);
  uint32_t all;
  group_scan(s, mine, &all);
  if (threadIdx.x == 0) counts[blockIdx.x] = all;
}

__global__ void __launch_bounds__(kSortThreads) number_runs_kernel(const uint32_t* keys, uint32_t tokens, uint32_t rows,
                                                                   uint32_t tile_length, const uint32_t* counts, Sorted to,
                                                                   int id_type, void* out_ids, int64_t* out_count) {
  __shared__ RankScratch s;
  uint32_t earlier = 0, in_all = 0;
  for (uint32_t b = threadIdx.x; b < gridDim.x; b += kSortThreads) {
    const uint32_t c = counts[b];
    in_all += c;
    if (b < blockIdx.x) earlier += c;
  }
  uint32_t number, total;
  group_scan(s, earlier, &number);
  group_scan(s, in_all, &total);
  const uint64_t tile = static_cast<uint64_t>(blockIdx.x) * tile_length;
  for (uint32_t part = 0; part < tile_length; part += kTile) {
    // kTileKeys places of a lane, one behind the other
    const uint64_t first = tile + part + threadIdx.x * kTileKeys;
    uint32_t key[kTileKeys + 2], mine = 0;  // and the places before and behind them
    bool begins[kTileKeys];
    for (int k = 0; k < kTileKeys + 2; k++) {
      const uint64_t i = first + k - 1;
      key[k] = i < tokens ? keys[i] : 0xffffffffu;  // before the first place, i wraps
    }
    for (int k = 0; k < kTileKeys; k++) {
      begins[k] = key[k + 1] < rows && key[k + 1] != key[k];
      mine += begins[k];
    }
    uint32_t here;
    uint32_t run = number + group_scan(s, mine, &here);  // runs that begin before this place
    for (int k = 0; k < kTileKeys; k++) {
      const uint64_t i = first + k;
      if (i >= tokens) break;
      if (begins[k]) {
        to.begin[run] = static_cast<uint32_t>(i);
        if (id_type == STEP_I32) static_cast<int32_t*>(out_ids)[run] = static_cast<int32_t>(key[k + 1]);
        else static_cast<int64_t*>(out_ids)[run] = key[k + 1];
        run++;
      }
      to.row_of[i] = key[k + 1] < rows ? run - 1 : rows;
      if (key[k + 1] < rows && key[k + 2] >= rows) to.begin[total] = static_cast<uint32_t>(i + 1);  // the last run's end
    }
    number += here;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *out_count = total;
}

// ---- sums ------------------------------------------------------------------------

// What lane `from` (the same for all) holds, for every lane of its wave.
__device__ __forceinline__ uint32_t broadcast(uint32_t x, uint32_t from) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_readlane(x, from);
#else
  return __shfl(x, static_cast<int>(from));
#endif
}

constexpr uint32_t kWindow = 8;     // places of the sorted order whose runs one row of lanes sums
constexpr uint32_t kNoRow = 0xffffffffu;
constexpr uint32_t kZeroRows = 64;  // rows of a workgroup that looks for empty ones

struct Sums {
  uint64_t stride, parts_stride;
  uint32_t tokens, rows, width;
  float scale;
  Sorted by;
  uint32_t piece, pieces;                   // length of a long run's parts, and how many places of that length there are
  uint32_t lanes, rows_per_group, chunks;   // RowShape
  uint32_t piece_groups, window_groups;     // workgroups of the parts and of the windows; the rest clear
};

template <typename T> __device__ __forceinline__ void add(float (&acc)[Vec<T>::kCount], const Vec<T>& v) {
  for (int n = 0; n < Vec<T>::kCount; n++) acc[n] += to_float(v.at[n]);
}

template <typename T, bool PASSING>
__device__ __forceinline__ void put(T* row, const float (&acc)[Vec<T>::kCount], float scale, uint32_t vector, uint32_t width) {
  Vec<T> v;
  for (int n = 0; n < Vec<T>::kCount; n++) v.at[n] = from_float<T>(scale * acc[n]);
  Access<T>::template store<PASSING>(row, v, vector, width);
}

// The runs that begin in a window and are no longer than a piece. A run's rows are added in the order of the tokens.
template <typename T, bool PASSING>
__device__ __forceinline__ void sum_window(const Sums& q, const T* values, T* out, uint32_t window, uint32_t vector) {
  constexpr int N = Vec<T>::kCount;
  const uint32_t column = Access<T>::column(vector, q.width);
  const uint64_t w0 = static_cast<uint64_t>(window) * kWindow, w1 = w0 + kWindow;
  auto row_at = [&](uint64_t i) { return i < q.tokens ? q.by.row_of[i] : kNoRow; };
  float acc[N];
  uint32_t before = w0 ? q.by.row_of[w0 - 1] : kNoRow, open = kNoRow;  // open: the row being summed
  for (uint64_t i = w0;; i += 8) {
    uint32_t row[8], ahead[8], order[8];
    for (int k = 0; k < 8; k++) {
      row[k] = row_at(i + k);
      ahead[k] = row_at(i + k + q.piece);
      order[k] = i + k < q.tokens ? q.by.order[i + k] : 0;
    }
    // what each place does: nothing, begin a run, go on with it
    bool take[8], begin[8], stop = false;
    for (int k = 0; k < 8; k++) {
      take[k] = begin[k] = false;
      if (stop) continue;
      if (row[k] != before) {
        before = row[k];
        // the end: of the window, of the rows (dropped ids and the places behind the last have larger numbers), or a
        // long run, which lasts beyond the window
        if (i + k >= w1 || row[k] >= q.rows || ahead[k] == row[k]) stop = true;
        else take[k] = begin[k] = true;
      } else {
        take[k] = open != kNoRow || (k && take[k - 1]);
        if (!take[k] && i + k >= w1) stop = true;                 // a run that began before the window and outlasts it
      }
    }
    Vec<T> v[8];
    for (int k = 0; k < 8; k++)
      if (take[k]) v[k] = Access<T>::load(values + order[k] * q.stride + column, q.width);
    for (int k = 0; k < 8; k++) {
      if (!take[k]) continue;
      if (begin[k]) {
        if (open != kNoRow) put<T, PASSING>(out + static_cast<uint64_t>(open) * q.width, acc, q.scale, vector, q.width);
        open = row[k];
        for (int n = 0; n < N; n++) acc[n] = 0.f;
      }
      add<T>(acc, v[k]);
    }
    if (stop || (open == kNoRow && i + 8 >= w1)) break;
  }
  if (open != kNoRow) put<T, PASSING>(out + static_cast<uint64_t>(open) * q.width, acc, q.scale, vector, q.width);
}

// The same where a row takes whole waves: the lanes of a wave look at 64 places at once and hand what they saw to all.
// `mine`: whether this lane has columns; the others only look.
template <typename T, bool PASSING>
__device__ __forceinline__ void sum_window_wide(const Sums& q, const T* values, T* out, uint32_t window, uint32_t vector, bool mine) {
  constexpr int N = Vec<T>::kCount;
  const uint32_t column = mine ? Access<T>::column(vector, q.width) : 0, lane = threadIdx.x % 64;
  const uint64_t w0 = static_cast<uint64_t>(window) * kWindow;
  float acc[N];
  uint32_t open = kNoRow;
  auto close = [&]() {
    if (mine && open != kNoRow) put<T, PASSING>(out + static_cast<uint64_t>(open) * q.width, acc, q.scale, vector, q.width);
  };
  for (uint64_t base = w0;; base += 64) {
    const uint64_t i = base + lane;
    const uint32_t row = i < q.tokens ? q.by.row_of[i] : kNoRow, order = i < q.tokens ? q.by.order[i] : 0;
    const uint32_t before = i && i - 1 < q.tokens ? q.by.row_of[i - 1] : kNoRow;
    const uint32_t ahead = i + q.piece < q.tokens ? q.by.row_of[i + q.piece] : kNoRow;
    const bool starts = row != before, usable = base == w0 && lane < kWindow && row < q.rows && ahead != row;
    // where runs of this window begin, and where there is nothing more to do: at a later window's run, at a dropped id
    // or behind the last place, at a long run
    const uint64_t begins = __ballot(starts && usable), stops = __ballot((starts || row == kNoRow) && !usable);
    const uint32_t end = stops ? static_cast<uint32_t>(__builtin_ctzll(stops)) : 64;
    uint32_t p = base == w0 ? (begins ? static_cast<uint32_t>(__builtin_ctzll(begins)) : 64) : 0;
    if (p >= end) break;
    auto add_rows = [&](auto rows) {
      constexpr int U = decltype(rows)::value;
      Vec<T> v[U];
#pragma unroll
      for (int k = 0; k < U; k++) {
        const uint32_t from = broadcast(order, p + k);
        if (mine) v[k] = Access<T>::load(values + from * q.stride + column, q.width);
      }
#pragma unroll
      for (int k = 0; k < U; k++) {
        if (begins >> (p + k) & 1) {
          close();
          open = broadcast(row, p + k);
          for (int n = 0; n < N; n++) acc[n] = 0.f;
        }
        if (mine) add<T>(acc, v[k]);
      }
      p += U;
    };
    while (end - p >= 16) add_rows(std::integral_constant<int, 16>());
    if (end - p >= 8) add_rows(std::integral_constant<int, 8>());
    if (end - p >= 4) add_rows(std::integral_constant<int, 4>());
    if (end - p >= 2) add_rows(std::integral_constant<int, 2>());
    if (end - p >= 1) add_rows(std::integral_constant<int, 1>());
    if (end < 64) break;
  }
  close();
}

// A long run's part: piece j holds the places j * piece .. of the sorted order. At most two long runs have a part in it,
// that of its first place (parts[2 j]) and that of its last (parts[2 j + 1]).
template <typename T, bool NUMBERED, bool WIDE>
__device__ __forceinline__ void sum_piece(const Sums& q, const T* values, float* parts, uint32_t piece, uint32_t vector, bool mine) {
  constexpr int N = Vec<T>::kCount;
  const uint32_t column = mine ? Access<T>::column(vector, q.width) : 0;
  const uint64_t first = static_cast<uint64_t>(piece) * q.piece;
  const uint32_t last = q.tokens - first < q.piece ? q.tokens - 1 : static_cast<uint32_t>(first) + q.piece - 1;
  for (int side = 0; side < 2; side++) {
    const uint32_t place = side ? last : static_cast<uint32_t>(first);
    const uint32_t run = q.by.row_of[place];
    if (run >= q.rows || (side && run == q.by.row_of[first])) continue;
    const uint32_t b = q.by.begin[run], e = NUMBERED ? q.by.begin[run + 1] : q.by.end[run];
    if (e - b <= q.piece) continue;
    uint32_t i = b > first ? b : static_cast<uint32_t>(first);
    const uint32_t end = e <= last ? e : last + 1;
    float acc[N] = {};
    auto add_rows = [&](auto rows, auto order) {
      constexpr int U = decltype(rows)::value;
      Vec<T> v[U];
#pragma unroll
      for (int k = 0; k < U; k++) {
        const uint32_t from = order(k);
        if (mine) v[k] = Access<T>::load(values + from * q.stride + column, q.width);
      }
#pragma unroll
      for (int k = 0; k < U; k++)
        if (mine) add<T>(acc, v[k]);
    };
    if (WIDE) {
      for (; i < end; i += 64) {
        const uint32_t left = end - i < 64 ? end - i : 64, lane = threadIdx.x % 64;
        const uint32_t order = lane < left ? q.by.order[i + lane] : 0;
        uint32_t p = 0;
        auto at = [&](int k) { return broadcast(order, p + k); };
        for (; p + 16 <= left; p += 16) add_rows(std::integral_constant<int, 16>(), at);
        if (p + 8 <= left) { add_rows(std::integral_constant<int, 8>(), at); p += 8; }
        for (; p < left; p++) add_rows(std::integral_constant<int, 1>(), at);
      }
    } else {
      auto at = [&](int k) { return q.by.order[i + k]; };
      for (; i + 8 <= end; i += 8) add_rows(std::integral_constant<int, 8>(), at);
      for (; i < end; i++) add_rows(std::integral_constant<int, 1>(), at);
    }
    if (!mine) continue;
    float* to = parts + (static_cast<uint64_t>(piece) * 2 + side) * q.parts_stride + column;
    const uint32_t skip = vector * N - column;   // what the vector before stores
    for (int n = 0; n < N; n++)
      if (static_cast<uint32_t>(n) >= skip) to[n] = acc[n];
  }
}

// WIDE: a row takes whole waves, so that all lanes of a wave have the same row: then they read 64 places of the order with
// one load each and hand them round, instead of 24 loads that every lane makes for 8 places. 1024 tokens of 512 f32 columns
// 16 -> 10 us; long calls do not change: 65536 tokens of 2048 bf16 columns into 131072 rows 186 us, 0.8 GB at 4.3 TB/s,
// where a copy of that size reaches 6.5.
template <typename T, bool NUMBERED, bool WIDE, bool PASSING>
__global__ void __launch_bounds__(256) sum_kernel(Sums q, const T* values, float* parts, T* out) {
  __shared__ uint32_t empty[kZeroRows];
  if (blockIdx.x < q.piece_groups + q.window_groups) {
    const bool pieces = blockIdx.x < q.piece_groups;
    const uint32_t group = pieces ? blockIdx.x : blockIdx.x - q.piece_groups;
    uint32_t slot = threadIdx.x / q.lanes;
    if (WIDE) slot = broadcast(slot, 0);
    const uint32_t vector = group % q.chunks * q.lanes + threadIdx.x % q.lanes;
    const bool mine = vector * Vec<T>::kCount < q.width;
    if (slot >= q.rows_per_group || (!WIDE && !mine)) return;
    const uint32_t number = group / q.chunks * q.rows_per_group + slot;
    if (pieces) {
      if (number < q.pieces) sum_piece<T, NUMBERED, WIDE>(q, values, parts, number, vector, mine);
    } else if (static_cast<uint64_t>(number) * kWindow < q.tokens) {
      if (WIDE) sum_window_wide<T, PASSING>(q, values, out, number, vector, mine);
      else sum_window<T, PASSING>(q, values, out, number, vector);
    }
    return;
  }
  // rows that no token has; not of numbered runs, which have none
  const uint64_t first = static_cast<uint64_t>(blockIdx.x - q.piece_groups - q.window_groups) * kZeroRows;
  for (uint32_t k = threadIdx.x; k < kZeroRows; k += 256) {
    const uint64_t r = first + k;
    // begin[r] holds anything if no token has row r: a run of r begins there only if the sorted ids say so
    bool begins = false;
    if (r < q.rows) {
      const uint32_t b = q.by.begin[r];
      begins = b < q.tokens && q.by.row_of[b] == r && (b == 0 || q.by.row_of[b - 1] != r);
    }
    empty[k] = r < q.rows && !begins;
  }
  __syncthreads();
  const uint32_t vectors = (q.width + Vec<T>::kCount - 1) / Vec<T>::kCount;
  const float zero[Vec<T>::kCount] = {};
  // whole waves go along a row
  const uint32_t per_row = vectors < 64 ? vectors : (vectors + 63) / 64 * 64;
  for (uint32_t at = threadIdx.x; at < kZeroRows * static_cast<uint64_t>(per_row); at += 256) {
    const uint32_t k = at / per_row, vector = at % per_row;
    if (vector < vectors && empty[k]) put<T, PASSING>(out + (first + k) * q.width, zero, 1.f, vector, q.width);
  }
}

// Long runs: the parts of the run that begins in piece j, in order.
template <typename T, bool NUMBERED>
__global__ void __launch_bounds__(256) join_kernel(Sums q, const float* parts, T* out) {
  constexpr int N = Vec<T>::kCount;
  const uint32_t slot = threadIdx.x / q.lanes, vector = blockIdx.x % q.chunks * q.lanes + threadIdx.x % q.lanes;
  const uint32_t piece = blockIdx.x / q.chunks * q.rows_per_group + slot;
  if (slot >= q.rows_per_group || vector * N >= q.width || piece >= q.pieces) return;
  const uint32_t column = Access<T>::column(vector, q.width);
  const uint64_t first = static_cast<uint64_t>(piece) * q.piece;
  const uint32_t run = q.by.row_of[q.tokens - first < q.piece ? q.tokens - 1 : static_cast<uint32_t>(first) + q.piece - 1];
  if (run >= q.rows) return;
  const uint32_t b = q.by.begin[run], e = NUMBERED ? q.by.begin[run + 1] : q.by.end[run];
  if (e - b <= q.piece || b < first) return;
  float acc[N] = {};
  auto part = [&](uint32_t j) { return parts + (static_cast<uint64_t>(j) * 2 + (b > static_cast<uint64_t>(j) * q.piece ? 1 : 0)) * q.parts_stride + column; };
  const uint32_t end = (e - 1) / q.piece + 1;
  uint32_t j = piece;
  for (; j + 8 <= end; j += 8) {
    float v[8][N];
    for (int k = 0; k < 8; k++)
      for (int n = 0; n < N; n++) v[k][n] = part(j + k)[n];
    for (int k = 0; k < 8; k++)
      for (int n = 0; n < N; n++) acc[n] += v[k][n];
  }
  for (; j < end; j++)
    for (int n = 0; n < N; n++) acc[n] += part(j)[n];
  put<T, false>(out + static_cast<uint64_t>(run) * q.width, acc, q.scale, vector, q.width);
}

// ---- host side --------------------------------------------------------------------

// The pieces of a workspace, each on a 256-byte boundary.
struct Layout {
  size_t keys[2], order[2], counts, row_of, begin, end, parts, bytes;
  uint32_t tile_length, tiles, piece, pieces;
  size_t parts_stride;
};

// A long run costs the additions of a part in a row, then one for each part: the longest are balanced at the square root.
uint32_t piece_for(size_t tokens) {
  uint32_t w = 64;
  while (static_cast<size_t>(w) * w * 4 < tokens) w *= 2;
  return w;
}

Layout layout_for(size_t tokens, size_t rows, size_t width, bool numbered) {
  Layout l = {};
  size_t at = 0;
  auto take = [&at](size_t bytes) {
    const size_t here = at;
    at += round_up(bytes, 256);
    return here;
  };
  l.piece = piece_for(tokens);
  l.pieces = tokens > l.piece ? static_cast<uint32_t>((tokens + l.piece - 1) / l.piece) : 0;  // else no run is longer
  l.tile_length = kTile;
  if (tokens > static_cast<size_t>(kTile) * kMostTiles)
    l.tile_length = static_cast<uint32_t>(round_up((tokens + kMostTiles - 1) / kMostTiles, kTile));
  l.tiles = static_cast<uint32_t>((tokens + l.tile_length - 1) / l.tile_length);
  const bool one = tokens <= (numbered ? kOneGroupNumbered : kOneGroup);
  for (int k = 0; k < 2; k++) {
    l.keys[k] = take(one ? (k ? 0 : tokens * 4) : tokens * 4);
    l.order[k] = take(one ? (k ? 0 : tokens * 4) : tokens * 4);
  }
  l.counts = take(one ? 0 : static_cast<size_t>(kBins) * l.tiles * 4);
  l.row_of = numbered && !one ? take(tokens * 4) : l.keys[0];
  const size_t runs = numbered ? (tokens < rows ? tokens : rows) + 1 : rows;
  l.begin = take(runs * 4);
  l.end = numbered ? l.begin : take(runs * 4);
  l.parts_stride = round_up(width, 64);
  l.parts = take(static_cast<size_t>(l.pieces) * 2 * l.parts_stride * 4);
  l.bytes = at ? at : 256;
  return l;
}

// Sorts the tokens and finds their runs, by number (sum_slices) or by key: see Sorted.
Sorted sort_tokens(const Layout& l, char* ws, const void* ids, int id_type, uint32_t tokens, uint32_t rows, bool numbered,
                   void* out_ids, int64_t* out_count, hipStream_t stream) {
  auto at = [ws](size_t offset) { return reinterpret_cast<uint32_t*>(ws + offset); };
  const Digits d = digits_for(rows);
  Sorted to = {at(l.order[0]), at(l.row_of), at(l.begin), at(l.end)};
  if (tokens <= (numbered ? kOneGroupNumbered : kOneGroup)) {
    auto sort = [&](auto keys) {
      hipLaunchKernelGGL((sort_one_kernel<decltype(keys)::value>), dim3(1), dim3(kSortThreads), 0, stream, ids, id_type,
                         tokens, rows, d.bits, d.passes, to, numbered ? 1 : 0, out_ids, out_count);
    };
    if (tokens <= kSortThreads) sort(std::integral_constant<int, 1>());
    else if (tokens <= 2 * kSortThreads) sort(std::integral_constant<int, 2>());
    else if (tokens <= 4 * kSortThreads) sort(std::integral_constant<int, 4>());
    else if (tokens <= 8 * kSortThreads) sort(std::integral_constant<int, 8>());
    else sort(std::integral_constant<int, 12>());
    return to;
  }
  const uint32_t* keys = nullptr;
  const uint32_t* order = nullptr;
  // the last pass ends in buffer 0
  for (int pass = 0; pass < d.passes; pass++) {
    const int into = (d.passes - 1 - pass) & 1;
    hipLaunchKernelGGL(count_kernel, dim3(l.tiles), dim3(kSortThreads), 0, stream, ids, id_type, keys, tokens, rows,
                       l.tile_length, pass * d.bits, d.bits, at(l.counts));
    hipLaunchKernelGGL(scatter_kernel, dim3(l.tiles), dim3(kSortThreads), 0, stream, ids, id_type, keys, order, tokens,
                       rows, l.tile_length, pass * d.bits, d.bits, static_cast<const uint32_t*>(at(l.counts)),
                       at(l.keys[into]), at(l.order[into]));
    keys = at(l.keys[into]);
    order = at(l.order[into]);
  }
  if (!numbered) {
    hipLaunchKernelGGL(runs_kernel, dim3((tokens + kSortThreads - 1) / kSortThreads), dim3(kSortThreads), 0, stream, keys,
                       tokens, rows, to);
  } else {
    hipLaunchKernelGGL(count_runs_kernel, dim3(l.tiles), dim3(kSortThreads), 0, stream, keys, tokens, rows, l.tile_length,
                       at(l.counts));
    hipLaunchKernelGGL(number_runs_kernel, dim3(l.tiles), dim3(kSortThreads), 0, stream, keys, tokens, rows,
                       l.tile_length, static_cast<const uint32_t*>(at(l.counts)), to, id_type, out_ids, out_count);
  }
  return to;
}

template <typename T, bool NUMBERED>
void sum_rows(const Layout& l, char* ws, const Sorted& by, const void* values, uint64_t stride, uint32_t tokens,
              uint32_t rows, uint32_t width, float scale, void* out, hipStream_t stream) {
  const RowShape s = row_shape((width + Vec<T>::kCount - 1) / Vec<T>::kCount);
  float* parts = reinterpret_cast<float*>(ws + l.parts);
  auto groups = [&](uint64_t number) { return static_cast<uint32_t>((number + s.rows_per_group - 1) / s.rows_per_group * s.chunks); };
  Sums q = {stride, l.parts_stride, tokens, rows, width, scale, by, l.piece, l.pieces, s.lanes, s.rows_per_group, s.chunks, 0, 0};
  q.piece_groups = groups(l.pieces);
  q.window_groups = groups((tokens + kWindow - 1) / kWindow);
  const uint32_t clearing = NUMBERED ? 0 : (rows + kZeroRows - 1) / kZeroRows;
  const dim3 grid(q.piece_groups + q.window_groups + clearing);
  const T* from = static_cast<const T*>(values);
  const bool passing = leaves_caches(NUMBERED && tokens < rows ? tokens : rows, width, sizeof(T));
  auto go = [&](auto wide, auto pass) {
    hipLaunchKernelGGL((sum_kernel<T, NUMBERED, decltype(wide)::value, decltype(pass)::value>), grid, dim3(256), 0, stream, q, from,
                       parts, static_cast<T*>(out));
  };
  if (s.lanes % 64) passing ? go(std::false_type(), std::true_type()) : go(std::false_type(), std::false_type());
  else passing ? go(std::true_type(), std::true_type()) : go(std::true_type(), std::false_type());
  if (l.pieces)
    hipLaunchKernelGGL((join_kernel<T, NUMBERED>), dim3(q.piece_groups), dim3(256), 0, stream, q,
                       static_cast<const float*>(parts), static_cast<T*>(out));
}

__global__ void zero_kernel(uint32_t* to, uint64_t words, uint16_t* tail, int has_tail) {
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * blockDim.x;
  const uint64_t first = static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  for (uint64_t i = first; i < words; i += step) to[i] = 0;
  if (has_tail && first == 0) *tail = 0;
}

// Whether the largest launch of sum_rows stays under the 2^32 lanes of one (a lookup looks for itself).
bool fits_launch(size_t tokens, size_t rows, size_t width, int dtype) {
  const RowShape s = row_shape((width * dtype_size(dtype) + 15) / 16);
  const uint64_t windows = (tokens + kWindow - 1) / kWindow, pieces = tokens / piece_for(tokens) + 1;
  const uint64_t groups = (pieces / s.rows_per_group + windows / s.rows_per_group + 2) * s.chunks + rows / kZeroRows + 1;
  return groups * 256 < uint64_t(1) << 32;
}

// A row's column ranges are grid y: 65535 of 256 lanes.
constexpr size_t kMostWidth = static_cast<size_t>(65535) * 256 * 4;

int check(const void* ids, int id_type, size_t tokens, const void* values, int dtype, size_t rows, size_t width,
          size_t stride) {
  if (id_type != STEP_I32 && id_type != STEP_I64) return STEP_ERR_DTYPE;
  if (!is_float(dtype)) return STEP_ERR_DTYPE;
  if (tokens > kMostSize || rows > kMostSize || width > kMostSize) return STEP_ERR_LIMIT;
  if (tokens && !ids) return STEP_ERR_ARGUMENT;
  if (width > kMostWidth) return STEP_ERR_LIMIT;
  if (stride < width) return STEP_ERR_ARGUMENT;
  if (!values && width && tokens) return STEP_ERR_ARGUMENT;
  return STEP_OK;
}

}  // namespace

int hip_fail(hipError_t e) {
  g_last_hip_error = static_cast<int>(e);
  return STEP_ERR_HIP;
}

}  // namespace step

using namespace step;

extern "C" {

int step_abi_version(void) { return STEP_ABI_VERSION; }

const char* step_status_string(int status) {
  switch (status) {
    case STEP_OK: return "ok";
    case STEP_ERR_DTYPE: return "Invalid tensor type passed.";
    case STEP_ERR_ARGUMENT: return "invalid argument";
    case STEP_ERR_HIP: return "HIP runtime call failed";
    case STEP_ERR_LIMIT: return "more than 2^31 - 1 tokens, rows or matrices, 67107840 columns, 2^32 - 1 lanes of a launch, "
                                "or a matrix to orthogonalize of more than 2^20 a side or 2^33 entries";
    default: return "unknown status";
  }
}

int step_last_hip_error(void) { return g_last_hip_error; }

int step_embedding_lookup(const void* ids, int id_type, size_t tokens, const void* weight, int dtype, size_t rows,
                          size_t width, size_t weight_stride, float scale, void* out, void* stream) {
  int rc = check(ids, id_type, tokens, rows ? weight : ids, dtype, rows, width, weight_stride);
  if (rc != STEP_OK) return rc;
  if (tokens == 0 || width == 0) return STEP_OK;
  if (!out) return STEP_ERR_ARGUMENT;
  const RowShape s = row_shape((width * dtype_size(dtype) + 15) / 16);
  const size_t per_group = static_cast<size_t>(s.rows_per_group) * kLookupRows;
  if ((tokens + per_group - 1) / per_group * 256 >= size_t(1) << 32) return STEP_ERR_LIMIT;  // lanes of a launch
  const dim3 grid(static_cast<uint32_t>((tokens + per_group - 1) / per_group), s.chunks);
  auto go = [&](auto type, auto pass) {
    typedef decltype(type) T;
    hipLaunchKernelGGL((lookup_kernel<T, decltype(pass)::value>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), ids, id_type,
                       static_cast<uint32_t>(tokens), static_cast<const T*>(weight), static_cast<uint32_t>(rows),
                       static_cast<uint32_t>(width), static_cast<uint64_t>(weight_stride), scale, static_cast<T*>(out),
                       s.lanes, s.rows_per_group);
  };
  auto by_size = [&](auto type) {
    if (leaves_caches(tokens, width, dtype_size(dtype))) go(type, std::true_type());
    else go(type, std::false_type());
  };
  if (dtype == STEP_F32) by_size(F32());
  else if (dtype == STEP_BF16) by_size(BF16());
  else by_size(F16());
  return launched();
}

size_t step_embedding_piece(size_t tokens) { return piece_for(tokens); }

size_t step_embedding_gradient_workspace(size_t tokens, size_t rows, size_t width) {
  if (tokens > kMostSize || rows > kMostSize || width > kMostSize) return 0;
  return layout_for(tokens, rows, width, false).bytes;
}

int step_embedding_gradient(const void* ids, int id_type, size_t tokens, const void* grad, int dtype, size_t rows,
                            size_t width, size_t grad_stride, float scale, void* out, void* workspace,
                            size_t workspace_bytes, void* stream_) {
  const int rc = check(ids, id_type, tokens, grad, dtype, rows, width, grad_stride);
  if (rc != STEP_OK) return rc;
  if (rows == 0 || width == 0) return STEP_OK;
  if (!out) return STEP_ERR_ARGUMENT;
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (tokens == 0) {
    const uint64_t bytes = static_cast<uint64_t>(rows) * width * dtype_size(dtype), words = bytes / 4;
    const uint64_t groups = (words + 255) / 256;
    hipLaunchKernelGGL(zero_kernel, dim3(static_cast<uint32_t>(groups < 1 ? 1 : groups > 4096 ? 4096 : groups)), dim3(256),
                       0, stream, static_cast<uint32_t*>(out), words,
                       reinterpret_cast<uint16_t*>(static_cast<char*>(out) + words * 4), bytes % 4 ? 1 : 0);
    return launched();
  }
  if (!fits_launch(tokens, rows, width, dtype)) return STEP_ERR_LIMIT;
  const Layout l = layout_for(tokens, rows, width, false);
  if (!workspace || workspace_bytes < l.bytes || reinterpret_cast<uintptr_t>(workspace) % 256) return STEP_ERR_ARGUMENT;
  char* ws = static_cast<char*>(workspace);
  const uint32_t t = static_cast<uint32_t>(tokens), v = static_cast<uint32_t>(rows), w = static_cast<uint32_t>(width);
  const Sorted by = sort_tokens(l, ws, ids, id_type, t, v, false, nullptr, nullptr, stream);
  if (dtype == STEP_F32) sum_rows<F32, false>(l, ws, by, grad, grad_stride, t, v, w, scale, out, stream);
  else if (dtype == STEP_BF16) sum_rows<BF16, false>(l, ws, by, grad, grad_stride, t, v, w, scale, out, stream);
  else sum_rows<F16, false>(l, ws, by, grad, grad_stride, t, v, w, scale, out, stream);
  return launched();
}

size_t step_sum_slices_workspace(size_t tokens, size_t rows, size_t width) {
  if (tokens > kMostSize || rows > kMostSize || width > kMostSize) return 0;
  return layout_for(tokens, rows, width, true).bytes;
}

int step_sum_slices(const void* ids, int id_type, size_t tokens, const void* values, int dtype, size_t rows, size_t width,
                    size_t values_stride, float scale, void* out_ids, void* out_values, int64_t* out_count,
                    void* workspace, size_t workspace_bytes, void* stream_) {
  const int rc = check(ids, id_type, tokens, values, dtype, rows, width, values_stride);
  if (rc != STEP_OK) return rc;
  if (!out_count) return STEP_ERR_ARGUMENT;
  hipStream_t stream = static_cast<hipStream_t>(stream_);
  if (tokens == 0 || rows == 0) {
    hipLaunchKernelGGL(zero_kernel, dim3(1), dim3(256), 0, stream, reinterpret_cast<uint32_t*>(out_count),
                       static_cast<uint64_t>(2), static_cast<uint16_t*>(nullptr), 0);
    return launched();
  }
  if (!out_ids || (width && !out_values)) return STEP_ERR_ARGUMENT;
  if (width && !fits_launch(tokens, 0, width, dtype)) return STEP_ERR_LIMIT;
  const Layout l = layout_for(tokens, rows, width, true);
  if (!workspace || workspace_bytes < l.bytes || reinterpret_cast<uintptr_t>(workspace) % 256) return STEP_ERR_ARGUMENT;
  char* ws = static_cast<char*>(workspace);
  const uint32_t t = static_cast<uint32_t>(tokens), v = static_cast<uint32_t>(rows), w = static_cast<uint32_t>(width);
  const Sorted by = sort_tokens(l, ws, ids, id_type, t, v, true, out_ids, out_count, stream);
  if (width == 0) return launched();
  if (dtype == STEP_F32) sum_rows<F32, true>(l, ws, by, values, values_stride, t, v, w, scale, out_values, stream);
  else if (dtype == STEP_BF16) sum_rows<BF16, true>(l, ws, by, values, values_stride, t, v, w, scale, out_values, stream);
  else sum_rows<F16, true>(l, ws, by, values, values_stride, t, v, w, scale, out_values, stream);
  return launched();
}

}  // extern "C"
