// What the kernels of the experts' products share (expert.hip, packed.hip): an expert's rows and
// their tiles, the order of tiles, parts of a contraction and their sum, launches.
#pragma once

#include <algorithm>
#include <type_traits>

#include "expert16.hpp"
#include "train.hpp"

namespace purin {
namespace train {

// The rows of expert e: [from, to), inside [0, rows] whatever the offsets hold.
__device__ __forceinline__ void segment(const int32_t* offsets, int e, int64_t rows, int64_t& from,
                                        int64_t& to) {
  from = e ? min((int64_t)max(offsets[e], 0), rows) : 0;
  to = min((int64_t)max(offsets[e + 1], 0), rows);
  to = max(to, from);
}

// The expert and the first row of tile number ``tile`` where every expert's rows are cut into
// tiles of ``height``; beyond the experts' tiles come those of the rows behind the last expert
// (expert -1: zeros).  False where the tile is past them all.  Every wavefront finds it by
// itself, 64 experts at a time.
__device__ __forceinline__ bool find_tile(const int32_t* offsets, int experts, int64_t rows,
                                          int height, int64_t tile, int& expert, int64_t& from,
                                          int64_t& to) {
  const int lane = threadIdx.x & 63;
  for (int e0 = 0; e0 < experts; e0 += 64) {
    const int e = e0 + lane;
    int64_t a = 0, z = 0;
    if (e < experts) segment(offsets, e, rows, a, z);
    int32_t n = (int32_t)((z - a + height - 1) / height);
    int32_t sum = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int32_t up = __shfl_up(sum, d, 64);
      if (lane >= d) sum += up;
    }
    const uint64_t here = __ballot(tile < sum);
    if (here) {
      const int at = __ffsll((unsigned long long)here) - 1;
      const int32_t first = __shfl(sum - n, at, 64);
      expert = e0 + at;
      segment(offsets, expert, rows, from, to);
      from += (tile - first) * height;
      return true;
    }
    tile -= __shfl(sum, 63, 64);
  }
  int64_t unused;
  segment(offsets, experts - 1, rows, unused, from);
  expert = -1;
  to = rows;
  from += tile * height;
  return from < to;
}

// Zeros for the rows behind the last expert's.
template <typename T>
__device__ __forceinline__ void zero_tile(T* c, int64_t ldc, int m, int n) {
  const int per = (n + kVec<T> - 1) / kVec<T>;
  for (int r = threadIdx.x; r < m * per; r += blockDim.x) {
    const int i = r / per, j = r % per * kVec<T>;
    store_upto(c + i * ldc + j, zeros16<T>(), n - j);
  }
}

// Tiles in 1-D order, XCD by XCD (workgroups are dealt to the 8 XCDs in
// turn, so number i is on XCD i % 8): an XCD's workgroups take neighbouring tiles, kGroup rows
// of tiles at a time, and find each other's operands in its L2.  The tiles shared out are those
// launched: where many rows have no expert, the last XCDs' share is tiles without work.
constexpr int kGroup = 4;
__device__ __forceinline__ void tile_order(int64_t tiles_m, int64_t tiles_n, int64_t& tm,
                                           int64_t& tn) {
  const int64_t n = tiles_m * tiles_n, per = (n + 7) / 8, id = blockIdx.x;
  int64_t at = (id & 7) * per + (id >> 3);
  const int64_t whole = n - (per - 1) * 8;  // XCDs that have per tiles, the others one fewer
  if ((id & 7) > whole) at -= (id & 7) - whole;
  const int64_t group = at / (kGroup * tiles_n), first = group * kGroup;
  const int64_t high = min<int64_t>(kGroup, tiles_m - first), in = at - first * tiles_n;
  tm = first + in % high;
  tn = in / high;
}

// The part of a contraction of ``depth`` that split number ``split`` of ``splits`` has: whole
// stages of kDepth16, the last one's end apart.
__device__ __forceinline__ void part_of(int64_t depth, int split, int splits, int64_t& first,
                                        int64_t& length) {
  const int64_t steps = (depth + kDepth16 - 1) / kDepth16, per = (steps + splits - 1) / splits;
  first = min(depth, split * per * kDepth16);
  length = min(depth - first, per * kDepth16);
}

// out = the sum of ``splits`` parts, in their order.
template <typename T>
static __global__ __launch_bounds__(256) void k_join(const float* __restrict__ parts, int splits,
                                              int64_t count, T* __restrict__ out) {
  constexpr int V = 4;
  typedef float F __attribute__((ext_vector_type(V), aligned(4)));
  const int64_t step = (int64_t)gridDim.x * 256 * V;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V; i < count; i += step) {
    if (i + V <= count) {
      F sum = *reinterpret_cast<const F*>(parts + i);
      for (int s = 1; s < splits; ++s) sum += *reinterpret_cast<const F*>(parts + s * count + i);
      typedef T O __attribute__((ext_vector_type(V), aligned(sizeof(T))));
      O v;
#pragma unroll
      for (int q = 0; q < V; ++q) v[q] = (T)sum[q];
      *reinterpret_cast<O*>(out + i) = v;
    } else {
      for (int64_t j = i; j < count; ++j) {
        float sum = parts[j];
        for (int s = 1; s < splits; ++s) sum += parts[s * count + j];
        out[j] = (T)sum;
      }
    }
  }
}

// A launch holds fewer than 2^32 threads: more tiles than that do not fit the card's memory.
static int check_grid(int64_t tiles, int threads) {
  if (tiles * threads < (int64_t(1) << 32)) return PURIN_CP_OK;
  return set_error(PURIN_CP_ERR_UNSUPPORTED, "too many tiles for a launch");
}

template <typename K, typename... A>
static int launch16(const char* name, K kernel, int64_t tiles, unsigned gy, unsigned gz,
                    int threads, int lds, hipStream_t st, A... args) {
  if (int rc = check_grid(tiles, threads)) return rc;
  const dim3 grid((unsigned)tiles, gy, gz);
  if (int rc = raise_lds_cap((const void*)kernel, (size_t)lds)) return rc;
  kernel<<<grid, dim3((unsigned)threads), (size_t)lds, st>>>(args...);
  return launched(name);
}

// Whether 16-byte pieces of rows ``ld`` elements apart lie at 16-byte addresses, all of a row's
// length, and the rows of one stage (at most 256) are within 31 bits of its first.
static bool direct_ok(const void* p, int64_t ld, int64_t length) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0 && length % 8 == 0 &&
         ld < (int64_t(1) << 21);
}

using std::integral_constant;
constexpr integral_constant<int, 1> i1;
constexpr integral_constant<int, 2> i2;
constexpr integral_constant<int, 4> i4;
constexpr integral_constant<int, 16> i16;
constexpr integral_constant<int, 32> i32;
constexpr integral_constant<int, 64> i64;
constexpr integral_constant<int, 128> i128;
constexpr integral_constant<int, 256> i256;

// The most tiles of ``height`` rows that any split of the rows over the experts needs, the rows
// behind the last expert among them.
static int64_t most_tiles(int64_t rows, int64_t experts, int64_t height) {
  return (rows + std::min(rows, experts + 1) * (height - 1)) / height;
}

static int64_t steps16(int64_t depth) { return (depth + kDepth16 - 1) / kDepth16; }
// Splits of at least ``part`` stages, ``groups`` workgroups each, up to ``room`` workgroups.
static int splits_of(int64_t room, int64_t groups, int64_t steps, int64_t part) {
  return (int)std::max<int64_t>(1, std::min(room / std::max<int64_t>(groups, 1), steps / part));
}
// The ``splits`` parts of ``count`` sums added up into out.
template <typename T>
static int join(hipStream_t st, const float* parts, int splits, int64_t count, T* out) {
  k_join<T><<<grid_of(count, 1024), dim3(256), 0, st>>>(parts, splits, count, out);
  return launched("k_join");
}

// Whether a weight is read along inner (a length of one has any stride); along outer otherwise.
static bool along_inner(int64_t inner, int64_t wi, int64_t wo) {
  return wo != 1 && (wi == 1 || inner <= 1);
}

// 32-bit sums of the parts, where a product is split.
static int64_t parts_bytes(int splits, int64_t count) {
  return splits > 1 ? splits * count * (int64_t)sizeof(float) : 0;
}

static int check_product(int32_t dtype, int64_t rows, int64_t inner, int64_t outer,
                         int64_t experts) {
  if (!known_dtype(dtype)) return refuse("unknown dtype");
  if (rows < 0 || inner < 0 || outer < 0 || experts < 1)
    return refuse("sizes must not be negative, experts must be positive");
  if (experts > PURIN_TRAIN_MAX_EXPERTS)
    return set_error(PURIN_CP_ERR_UNSUPPORTED, "more than 1024 experts");
  if (rows >= (int64_t(1) << 31))
    return set_error(PURIN_CP_ERR_UNSUPPORTED, "rows must stay below 2^31");
  // so that 64 bits hold the sizes' products
  if (inner > (int64_t(1) << 22) || outer > (int64_t(1) << 22))
    return set_error(PURIN_CP_ERR_UNSUPPORTED, "inner and outer must not exceed 2^22");
  return PURIN_CP_OK;
}

}  // namespace train
}  // namespace purin
