// The experts' products on rows sorted by expert, and the gradient of their weights
// (include/purin_train.h: expert_product, expert_weights_vjp).
//
//   out(p) = a(p) W[e]                     for the rows p of expert e
//   g_W[e] = sum over those p of a(p)^T g(p)
//
// Products of tiles on the matrix units; a tile belongs to one expert.  The tiles of out are found
// from the offsets on the device, so the host never waits for the counts: the launch holds the
// most tiles that any split of the rows can need, and what is left over ends at once.  The same
// goes for the cuts below, which count rows that no expert has.

#include <algorithm>
#include <type_traits>

#include "expert16.hpp"
#include "expert32.hpp"
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

template <typename T, int BM, int BN, int WM, int WN, bool ALONG_B, bool DIRECT, int S>
__global__ __launch_bounds__(WM* WN * 64) void k_product16(
    const T* __restrict__ a, int64_t lda, const T* __restrict__ w, int64_t we, int64_t ldw,
    int64_t rows, int64_t inner, int64_t outer, int experts, int64_t tiles_m, int64_t tiles_n,
    const int32_t* __restrict__ offsets, T* __restrict__ out, int64_t ldo) {
  extern __shared__ __align__(16) unsigned char lds16[];
  int64_t tm, tn;
  tile_order(tiles_m, tiles_n, tm, tn);
  int e;
  int64_t from, to;
  if (!find_tile(offsets, experts, rows, BM, tm, e, from, to)) return;
  e = __builtin_amdgcn_readfirstlane(e);
  const int64_t col = tn * BN;
  const int m = __builtin_amdgcn_readfirstlane((int)min<int64_t>(BM, to - from));
  const int n = (int)min<int64_t>(BN, outer - col);
  T* c = out + from * ldo + col;
  if (e < 0) {
    zero_tile(c, ldo, m, n);
    return;
  }
  tile16<T, T, BM, BN, WM, WN, true, ALONG_B, DIRECT, S>(
      {a + from * lda, lda, m}, {w + e * we + (ALONG_B ? col * ldw : col), ldw, n, col > 0}, inner,
      lds16, c, ldo);
}

// out = the sum of ``splits`` parts, in their order.
template <typename T>
__global__ __launch_bounds__(256) void k_join(const float* __restrict__ parts, int splits,
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

// Experts with few rows, or few tiles in all: column tiles of 64 for BM rows at a time.  Split
// number blockIdx.y of the contraction writes its own ``out``.
template <typename T, typename C, int BM, int BN, bool ALONG_B, bool DIRECT>
__global__ __launch_bounds__(256) void k_product_thin(
    const T* __restrict__ a, int64_t lda, const T* __restrict__ w, int64_t we, int64_t ldw,
    int64_t rows, int64_t inner, int64_t outer, int experts, int64_t tiles_n,
    const int32_t* __restrict__ offsets, C* __restrict__ out, int64_t ldo) {
  extern __shared__ __align__(16) unsigned char lds16[];
  const int64_t tm = blockIdx.x / tiles_n, tn = blockIdx.x - tm * tiles_n;
  int e;
  int64_t from, to;
  if (!find_tile(offsets, experts, rows, BM, tm, e, from, to)) return;
  e = __builtin_amdgcn_readfirstlane(e);
  const int64_t col = tn * BN;
  const int m = __builtin_amdgcn_readfirstlane((int)min<int64_t>(BM, to - from));
  const int n = (int)min<int64_t>(BN, outer - col);
  C* c = out + (int64_t)blockIdx.y * rows * ldo + from * ldo + col;
  if (e < 0) {
    zero_tile(c, ldo, m, n);
    return;
  }
  int64_t k, length;
  part_of(inner, (int)blockIdx.y, (int)gridDim.y, k, length);
  thin16<T, C, BM, BN, ALONG_B, DIRECT>(
      {a + from * lda + k, lda, m},
      {w + e * we + (ALONG_B ? col * ldw + k : col + k * ldw), ldw, n, col > 0}, length, lds16, c,
      ldo);
}

// Split number blockIdx.z of an expert's rows writes its own ``gw`` (experts x inner x outer).
template <typename T, typename C, int BM, int BN, int WM, int WN, bool DIRECT, int S>
__global__ __launch_bounds__(WM* WN * 64) void k_weights_vjp16(
    const T* __restrict__ a, int64_t lda, const T* __restrict__ g, int64_t ldg, int64_t rows,
    int64_t inner, int64_t outer, int64_t tiles_m, int64_t tiles_n,
    const int32_t* __restrict__ offsets, C* __restrict__ gw) {
  extern __shared__ __align__(16) unsigned char lds16[];
  int64_t tm, tn;
  tile_order(tiles_m, tiles_n, tm, tn);
  const int e = (int)blockIdx.y;
  int64_t from, to, k, length;
  segment(offsets, e, rows, from, to);
  part_of(to - from, (int)blockIdx.z, (int)gridDim.z, k, length);
  from += k;
  const int64_t i = tm * BM, j = tn * BN;
  tile16<T, C, BM, BN, WM, WN, false, false, DIRECT, S>(
      {a + from * lda + i, lda, (int)min<int64_t>(BM, inner - i), i > 0},
      {g + from * ldg + j, ldg, (int)min<int64_t>(BN, outer - j), j > 0}, length, lds16,
      gw + ((int64_t)blockIdx.z * gridDim.y + e) * inner * outer + i * outer + j, outer);
}

// 32- and 64-bit types.  Split number blockIdx.y of the contraction writes its own ``out``.
template <typename T, int BM, int BN, int WM, int WN, bool ALONG_B>
__global__ __launch_bounds__(256, 2) void k_product32(
    const T* __restrict__ a, int64_t lda, const T* __restrict__ w, int64_t we, int64_t ldw,
    int64_t rows, int64_t inner, int64_t outer, int experts, int64_t tiles_m, int64_t tiles_n,
    const int32_t* __restrict__ offsets, T* __restrict__ out, int64_t ldo) {
  __shared__ __align__(16) unsigned char lds[lds32<T, BM, BN, true, ALONG_B>()];
  int64_t tm, tn;
  tile_order(tiles_m, tiles_n, tm, tn);
  int e;
  int64_t from, to;
  if (!find_tile(offsets, experts, rows, BM, tm, e, from, to)) return;
  e = __builtin_amdgcn_readfirstlane(e);
  const int64_t col = tn * BN;
  const int m = __builtin_amdgcn_readfirstlane((int)min<int64_t>(BM, to - from));
  const int n = (int)min<int64_t>(BN, outer - col);
  T* c = out + (int64_t)blockIdx.y * rows * ldo + from * ldo + col;
  if (e < 0) {
    zero_tile(c, ldo, m, n);
    return;
  }
  int64_t k, length;
  part_of(inner, (int)blockIdx.y, (int)gridDim.y, k, length);
  tile32<T, BM, BN, WM, WN, true, ALONG_B, 3>(
      {a + from * lda + k, lda, m},
      {w + e * we + (ALONG_B ? col * ldw + k : col + k * ldw), ldw, n, col > 0}, length, (T*)lds, c,
      ldo);
}

// Split number blockIdx.z of an expert's rows writes its own ``gw``.
template <typename T, int BM, int BN>
__global__ __launch_bounds__(256, 2) void k_weights_vjp32(
    const T* __restrict__ a, int64_t lda, const T* __restrict__ g, int64_t ldg, int64_t rows,
    int64_t inner, int64_t outer, int64_t tiles_m, int64_t tiles_n,
    const int32_t* __restrict__ offsets, T* __restrict__ gw) {
  __shared__ __align__(16) unsigned char lds[lds32<T, BM, BN, false, false>()];
  int64_t tm, tn;
  tile_order(tiles_m, tiles_n, tm, tn);
  const int e = (int)blockIdx.y;
  int64_t from, to, k, length;
  segment(offsets, e, rows, from, to);
  part_of(to - from, (int)blockIdx.z, (int)gridDim.z, k, length);
  from += k;
  const int64_t i = tm * BM, j = tn * BN;
  tile32<T, BM, BN, 2, 2, false, false, BM == 128 ? 1 : 3>(
      {a + from * lda + i, lda, (int)min<int64_t>(BM, inner - i), i > 0},
      {g + from * ldg + j, ldg, (int)min<int64_t>(BN, outer - j), j > 0}, length, (T*)lds,
      gw + ((int64_t)blockIdx.z * gridDim.y + e) * inner * outer + i * outer + j, outer);
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
constexpr integral_constant<int, 32> i32;
constexpr integral_constant<int, 64> i64;
constexpr integral_constant<int, 128> i128;
constexpr integral_constant<int, 256> i256;

// The most tiles of ``height`` rows that any split of the rows over the experts needs, the rows
// behind the last expert among them.
static int64_t most_tiles(int64_t rows, int64_t experts, int64_t height) {
  return (rows + std::min(rows, experts + 1) * (height - 1)) / height;
}

// How the 16-bit kernels cut a product.  ``tiles``: the 128 x 128 tiles, ``steps``: the stages of
// the contraction.  us of 1000 rows, 8 experts, 1024 x 1024 | 3000, 60, 2048 x 512 | 2048, 2,
// 2048 x 2048 | 32768, 16, 2048 x 4096, bf16:
//   thin    32 x 64 tiles: the experts' weights at the rate of memory where rows are few, and
//           eight times the workgroups where tiles are few       9.5 |  41 |   - |   -
//           64 x 64 ones from 16 rows to an expert on, where they fill the CUs: a second tile of
//           an expert reads its weights again (768 rows, 32 experts of unequal shares,
//           4096 x 1536: 99 us with 32, 87 with 64; 512 rows, 64 experts, 1024 x 1024: 30, 32)
//   deep    up to one 128 x 128 tile a CU there is room for 4 stages, three on their way: the
//           stages' latency is what counts then                 15.5 |   - |   - |   -
//   128     two workgroups a CU of 2 stages                        - |  32 |  34 | 660
//   256     half the LDS reads and operand traffic of 128; from 4 tiles to a CU on its single
//           workgroup a CU does not leave CUs idle at the end      - |   - |  57 | 600
// Where even so CUs are idle and the contraction is long, it is split into parts of 32-bit
// sums, which a second kernel adds up.
enum Shape16 { kThin16, kDeep16, k128, k256 };
struct Cut16 {
  Shape16 shape;
  int height, splits;
};
static int64_t steps16(int64_t depth) { return (depth + kDepth16 - 1) / kDepth16; }
// Splits of at least ``part`` stages, ``groups`` workgroups each, up to ``room`` workgroups.
static int splits_of(int64_t room, int64_t groups, int64_t steps, int64_t part) {
  return (int)std::max<int64_t>(1, std::min(room / std::max<int64_t>(groups, 1), steps / part));
}
static Cut16 cut_product16(int64_t rows, int64_t inner, int64_t outer, int64_t experts) {
  const int64_t tiles = most_tiles(rows, experts, 128) * ((outer + 127) / 128);
  if (rows <= 32 * experts || tiles <= 128) {
    const int64_t across = (outer + 63) / 64;
    const bool tall = rows > 16 * experts && most_tiles(rows, experts, 64) * across >= 256;
    if (tall) return {kThin16, 64, 1};
    return {kThin16, 32, splits_of(256, most_tiles(rows, experts, 32) * across, steps16(inner), 16)};
  }
  if (tiles >= 16 * 256) return {k256, 256, 1};
  return {tiles <= 256 ? kDeep16 : k128, 128, 1};
}
static Cut16 cut_weights16(int64_t rows, int64_t inner, int64_t outer, int64_t experts) {
  const int64_t tiles = ((inner + 127) / 128) * ((outer + 127) / 128) * experts;
  const int splits = splits_of(256, tiles, steps16(rows / experts), 12);
  if (tiles >= 16 * 256) return {k256, 256, 1};
  return {tiles * splits <= 256 ? kDeep16 : k128, 128, splits};
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

template <typename T>
static int product16(hipStream_t st, int64_t rows, int64_t inner, int64_t outer, int64_t experts,
                     const T* a, int64_t lda, const T* w, int64_t we, int64_t wi, int64_t wo,
                     const int32_t* offsets, void* ws, T* out, int64_t ldo) {
  const bool along = along_inner(inner, wi, wo);
  const int64_t ldw = along ? wo : wi;
  const bool direct = direct_ok(a, lda, inner) && direct_ok(w, ldw, along ? inner : outer) &&
                      we % 8 == 0;
  Cut16 cut = cut_product16(rows, inner, outer, experts);
  if (ldo != outer) cut.splits = 1;  // the parts are added up as one row
  if (cut.shape == kThin16) {
    constexpr int TN = 64;
    const int64_t tm = most_tiles(rows, experts, cut.height), tn = (outer + TN - 1) / TN;
    auto thin = [&](auto c, auto h) {
      using C = decltype(c);
      constexpr int TM = h;
      auto kernel = along ? (direct ? k_product_thin<T, C, TM, TN, true, true>
                                    : k_product_thin<T, C, TM, TN, true, false>)
                          : (direct ? k_product_thin<T, C, TM, TN, false, true>
                                    : k_product_thin<T, C, TM, TN, false, false>);
      return launch16("k_product_thin", kernel, tm * tn, (unsigned)cut.splits, 1, 256,
                      thin_lds<TM, TN>(), st, a, lda, w, we, ldw, rows, inner, outer, (int)experts,
                      tn, offsets, cut.splits > 1 ? (C*)ws : (C*)out, ldo);
    };
    if (cut.splits == 1) return cut.height == 32 ? thin(T{}, i32) : thin(T{}, i64);
    if (int rc = thin(float{}, i32)) return rc;
    return join(st, (const float*)ws, cut.splits, rows * outer, out);
  }
  auto go = [&](auto bm, auto wn, auto s) {
    constexpr int B = bm, WN = wn, S = s;
    const int64_t tm = most_tiles(rows, experts, B), tn = (outer + B - 1) / B;
    auto kernel = along ? (direct ? k_product16<T, B, B, 2, WN, true, true, S>
                                  : k_product16<T, B, B, 2, WN, true, false, S>)
                        : (direct ? k_product16<T, B, B, 2, WN, false, true, S>
                                  : k_product16<T, B, B, 2, WN, false, false, S>);
    return launch16("k_product16", kernel, tm * tn, 1, 1, 2 * WN * 64,
                    tile16_lds<T, T, B, B, S>(), st, a, lda, w, we, ldw, rows, inner, outer,
                    (int)experts, tm, tn, offsets, out, ldo);
  };
  if (cut.shape == k256) return go(i256, i4, i2);
  return cut.shape == kDeep16 ? go(i128, i2, i4) : go(i128, i2, i2);
}

template <typename T>
static int weights_vjp16(hipStream_t st, int64_t rows, int64_t inner, int64_t outer,
                         int64_t experts, const T* a, int64_t lda, const T* g, int64_t ldg,
                         const int32_t* offsets, void* ws, T* gw) {
  const bool direct = direct_ok(a, lda, inner) && direct_ok(g, ldg, outer);
  const Cut16 cut = cut_weights16(rows, inner, outer, experts);
  auto go = [&](auto c, auto bm, auto wn, auto s) {
    using C = decltype(c);
    constexpr int B = bm, WN = wn, S = s;
    const int64_t tm = (inner + B - 1) / B, tn = (outer + B - 1) / B;
    auto kernel = direct ? k_weights_vjp16<T, C, B, B, 2, WN, true, S>
                         : k_weights_vjp16<T, C, B, B, 2, WN, false, S>;
    return launch16("k_weights_vjp16", kernel, tm * tn, (unsigned)experts,
                    (unsigned)cut.splits, 2 * WN * 64, tile16_lds<T, C, B, B, S>(), st, a, lda, g, ldg, rows, inner, outer, tm, tn,
                    offsets, cut.splits > 1 ? (C*)ws : (C*)gw);
  };
  if (cut.splits > 1) {
    if (int rc = go(float{}, i128, i2, i4)) return rc;
    return join(st, (const float*)ws, cut.splits, experts * inner * outer, gw);
  }
  if (cut.shape == k256) return go(T{}, i256, i4, i2);
  return cut.shape == kDeep16 ? go(T{}, i128, i2, i4) : go(T{}, i128, i2, i2);
}

// How the 32- and 64-bit kernels cut a product: 32 x 64 tiles where rows, or tiles, are few, else
// 64 x 64, in 32 bits with the contraction split as in 16, but up to four workgroups a CU: what
// one wavefront a SIMD leaves of the matrix units' time between its reads and barriers, others
// use (f32, 700 rows, 4 experts, 4096 x 256: 43 us with one, 31 with four).  128 x 128 tiles read
// half as much, and were 2 % faster at 32768 rows, 16 experts, 2048 x 4096 (4630 us against 4740)
// and slower wherever fewer of them run side by side (16384, 8, 512 x 512: 113 against 101).
struct Cut32 {
  int height, splits;
};
static Cut32 cut_product32(bool wide, int64_t rows, int64_t inner, int64_t outer, int64_t experts) {
  const int64_t across = (outer + 63) / 64;
  const int height = rows <= 32 * experts || most_tiles(rows, experts, 64) * across < 512 ? 32 : 64;
  const int64_t groups = most_tiles(rows, experts, height) * across;
  return {height, wide ? 1 : splits_of(1024, groups, steps16(inner), 4)};
}
// The weights' gradient: both operands are read across their rows, and 128 x 128 tiles are ahead
// from twice the CUs on (8192 rows, 64 experts, 1024 x 1024: 200 us against 213).
static Cut32 cut_weights32(bool wide, int64_t rows, int64_t inner, int64_t outer, int64_t experts) {
  if (!wide && ((inner + 127) / 128) * ((outer + 127) / 128) * experts >= 512) return {128, 1};
  const int64_t groups = ((inner + 63) / 64) * ((outer + 63) / 64) * experts;
  return {64, wide ? 1 : splits_of(1024, groups, steps16(rows / experts), 4)};
}

template <typename T>
static int product32(hipStream_t st, int64_t rows, int64_t inner, int64_t outer, int64_t experts,
                     const T* a, int64_t lda, const T* w, int64_t we, int64_t wi, int64_t wo,
                     const int32_t* offsets, void* ws, T* out, int64_t ldo) {
  const bool along = along_inner(inner, wi, wo);
  const int64_t ldw = along ? wo : wi;
  Cut32 cut = cut_product32(sizeof(T) == 8, rows, inner, outer, experts);
  if (ldo != outer) cut.splits = 1;  // the parts are added up as one row
  auto shape = [&](auto bm, auto wm, auto wn) {
    constexpr int BM = bm, WM = wm, WN = wn;
    const int64_t tm = most_tiles(rows, experts, BM), tn = (outer + 63) / 64;
    if (int e = check_grid(tm * tn, 256)) return e;
    auto kernel = along ? k_product32<T, BM, 64, WM, WN, true> : k_product32<T, BM, 64, WM, WN, false>;
    kernel<<<dim3((unsigned)(tm * tn), (unsigned)cut.splits), dim3(256), 0, st>>>(
        a, lda, w, we, ldw, rows, inner, outer, (int)experts, tm, tn, offsets,
        cut.splits > 1 ? (T*)ws : out, ldo);
    return launched("k_product32");
  };
  const int rc = cut.height == 32 ? shape(i32, i1, i4) : shape(i64, i2, i2);
  if constexpr (sizeof(T) == 4)
    if (!rc && cut.splits > 1) return join(st, (const float*)ws, cut.splits, rows * outer, out);
  return rc;
}

template <typename T>
static int weights_vjp32(hipStream_t st, int64_t rows, int64_t inner, int64_t outer,
                         int64_t experts, const T* a, int64_t lda, const T* g, int64_t ldg,
                         const int32_t* offsets, void* ws, T* gw) {
  const Cut32 cut = cut_weights32(sizeof(T) == 8, rows, inner, outer, experts);
  auto go = [&](int b, auto kernel) {
    const int64_t tm = (inner + b - 1) / b, tn = (outer + b - 1) / b;
    if (int e = check_grid(tm * tn, 256)) return e;
    kernel<<<dim3((unsigned)(tm * tn), (unsigned)experts, (unsigned)cut.splits), dim3(256), 0, st>>>(
        a, lda, g, ldg, rows, inner, outer, tm, tn, offsets, cut.splits > 1 ? (T*)ws : gw);
    return launched("k_weights_vjp32");
  };
  if constexpr (sizeof(T) == 4)
    if (cut.height == 128) return go(128, k_weights_vjp32<T, 128, 128>);
  if (int rc = go(64, k_weights_vjp32<T, 64, 64>)) return rc;
  if constexpr (sizeof(T) == 4)
    if (cut.splits > 1)
      return join(st, (const float*)ws, cut.splits, experts * inner * outer, gw);
  return PURIN_CP_OK;
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

using namespace purin;
using namespace purin::train;

extern "C" {

int64_t purin_train_expert_product_workspace_bytes(int32_t dtype, int64_t rows, int64_t inner,
                                                   int64_t outer, int64_t experts) {
  int64_t need = -1;
  (void)guarded([&] {
    if (int rc = check_product(dtype, rows, inner, outer, experts)) return rc;
    need = 0;
    if (rows && outer)
      need = parts_bytes(dtype_bytes(dtype) == 2
                             ? cut_product16(rows, inner, outer, experts).splits
                             : cut_product32(dtype == PURIN_TRAIN_F64, rows, inner, outer, experts)
                                   .splits,
                         rows * outer);
    return (int)PURIN_CP_OK;
  });
  return need;
}

int purin_train_expert_product(void* stream, int32_t dtype, int64_t rows, int64_t inner,
                               int64_t outer, int64_t experts, const void* a, int64_t lda,
                               const void* weight, int64_t we, int64_t wi, int64_t wo,
                               const int32_t* offsets, void* workspace, int64_t workspace_bytes,
                               void* out, int64_t ldo) {
  return guarded([&] {
    if (int rc = check_product(dtype, rows, inner, outer, experts)) return rc;
    if (!rows || !outer) return (int)PURIN_CP_OK;
    if (!offsets || !out || (inner && (!a || !weight))) return refuse("NULL array");
    if ((rows > 1 && lda < inner) || (rows > 1 && ldo < outer))
      return refuse("a row pitch is below the row's length");
    if (wi != 1 && wo != 1 && inner > 1 && outer > 1)
      return refuse("the weight needs a unit stride along inner or outer");
    if (we < 0 || wi < 0 || wo < 0) return refuse("the weight's strides must not be negative");
    if (int rc = check_workspace(workspace, workspace_bytes,
                                 purin_train_expert_product_workspace_bytes(dtype, rows, inner,
                                                                            outer, experts)))
      return rc;
    return by_dtype(dtype, [&](auto v) {
      using T = decltype(v);
      if constexpr (sizeof(T) == 2)
        return product16<T>((hipStream_t)stream, rows, inner, outer, experts, (const T*)a, lda,
                            (const T*)weight, we, wi, wo, offsets, workspace, (T*)out, ldo);
      else
        return product32<T>((hipStream_t)stream, rows, inner, outer, experts, (const T*)a, lda,
                            (const T*)weight, we, wi, wo, offsets, workspace, (T*)out, ldo);
    });
  });
}

int64_t purin_train_expert_weights_vjp_workspace_bytes(int32_t dtype, int64_t rows, int64_t inner,
                                                       int64_t outer, int64_t experts) {
  int64_t need = -1;
  (void)guarded([&] {
    if (int rc = check_product(dtype, rows, inner, outer, experts)) return rc;
    need = 0;
    if (inner && outer)
      need = parts_bytes(dtype_bytes(dtype) == 2
                             ? cut_weights16(rows, inner, outer, experts).splits
                             : cut_weights32(dtype == PURIN_TRAIN_F64, rows, inner, outer, experts)
                                   .splits,
                         experts * inner * outer);
    return (int)PURIN_CP_OK;
  });
  return need;
}

int purin_train_expert_weights_vjp(void* stream, int32_t dtype, int64_t rows, int64_t inner,
                                   int64_t outer, int64_t experts, const void* a, int64_t lda,
                                   const void* g, int64_t ldg, const int32_t* offsets,
                                   void* workspace, int64_t workspace_bytes, void* g_weight) {
  return guarded([&] {
    if (int rc = check_product(dtype, rows, inner, outer, experts)) return rc;
    if (!inner || !outer) return (int)PURIN_CP_OK;
    if (!offsets || !g_weight || (rows && (!a || !g))) return refuse("NULL array");
    if (rows > 1 && (lda < inner || ldg < outer))
      return refuse("a row pitch is below the row's length");
    if (int rc = check_workspace(workspace, workspace_bytes,
                                 purin_train_expert_weights_vjp_workspace_bytes(
                                     dtype, rows, inner, outer, experts)))
      return rc;
    return by_dtype(dtype, [&](auto v) {
      using T = decltype(v);
      if constexpr (sizeof(T) == 2)
        return weights_vjp16<T>((hipStream_t)stream, rows, inner, outer, experts, (const T*)a, lda,
                                (const T*)g, ldg, offsets, workspace, (T*)g_weight);
      else
        return weights_vjp32<T>((hipStream_t)stream, rows, inner, outer, experts, (const T*)a, lda,
                                (const T*)g, ldg, offsets, workspace, (T*)g_weight);
    });
  });
}

}  // extern "C"
