// The experts' products with microscaled 4-bit weights (include/purin_train.h:
// expert_product_packed): out(p) = a(p) W[e] with W[e] a product of codes and powers of two.

#include "packed.hpp"
#include "tiles.hpp"

namespace purin {
namespace train {

template <typename T, int B, int WN, int S>
__global__ __launch_bounds__(2 * WN * 64) void k_product_packed(
    const T* __restrict__ a, int64_t lda, const uint8_t* __restrict__ codes,
    const uint8_t* __restrict__ scales, int64_t rows, int64_t inner, int64_t outer, int experts,
    int64_t tiles_m, int64_t tiles_n, const int32_t* __restrict__ offsets, T* __restrict__ out,
    int64_t ldo) {
  extern __shared__ __align__(16) unsigned char lds16[];
  int64_t tm, tn;
  tile_order(tiles_m, tiles_n, tm, tn);
  int e;
  int64_t from, to;
  if (!find_tile(offsets, experts, rows, B, tm, e, from, to)) return;
  e = __builtin_amdgcn_readfirstlane(e);
  const int64_t col = tn * B;
  const int m = __builtin_amdgcn_readfirstlane((int)min<int64_t>(B, to - from));
  const int n = (int)min<int64_t>(B, outer - col);
  T* c = out + from * ldo + col;
  if (e < 0) {
    zero_tile(c, ldo, m, n);
    return;
  }
  TileHalf<T, B, B, 2, WN, S>::run(a + from * lda, lda, m, inner,
                                   Codes(codes, scales, e * outer + col, inner), n, lds16, c, ldo);
}

// Split number blockIdx.y of the contraction writes its own ``out``.
template <typename T, typename C, int BM, int S>
__global__ __launch_bounds__(256) void k_product_packed_thin(
    const T* __restrict__ a, int64_t lda, const uint8_t* __restrict__ codes,
    const uint8_t* __restrict__ scales, int64_t rows, int64_t inner, int64_t outer, int experts,
    int64_t tiles_n, const int32_t* __restrict__ offsets, C* __restrict__ out, int64_t ldo) {
  extern __shared__ __align__(16) unsigned char lds16[];
  const int64_t tm = blockIdx.x / tiles_n, tn = blockIdx.x - tm * tiles_n;
  int e;
  int64_t from, to;
  if (!find_tile(offsets, experts, rows, BM, tm, e, from, to)) return;
  e = __builtin_amdgcn_readfirstlane(e);
  const int64_t col = tn * 64;
  const int m = __builtin_amdgcn_readfirstlane((int)min<int64_t>(BM, to - from));
  const int n = (int)min<int64_t>(64, outer - col);
  C* c = out + (int64_t)blockIdx.y * rows * ldo + from * ldo + col;
  if (e < 0) {
    zero_tile(c, ldo, m, n);
    return;
  }
  using Thin = ThinPacked<T, BM, 1, S>;
  F16x acc[BM / 32][2];
#pragma unroll
  for (int x = 0; x < BM / 32; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.0f;
  const Codes b(codes, scales, e * outer + col, inner);
  const int64_t stages = (b.blocks + 7) / 8, per = (stages + gridDim.y - 1) / gridDim.y;
  const int64_t first = min<int64_t>(b.blocks, blockIdx.y * per * 8);
  const T* const from_a[1] = {a + from * lda};
  Thin::run(from_a, [&](int r) { return r < m ? (uint32_t)r * (uint32_t)lda * 2u : kOutside; }, inner,
            b, [&](int j) { return j < n ? j : -1; }, first, min<int64_t>(b.blocks - first, per * 8),
            lds16, acc);
  float* sums = reinterpret_cast<float*>(lds16);
  thin_parts<BM>(acc, sums);
  constexpr int V = kVec<C>;
  for (int at = threadIdx.x; at < BM * 64 / V; at += 256) {
    const int i = at / (64 / V), j = at % (64 / V) * V;
    if (i >= m || j >= n) continue;
    Pack<C> v;
#pragma unroll
    for (int q = 0; q < V; ++q) v.v[q] = (C)thin_sum<BM>(sums, i, j + q);
    store_upto(c + i * ldo + j, v, n - j);
  }
}

template <typename C, int B, int WN, int S>
__global__ __launch_bounds__(2 * WN * 64) void k_product_both(
    const uint8_t* __restrict__ a, const uint8_t* __restrict__ a_scales,
    const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t rows,
    int64_t inner, int64_t outer, int experts, int64_t tiles_m, int64_t tiles_n,
    const int32_t* __restrict__ offsets, C* __restrict__ out, int64_t ldo) {
  extern __shared__ __align__(16) unsigned char lds16[];
  int64_t tm, tn;
  tile_order(tiles_m, tiles_n, tm, tn);
  int e;
  int64_t from, to;
  if (!find_tile(offsets, experts, rows, B, tm, e, from, to)) return;
  e = __builtin_amdgcn_readfirstlane(e);
  const int64_t col = tn * B;
  const int m = __builtin_amdgcn_readfirstlane((int)min<int64_t>(B, to - from));
  const int n = (int)min<int64_t>(B, outer - col);
  C* c = out + from * ldo + col;
  if (e < 0) {
    zero_tile(c, ldo, m, n);
    return;
  }
  TileBoth<C, B, B, 2, WN, S>::run(Codes(a, a_scales, from, inner), m,
                                   Codes(codes, scales, e * outer + col, inner), n, lds16, c, ldo);
}

enum ShapePacked { kThinPacked, k128Packed, k256Packed };
struct CutPacked {
  ShapePacked shape;
  int height, splits;
};
static CutPacked cut_packed(bool both, int64_t rows, int64_t inner, int64_t outer, int64_t experts) {
  const int64_t tiles = most_tiles(rows, experts, 128) * ((outer + 127) / 128);
  if (!both && (rows <= 32 * experts || tiles <= 128)) {
    const int64_t across = (outer + 63) / 64;
    const bool tall = rows > 16 * experts && most_tiles(rows, experts, 64) * across >= 256;
    if (tall) return {kThinPacked, 64, 1};
    const int64_t stages = (inner + 255) / 256;
    return {kThinPacked, 32, splits_of(512, most_tiles(rows, experts, 32) * across, stages, 4)};
  }
  return {tiles >= 16 * 256 ? k256Packed : k128Packed, tiles >= 16 * 256 ? 256 : 128, 1};
}

template <typename T>
static int product_packed(hipStream_t st, int64_t rows, int64_t inner, int64_t outer,
                          int64_t experts, const T* a, int64_t lda, const uint8_t* codes,
                          const uint8_t* scales, const int32_t* offsets, uint8_t* ws, T* out,
                          int64_t ldo) {
  if (inner && !direct_ok(a, lda, inner)) {
    if (int rc = align_rows<T>(st, a, lda, rows, inner, (T*)ws)) return rc;
    a = (const T*)ws;
    lda = (inner + 7) / 8 * 8;
  }
  CutPacked cut = cut_packed(false, rows, inner, outer, experts);
  if (ldo != outer) cut.splits = 1;  // the parts are added up as one row
  if (cut.shape == kThinPacked) {
    float* parts = (float*)(ws + aligned_bytes(rows, inner));
    const int64_t tm = most_tiles(rows, experts, cut.height), tn = (outer + 63) / 64;
    auto thin = [&](auto c, auto h) {
      using C = decltype(c);
      constexpr int BM = h, S = BM == 32 ? 3 : 3;
      constexpr int ring = ThinPacked<T, BM, 1, S>::kRing;
      return launch16("k_product_packed_thin", k_product_packed_thin<T, C, BM, S>, tm * tn,
                      (unsigned)cut.splits, 1, 256, ring > kThinSums<BM> ? ring : kThinSums<BM>, st,
                      a, lda, codes, scales, rows, inner, outer, (int)experts, tn, offsets,
                      cut.splits > 1 ? (C*)parts : (C*)out, ldo);
    };
    if (cut.splits == 1) return cut.height == 32 ? thin(T{}, i32) : thin(T{}, i64);
    if (int rc = thin(float{}, i32)) return rc;
    return join(st, parts, cut.splits, rows * outer, out);
  }
  auto go = [&](auto bm, auto wn, auto s) {
    constexpr int B = bm, WN = wn, S = s;
    const int64_t tm = most_tiles(rows, experts, B), tn = (outer + B - 1) / B;
    return launch16("k_product_packed", k_product_packed<T, B, WN, S>, tm * tn, 1, 1, 2 * WN * 64,
                    TileHalf<T, B, B, 2, WN, S>::kLds, st, a, lda, codes, scales, rows, inner, outer,
                    (int)experts, tm, tn, offsets, out, ldo);
  };
  if (cut.shape == k256Packed) return go(i256, i4, integral_constant<int, 3>{});
  return go(i128, i2, integral_constant<int, 3>{});
}

template <typename C>
static int product_both(hipStream_t st, int64_t rows, int64_t inner, int64_t outer, int64_t experts,
                        const uint8_t* a, const uint8_t* a_scales, const uint8_t* codes,
                        const uint8_t* scales, const int32_t* offsets, C* out, int64_t ldo) {
  const CutPacked cut = cut_packed(true, rows, inner, outer, experts);
  auto go = [&](auto bm, auto wn, auto s) {
    constexpr int B = bm, WN = wn, S = s;
    const int64_t tm = most_tiles(rows, experts, B), tn = (outer + B - 1) / B;
    return launch16("k_product_both", k_product_both<C, B, WN, S>, tm * tn, 1, 1, 2 * WN * 64,
                    TileBoth<C, B, B, 2, WN, S>::kLds, st, a, a_scales, codes, scales, rows, inner,
                    outer, (int)experts, tm, tn, offsets, out, ldo);
  };
  // a tile of 256 x 256 sums in 32 bits does not fit LDS on its way out
  if constexpr (sizeof(C) == 2)
    if (cut.shape == k256Packed) return go(i256, i4, i2);
  return go(i128, i2, i2);
}

static int check_packed(int32_t dtype, int32_t both, int64_t rows, int64_t inner, int64_t outer,
                        int64_t experts) {
  if (int rc = check_product(dtype, rows, inner, outer, experts)) return rc;
  if (dtype == PURIN_TRAIN_F64 || (dtype == PURIN_TRAIN_F32 && !both))
    return set_error(PURIN_CP_ERR_UNSUPPORTED,
                     "packed weights take rows of 16 bits, or packed rows with results of at most 32");
  return PURIN_CP_OK;
}

}  // namespace train
}  // namespace purin

using namespace purin;
using namespace purin::train;

extern "C" {

int64_t purin_train_expert_product_packed_workspace_bytes(int32_t dtype, int32_t rows_packed,
                                                          int64_t rows, int64_t inner,
                                                          int64_t outer, int64_t experts) {
  int64_t need = -1;
  (void)guarded([&] {
    if (int rc = check_packed(dtype, rows_packed, rows, inner, outer, experts)) return rc;
    need = 0;
    if (rows && outer && inner && !rows_packed) {
      const int splits = cut_packed(false, rows, inner, outer, experts).splits;
      // rows whose length is a multiple of 8 may still lie at other addresses
      need = aligned_bytes(rows, inner) + parts_bytes(splits, rows * outer);
    }
    return (int)PURIN_CP_OK;
  });
  return need;
}

int purin_train_expert_product_packed(void* stream, int32_t dtype, int64_t rows, int64_t inner,
                                      int64_t outer, int64_t experts, const void* a, int64_t lda,
                                      const void* a_scales, const void* codes, const void* scales,
                                      const int32_t* offsets, void* workspace,
                                      int64_t workspace_bytes, void* out, int64_t ldo) {
  return guarded([&] {
    const int32_t both = a_scales != nullptr;
    if (int rc = check_packed(dtype, both, rows, inner, outer, experts)) return rc;
    if (!rows || !outer) return (int)PURIN_CP_OK;
    if (!offsets || !out || (inner && (!a || !codes || !scales))) return refuse("NULL array");
    if (rows > 1 && ((!both && lda < inner) || ldo < outer))
      return refuse("a row pitch is below the row's length");
    const uintptr_t odd = (reinterpret_cast<uintptr_t>(codes) % 16) |
                          (reinterpret_cast<uintptr_t>(scales) % 4) |
                          (both ? reinterpret_cast<uintptr_t>(a) % 16 |
                                      reinterpret_cast<uintptr_t>(a_scales) % 4
                                : 0);
    if (odd) return refuse("codes must lie at 16 bytes, scales at 4");
    if (int rc = check_workspace(workspace, workspace_bytes,
                                 purin_train_expert_product_packed_workspace_bytes(
                                     dtype, both, rows, inner, outer, experts)))
      return rc;
    auto dense = [&](auto v) {
      using T = decltype(v);
      return product_packed<T>((hipStream_t)stream, rows, inner, outer, experts, (const T*)a, lda,
                               (const uint8_t*)codes, (const uint8_t*)scales, offsets,
                               (uint8_t*)workspace, (T*)out, ldo);
    };
    auto packed = [&](auto v) {
      using C = decltype(v);
      return product_both<C>((hipStream_t)stream, rows, inner, outer, experts, (const uint8_t*)a,
                             (const uint8_t*)a_scales, (const uint8_t*)codes,
                             (const uint8_t*)scales, offsets, (C*)out, ldo);
    };
    if (both)
      return dtype == PURIN_TRAIN_BF16 ? packed(bf16{})
                                       : dtype == PURIN_TRAIN_F16 ? packed(f16{}) : packed(float{});
    return dtype == PURIN_TRAIN_BF16 ? dense(bf16{}) : dense(f16{});
  });
}

}  // extern "C"
