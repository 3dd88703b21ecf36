// The experts' products with microscaled 4-bit weights (include/purin_train.h:
// expert_product_packed): out(p) = a(p) W[e] with W[e] a product of codes and powers of two.

#include "packed.hpp"
#include "tiles.hpp"

namespace purin {
namespace train {

template <typename T, int B, int WN>
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
  TileHalf<T, B, WN>::run(a + from * lda, lda, m, inner,
                          Codes(codes, scales, e * outer + col, inner), n, lds16, c, ldo);
}

// Split number blockIdx.y of the contraction writes its own ``out``.  A tile has 64 columns to each
// set of ``parts`` wavefronts.  An expert's tiles are dealt to all XCDs, which reads its rows into each
// L2 (32 experts, 4096 x 1536, 24 rows to each: 165 MB, 115 of them needed): on one XCD they read 120 MB,
// but the same rows' lines at the same time, and take 44 us for 37.
template <typename T, typename C, int BM>
__global__ __launch_bounds__(256, 2) void k_product_packed_thin(
    Rows a, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t rows,
    int64_t inner, int64_t outer, int experts, int parts, int64_t tiles_n,
    const int32_t* __restrict__ offsets, C* __restrict__ out, int64_t ldo) {
  constexpr int kLds = kThinSums<BM> > kLineLds ? kThinSums<BM> : kLineLds;
  __shared__ __align__(16) uint8_t lds[kLds];
  const int64_t tm = blockIdx.x / tiles_n, tn = blockIdx.x - tm * tiles_n;
  int e;
  int64_t from, to;
  if (!find_tile(offsets, experts, rows, BM, tm, e, from, to)) return;
  e = __builtin_amdgcn_readfirstlane(e);
  const int wide = 64 * (4 / parts);
  const int64_t col = tn * wide;
  const int m = __builtin_amdgcn_readfirstlane((int)min<int64_t>(BM, to - from));
  const int n = (int)min<int64_t>(wide, outer - col);
  C* c = out + (int64_t)blockIdx.y * rows * ldo + from * ldo + col;
  if (e < 0) {
    zero_tile(c, ldo, m, n);
    return;
  }
  ThinAcc<BM> acc;
  const Codes b(codes, scales, (int64_t)e * outer, inner);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int own = wave / parts * 64;  // the wavefront's columns
  Columns cols;
  cols.first[0] = col + own;
  cols.first[1] = col + own + 32;
  cols.n[0] = max(min(n - own, 32), 0);
  cols.n[1] = max(min(n - own - 32, 32), 0);
  const Rows from_a[1] = {{(const uint8_t*)a.p + from * a.pitch, a.step, a.pitch}};
  int first, end, at, upto;
  share_lines(0, cols.n[0] ? b.lines() : 0, (int)blockIdx.y, (int)gridDim.y, first, end);
  share_lines(first, end, wave % parts, parts, at, upto);
  StreamCodes<T, BM, 1>::run(from_a, [&](int r) { return r < m ? r : -1; }, inner, b, cols, at, upto,
                             lds, acc);
  float* sums = reinterpret_cast<float*>(lds);
  __syncthreads();
  thin_parts<BM>(acc, sums);
  constexpr int V = kVec<C>;
  for (int i = threadIdx.x; i < m * (wide / V); i += 256) {
    const int r = i / (wide / V), j = i % (wide / V) * V;
    if (j >= n) continue;
    Pack<C> v;
#pragma unroll
    for (int q = 0; q < V; ++q) v.v[q] = (C)thin_sum<BM>(sums, parts, r, j + q);
    store_upto(c + r * ldo + j, v, n - j);
  }
}

template <typename C, int B, int WN, bool CHUNKS>
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
  TileBoth<C, B, WN, CHUNKS>::run(Codes(a, a_scales, from, inner), m,
                                  Codes(codes, scales, e * outer + col, inner), n, lds16, c, ldo);
}

// How a product is cut.  us of 32 experts, 4096 x 1536, so many rows to each, bf16:
//   rows     1     8    16    24    32    48    64    96   192   400
//   16    27.2  28.0  31.0    51    49    67     -     -     -     -   streams, 16 rows to a tile
//   32    30.1  32.4  36.1  38.8    43    67    74    92   158   270   32 rows
//   128   54.8  54.8  57.1  58.9    59    89    91    98   129   225   128 x 128 tiles
//   256     89    85    85    85    86    88    89   169   182   203   256 x 256
// Streams are bound by memory (27.2 us: 4.1 TB/s) until an expert's rows take a second tile, which
// reads its weights again.  16 experts, 2048 x 4096, 128 | 256, rows of 16 bits: 8192 rows 167 | 171,
// 16384 293 | 285, 32768 591 | 522; packed rows 66 | 67, 115 | 111, 234 | 201: from 16 tiles of
// 128 x 128 to a CU on, as in 16 bits.  Where CUs are idle a stream's contraction is split.
// Packed rows take tiles always: 8 rows, 2 experts, 4096 x 4096 15 us, where 16-bit rows take 13 for
// the stream and 2-4 for joining its parts; 768 rows, 32 experts, 4096 x 1536 28, those 37 and 5.5 for
// laying the rows side by side.
enum ShapePacked { kThinPacked, k128Packed, k256Packed };
struct CutPacked {
  ShapePacked shape;
  int height, parts, splits;
};
static CutPacked cut_packed(bool both, int64_t rows, int64_t inner, int64_t outer, int64_t experts) {
  const int64_t tiles = most_tiles(rows, experts, 128) * ((outer + 127) / 128);
  if (!both && (rows <= 96 * experts || tiles <= 64)) {
    const int height = rows <= 12 * experts ? 16 : 32;
    const int64_t streams = most_tiles(rows, experts, height) * ((outer + 63) / 64);
    const int parts = stream_parts(streams);
    return {kThinPacked, height, parts,
            splits_of(1024, streams * parts / 4, (inner + 255) / 256, parts)};
  }
  return {tiles >= 16 * 256 ? k256Packed : k128Packed, 0, 0, 1};
}

template <typename T>
static int product_packed(hipStream_t st, int64_t rows, int64_t inner, int64_t outer,
                          int64_t experts, const T* a, int64_t lda, const uint8_t* codes,
                          const uint8_t* scales, const int32_t* offsets, uint8_t* ws, T* out,
                          int64_t ldo) {
  if (rows == 1) lda = 0;  // one row has any pitch
  CutPacked cut = cut_packed(false, rows, inner, outer, experts);
  if (ldo != outer) cut.splits = 1;  // the parts are added up as one row
  if (cut.shape == kThinPacked) {
    Rows from{a, 16u, (uint32_t)lda * 2u};
    // rows that fill their tiles are worth a launch that lays them side by side (32 experts, 4096 x
    // 1536, 48 rows to each: 67 us, 80 without; 24 to each, unequal: 47.6, 51; 16 to each: 34, 31)
    if (inner && (rows > 16 * experts || !direct_ok(a, lda, inner))) {
      if (int rc = turn_rows<T>(st, a, lda, rows, inner, ws)) return rc;
      from = {ws, (uint32_t)rows * 16u, 16u};
    }
    float* parts = (float*)(ws + aligned_bytes(rows, inner));
    const int wide = 64 * (4 / cut.parts);
    const int64_t tm = most_tiles(rows, experts, cut.height), tn = (outer + wide - 1) / wide;
    auto thin = [&](auto c) {
      using C = decltype(c);
      return launch16("k_product_packed_thin",
                      cut.height == 16 ? k_product_packed_thin<T, C, 16> : k_product_packed_thin<T, C, 32>,
                      tm * tn, (unsigned)cut.splits, 1, 256, 0, st, from, codes, scales, rows, inner,
                      outer, (int)experts, cut.parts, tn, offsets, cut.splits > 1 ? (C*)parts : (C*)out,
                      ldo);
    };
    if (cut.splits == 1) return thin(T{});
    if (int rc = thin(float{})) return rc;
    return join(st, parts, cut.splits, rows * outer, out);
  }
  if (inner && !direct_ok(a, lda, inner)) {
    if (int rc = align_rows<T>(st, a, lda, rows, inner, ws)) return rc;
    a = (const T*)ws;
    lda = (inner + 7) / 8 * 8;
  }
  auto go = [&](auto bm, auto wn) {
    constexpr int B = bm, WN = wn;
    const int64_t tm = most_tiles(rows, experts, B), tn = (outer + B - 1) / B;
    return launch16("k_product_packed", k_product_packed<T, B, WN>, tm * tn, 1, 1, 2 * WN * 64,
                    TileHalf<T, B, WN>::kLds, st, a, lda, codes, scales, rows, inner, outer, (int)experts,
                    tm, tn, offsets, out, ldo);
  };
  return cut.shape == k256Packed ? go(i256, i4) : go(i128, i2);
}

template <typename C>
static int product_both(hipStream_t st, int64_t rows, int64_t inner, int64_t outer, int64_t experts,
                        const uint8_t* a, const uint8_t* a_scales, const uint8_t* codes,
                        const uint8_t* scales, const int32_t* offsets, C* out, int64_t ldo) {
  const CutPacked cut = cut_packed(true, rows, inner, outer, experts);
  auto go = [&](auto bm, auto wn) {
    constexpr int B = bm, WN = wn;
    const int64_t tm = most_tiles(rows, experts, B), tn = (outer + B - 1) / B;
    auto run = [&](auto chunks) {
      using Tile = TileBoth<C, B, WN, chunks>;
      return launch16("k_product_both", k_product_both<C, B, WN, chunks>, tm * tn, 1, 1, 2 * WN * 64,
                      Tile::kLds, st, a, a_scales, codes, scales, rows, inner, outer, (int)experts, tm,
                      tn, offsets, out, ldo);
    };
    // whole pieces of 16 bytes of a row's scales
    const bool chunks = micro_filled(micro_blocks(inner)) % 16 == 0 &&
                        reinterpret_cast<uintptr_t>(scales) % 16 == 0 &&
                        reinterpret_cast<uintptr_t>(a_scales) % 16 == 0;
    return chunks ? run(std::true_type{}) : run(std::false_type{});
  };
  // a tile of 256 x 256 sums in 32 bits does not fit LDS on its way out
  if constexpr (sizeof(C) == 2)
    if (cut.shape == k256Packed) return go(i256, i4);
  return go(i128, i2);
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
