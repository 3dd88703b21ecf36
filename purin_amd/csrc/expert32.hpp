// Tiles of the experts' products in 32- and 64-bit types on the matrix units: c = sum over k of
// a(i, k) b(j, k).
//
// The matrix units take one value a lane of these types (16 x 16 x 4), at 64 operations a cycle
// and SIMD (32 in 64 bits), so that their time covers the LDS reads with room to spare.  A stage
// is 128 bytes along the contraction, and passes through registers, which takes any alignment and
// length; three are on their way, each in registers of its own, but for the 128 x 128 tiles, whose
// sums leave room for one.  A lane reads 16 bytes along the
// contraction at once: step t of a stage multiplies the t-th value of each lane group's 16
// bytes, an order that both operands share.
//
// f32 reaches 115 TFLOP/s at 32768 rows, 16 experts, 2048 x 4096 (119 the weights' gradient; a
// library's product of 8192 153), 60 at 3001 rows, 7 experts, 515 x 777, where 2.4 workgroups a
// CU leave the units idle between their reads and barriers.
//
// Sums: the units add in 32 bits one after another.  Every kBlock of the contraction the sums
// are added to a second set, so that the rounding errors grow with the square roots of kBlock
// and of the number of blocks, not of the whole length.
#pragma once

#include "stages.hpp"

namespace purin {
namespace train {

typedef float F4 __attribute__((ext_vector_type(4)));
typedef double D4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ F4 mma4(float a, float b, F4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ D4 mma4(double a, double b, D4 c) {
  return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0);
}
template <typename T>
struct Wide {
  using Acc = F4;
  // sum r of a lane is row(lane, r) of the first operand, column lane % 16 of the second
  static __device__ __forceinline__ int row(int lane, int r) { return 4 * (lane >> 4) + r; }
};
template <>
struct Wide<double> {
  using Acc = D4;
  static __device__ __forceinline__ int row(int lane, int r) { return 4 * r + (lane >> 4); }
};

template <typename T>
constexpr int kDepth32 = 128 / (int)sizeof(T);
constexpr int kBlock32 = 64;

template <typename T, int N, bool ALONG, int THREADS>
struct Layout32 {
  static constexpr int V = kVec<T>, D = kDepth32<T>;
  static constexpr int kPieces = N * D / V;
  static constexpr int kMine = (kPieces + THREADS - 1) / THREADS;

  static __device__ __forceinline__ bool piece(int m, int& row, int& first) {
    const int at = m * THREADS + (int)threadIdx.x;
    constexpr int per = (ALONG ? D : N) / V;
    row = at / per;
    first = at % per * V;
    return kPieces % THREADS == 0 || at < kPieces;
  }
};

template <typename T, int N, bool ALONG, int THREADS>
struct Stage32 : Pieces<T, N, kDepth32<T>, ALONG, Layout32<T, N, ALONG, THREADS>> {
  using Layout = Layout32<T, N, ALONG, THREADS>;
  static constexpr int V = kVec<T>, D = kDepth32<T>, kMine = Layout::kMine;
  static constexpr bool kAlong = ALONG;
  // elements of a row in LDS: 144 bytes a row, whose 16-byte pieces at 8 rows fall on different
  // banks; or N elements and a pad that puts the 4 lane groups' rows on different banks
  static constexpr int kPitch = ALONG ? D + V : N + (sizeof(T) == 4 ? 4 : 8);
  static constexpr int kElems = (ALONG ? N : D) * kPitch;

  static __device__ __forceinline__ void store_piece(int m, const Pack<T>& v, T* lds) {
    int row, first;
    if (!Layout::piece(m, row, first)) return;
    typedef T W __attribute__((ext_vector_type(V)));
    W x;
#pragma unroll
    for (int q = 0; q < V; ++q) x[q] = v.v[q];
    *reinterpret_cast<W*>(lds + row * kPitch + first) = x;
  }
  static __device__ __forceinline__ void store(const Pack<T> (&v)[kMine], T* lds) {
#pragma unroll
    for (int m = 0; m < kMine; ++m) store_piece(m, v[m], lds);
  }
  // the pieces that ``move`` names moved into place on their way
  static __device__ __forceinline__ void store_settled(uint32_t move, int by,
                                                       const Pack<T> (&v)[kMine], T* lds) {
    if (ALONG || by == 0) return store(v, lds);
#pragma unroll
    for (int m = 0; m < kMine; ++m)
      store_piece(m, moved(v[m], (move >> m) & 1u ? by : 0), lds);
  }
  // a lane's V values of row i0 + lane % 16 in part ``half`` of the stage
  static __device__ __forceinline__ Pack<T> fragment(const T* lds, int i0, int half) {
    const int lane = threadIdx.x & 63, i = i0 + (lane & 15), k = V * (lane >> 4) + half * (D / 2);
    Pack<T> f;
    if constexpr (ALONG) {
      typedef T W __attribute__((ext_vector_type(V)));
      const W x = *reinterpret_cast<const W*>(lds + i * kPitch + k);
#pragma unroll
      for (int q = 0; q < V; ++q) f.v[q] = x[q];
    } else {
#pragma unroll
      for (int q = 0; q < V; ++q) f.v[q] = lds[(k + q) * kPitch + i];
    }
    return f;
  }
};

template <typename T, int BM, int BN, bool ALONG_A, bool ALONG_B>
constexpr int lds32() {
  return 2 * (Stage32<T, BM, ALONG_A, 256>::kElems + Stage32<T, BN, ALONG_B, 256>::kElems) *
         (int)sizeof(T);
}

// A workgroup of WM * WN = 4 wavefronts; AHEAD stages are on their way in registers.
template <typename T, int BM, int BN, int WM, int WN, bool ALONG_A, bool ALONG_B, int AHEAD>
__device__ __forceinline__ void tile32(Side<T> a, Side<T> b, int64_t depth, T* lds, T* c,
                                       int64_t ldc) {
  static_assert(WM * WN == 4, "four wavefronts");
  constexpr int X = BM / WM / 16, Y = BN / WN / 16, V = kVec<T>, D = kDepth32<T>;
  using SA = Stage32<T, BM, ALONG_A, 256>;
  using SB = Stage32<T, BN, ALONG_B, 256>;
  using Acc = typename Wide<T>::Acc;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wi = (wave / WN) * (BM / WM), wj = (wave % WN) * (BN / WN);
  Acc acc[X][Y], all[X][Y];
#pragma unroll
  for (int x = 0; x < X; ++x)
#pragma unroll
    for (int y = 0; y < Y; ++y) acc[x][y] = all[x][y] = Acc{0, 0, 0, 0};
  through_registers<T, D, SA, SB, 2, AHEAD>(
      a, b, depth, lds, [&](const T* la, const T* lb, int64_t t) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          Pack<T> fa[X], fb[Y];
#pragma unroll
          for (int x = 0; x < X; ++x) fa[x] = SA::fragment(la, wi + 16 * x, half);
#pragma unroll
          for (int y = 0; y < Y; ++y) fb[y] = SB::fragment(lb, wj + 16 * y, half);
#pragma unroll
          for (int q = 0; q < V; ++q)
#pragma unroll
            for (int x = 0; x < X; ++x)
#pragma unroll
              for (int y = 0; y < Y; ++y) acc[x][y] = mma4(fa[x].v[q], fb[y].v[q], acc[x][y]);
        }
        if constexpr (sizeof(T) == 4)
          if (t % (kBlock32 / D) == kBlock32 / D - 1) {
#pragma unroll
            for (int x = 0; x < X; ++x)
#pragma unroll
              for (int y = 0; y < Y; ++y) {
                all[x][y] += acc[x][y];
                acc[x][y] = Acc{0, 0, 0, 0};
              }
          }
      });
#pragma unroll
  for (int x = 0; x < X; ++x)
#pragma unroll
    for (int y = 0; y < Y; ++y) {
      const Acc sum = all[x][y] + acc[x][y];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = wi + 16 * x + Wide<T>::row(lane, r), j = wj + 16 * y + (lane & 15);
        if (i < a.n && j < b.n) c[i * ldc + j] = sum[r];
      }
    }
}

}  // namespace train
}  // namespace purin
