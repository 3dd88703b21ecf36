// Tiles of the experts' products in 32- and 64-bit types on the matrix units: c = sum over k of
// a(i, k) b(j, k).
//
// The matrix units take one value a lane of these types (16 x 16 x 4), at 64 operations a cycle
// and SIMD (32 in 64 bits), so that their time covers the LDS reads with room to spare and one
// stage of 128 bytes along the contraction on its way is enough.  Stages pass
// through registers, which takes any alignment and length.  A lane reads 16 bytes along the
// contraction at once: step t of a stage multiplies the t-th value of each lane group's 16
// bytes, an order that both operands share.
//
// Sums: the units add in 32 bits one after another.  Every kBlock of the contraction the sums
// are added to a second set, so that the rounding errors grow with the square roots of kBlock
// and of the number of blocks, not of the whole length.
#pragma once

#include "train.hpp"

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

// An operand: element (i, k) at p + i * ld + k (ALONG) or p + k * ld + i; n rows are there.
template <typename T>
struct Side32 {
  const T* p;
  int64_t ld;
  int n;
};

template <typename T, int N, bool ALONG, int THREADS>
struct Stage32 {
  static constexpr int V = kVec<T>, D = kDepth32<T>;
  // elements of a row in LDS: 144 bytes a row, whose 16-byte pieces at 8 rows fall on different
  // banks; or N elements and a pad that puts the 4 lane groups' rows on different banks
  static constexpr int kPitch = ALONG ? D + V : N + (sizeof(T) == 4 ? 4 : 8);
  static constexpr int kElems = (ALONG ? N : D) * kPitch;
  static constexpr int kPieces = N * D / V;
  static constexpr int kMine = (kPieces + THREADS - 1) / THREADS;

  static __device__ __forceinline__ bool piece(int m, int& row, int& first) {
    const int at = m * THREADS + (int)threadIdx.x;
    constexpr int per = (ALONG ? D : N) / V;
    row = at / per;
    first = at % per * V;
    return kPieces % THREADS == 0 || at < kPieces;
  }
  static __device__ __forceinline__ void load(const Side32<T>& o, const T* p, int64_t left,
                                              Pack<T> (&v)[kMine]) {
    // whole stages load without a condition (rows past the last are read as the last: they reach
    // no sum that is kept), so that no load waits for another's
    if (left >= D && (ALONG || o.n == N)) {
#pragma unroll
      for (int m = 0; m < kMine; ++m) {
        int row, first;
        if (piece(m, row, first)) v[m] = load16(p + (ALONG ? min(row, o.n - 1) : row) * o.ld + first);
      }
      return;
    }
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      int row, first;
      const bool in = piece(m, row, first);
      const int64_t rows = ALONG ? o.n : left, cols = ALONG ? left : o.n;
      if (!in || row >= rows || first >= cols) v[m] = zeros16<T>();
      else v[m] = load_upto(p + row * o.ld + first, cols - first);
    }
  }
  static __device__ __forceinline__ void store(const Pack<T> (&v)[kMine], T* lds) {
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      int row, first;
      if (piece(m, row, first)) {
        typedef T W __attribute__((ext_vector_type(V)));
        W x;
#pragma unroll
        for (int q = 0; q < V; ++q) x[q] = v[m].v[q];
        *reinterpret_cast<W*>(lds + row * kPitch + first) = x;
      }
    }
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
__device__ __forceinline__ void tile32(Side32<T> a, Side32<T> b, int64_t depth, T* lds, T* c,
                                       int64_t ldc) {
  static_assert(WM * WN == 4, "four wavefronts");
  constexpr int X = BM / WM / 16, Y = BN / WN / 16, V = kVec<T>, D = kDepth32<T>;
  using SA = Stage32<T, BM, ALONG_A, 256>;
  using SB = Stage32<T, BN, ALONG_B, 256>;
  using Acc = typename Wide<T>::Acc;
  constexpr int kStage = SA::kElems + SB::kElems;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wi = (wave / WN) * (BM / WM), wj = (wave % WN) * (BN / WN);
  Acc acc[X][Y], all[X][Y];
#pragma unroll
  for (int x = 0; x < X; ++x)
#pragma unroll
    for (int y = 0; y < Y; ++y) acc[x][y] = all[x][y] = Acc{0, 0, 0, 0};
  Pack<T> va[AHEAD][SA::kMine], vb[AHEAD][SB::kMine];
  const T *pa = a.p, *pb = b.p;
  int64_t left = depth;
  auto load = [&](int v) {
    SA::load(a, pa, left, va[v]);
    SB::load(b, pb, left, vb[v]);
    pa += ALONG_A ? D : D * a.ld;
    pb += ALONG_B ? D : D * b.ld;
    left -= D;
  };
  auto put = [&](int v, T* to) {
    SA::store(va[v], to);
    SB::store(vb[v], to + SA::kElems);
  };
  const int64_t steps = (depth + D - 1) / D;
#pragma unroll
  for (int s = 0; s < AHEAD; ++s) load(s);
  put(0, lds);
  T *now = lds, *next = lds + kStage;
  for (int64_t t0 = 0; t0 < steps; t0 += AHEAD) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int64_t t = t0 + u;
      if (t >= steps) break;
      __syncthreads();
      if (t + AHEAD < steps) load(u);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        Pack<T> fa[X], fb[Y];
#pragma unroll
        for (int x = 0; x < X; ++x) fa[x] = SA::fragment(now, wi + 16 * x, half);
#pragma unroll
        for (int y = 0; y < Y; ++y) fb[y] = SB::fragment(now + SA::kElems, wj + 16 * y, half);
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
      if (t + 1 < steps) put((u + 1) % AHEAD, next);
      T* swap = now;
      now = next;
      next = swap;
    }
  }
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
