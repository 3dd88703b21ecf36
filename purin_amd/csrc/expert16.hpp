// Tiles of the experts' products in 16-bit types on the matrix units: c = sum over k of
// a(i, k) b(j, k), sums in 32 bits, for a workgroup's BM x BN tile.
//
// The operands pass through LDS kDepth16 of the contraction at a time, in a ring of stages (two;
// four where tiles, or their rows, are few), the next ones loading while the present one is
// multiplied.  A stage of an operand whose contraction is contiguous in memory is [i][k]; one
// whose rows are contiguous is [k][i], and is transposed by the LDS reads themselves
// (ds_read_b64_tr_b16: 16 lanes read a 4 x 16 block and get its columns).  Both are stored in
// 16-byte pieces whose places are exchanged by an XOR, which spreads the lanes of one read over
// the banks:
//   [i][k]   piece k / 8 of row i at (k / 8) ^ (i % 8): 8 rows' reads of one piece fall on 8 places
//   [k][i]   pair i / 16 of row k at (i / 16) ^ s(k), s(k) = 2 (k % 4) + (k / 8) % 2 (2 ((k / 2) % 2)
//            in rows of 64, two of which cover the banks): the 8 blocks of 32 bytes that half a
//            wavefront reads at once fall on 8 places
// Counted over the large products, conflicts take 40-50 % of the LDS cycles with [i][k] stages and
// 4 % in the weights' gradient, which has [k][i] ones alone.
// With 16-byte rows at 16-byte addresses the stages are loaded straight into LDS (buffer loads
// whose addresses outside the operand read zeros); others pass through registers.
//
// 256 x 256 tiles are bound by the matrix units and what the LDS reads and barriers leave of
// them: 0.95 PFLOP/s, 1.05 for the weights' gradient (32768 rows, 16 experts, 2048 x 4096, bf16;
// a library's single product of 8192 reaches 1.2), 0.58 through registers at 1613 x 3618.  The
// tiles for few rows are bound by memory: 4.6-4.8 TB/s (768 rows, 32 experts, 4096 x 1536).
#pragma once

#include "stages.hpp"

namespace purin {
namespace train {

typedef bf16 B8 __attribute__((ext_vector_type(8)));
typedef f16 H8 __attribute__((ext_vector_type(8)));
typedef short S4 __attribute__((ext_vector_type(4)));
typedef short S8 __attribute__((ext_vector_type(8)));
typedef float F16x __attribute__((ext_vector_type(16)));

constexpr int kDepth16 = 64;

__device__ __forceinline__ F16x mma32(bf16, S8 a, S8 b, F16x c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(B8, a),
                                                 __builtin_bit_cast(B8, b), c, 0, 0, 0);
}
__device__ __forceinline__ F16x mma32(f16, S8 a, S8 b, F16x c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(H8, a),
                                                __builtin_bit_cast(H8, b), c, 0, 0, 0);
}

typedef uint32_t U4 __attribute__((ext_vector_type(4)));

// A buffer descriptor of 2 GiB from p on: reads beyond give zeros.
template <typename T>
__device__ __forceinline__ U4 buffer_at(const T* p) {
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  return U4{(uint32_t)u, (uint32_t)(u >> 32) & 0xffffu, 0x7ffffff0u, 0x00020000u};
}
template <typename T>
__device__ __forceinline__ uint32_t lds_address(const T* lds) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) T*)lds;
}
// 16 bytes a lane from the buffer to ``to`` + 16 * lane in LDS.  Written out, without an output
// register: the compiler would have every later LDS read wait for it, also one of the other
// stage.  The loop waits for its stage itself.  M0 holds the place; a load into LDS that follows
// a scalar write of M0 needs one wait state between them, which nothing but the s_nop supplies
// (hardware does not, and the compiler does not look inside).
__device__ __forceinline__ void load_to_lds(U4 r, uint32_t at, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane((int)to)), "v"(at), "s"(r)
               : "memory", "m0");
}

template <int N>
__device__ __forceinline__ int pair_swap(int k) {
  if constexpr (N == 64) return 2 * ((k >> 1) & 1);
  else return 2 * (k & 3) + ((k >> 3) & 1);
}

template <int N, bool ALONG, int THREADS>
struct Layout16 {
  static constexpr int kPieces = N * kDepth16 / 8;  // 16 bytes each
  static constexpr int kMine = kPieces / THREADS;
  static_assert(kPieces % THREADS == 0, "whole pieces per thread");

  static __device__ __forceinline__ bool piece(int m, int& row, int& first) {
    const int at = m * THREADS + (int)threadIdx.x;
    if constexpr (ALONG) {
      row = at >> 3;
      first = ((at & 7) ^ (row & 7)) * 8;
    } else {
      constexpr int per = N / 8;
      row = at / per;
      const int c = at % per;
      first = ((((c >> 1) ^ pair_swap<N>(row)) << 1) | (c & 1)) * 8;
    }
    return true;
  }
};

template <typename T, int N, bool ALONG, int THREADS>
struct Stage : Pieces<T, N, kDepth16, ALONG, Layout16<N, ALONG, THREADS>> {
  using Layout = Layout16<N, ALONG, THREADS>;
  static constexpr int kMine = Layout::kMine;
  static constexpr int kElems = N * kDepth16;
  static constexpr bool kAlong = ALONG;

  // byte offsets of this thread's pieces from the stage's first element; ~0 outside the rows
  static __device__ __forceinline__ void offsets(const Side<T>& o, uint32_t (&off)[kMine]) {
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      int row, first;
      Layout::piece(m, row, first);
      const bool in = (ALONG ? row : first) < o.n;
      off[m] = in ? (uint32_t)(row * (int)o.ld + first) * 2u : 0x80000000u;
    }
  }

  // straight into LDS; ``left``: what is left of the contraction
  static __device__ __forceinline__ void load_lds(const T* p, const uint32_t (&off)[kMine],
                                                  int64_t left, T* lds) {
    const U4 r = buffer_at(p);
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      uint32_t at = off[m];
      if (left < kDepth16) {
        int row, first;
        Layout::piece(m, row, first);
        if ((ALONG ? first : row) >= left) at = 0x80000000u;
      }
      load_to_lds(r, at, lds_address(lds) + (uint32_t)(m * THREADS + wave * 64) * 16u);
    }
  }

  static __device__ __forceinline__ void store_piece(int m, const Pack<T>& v, T* lds) {
    *reinterpret_cast<S8*>(lds + (m * THREADS + (int)threadIdx.x) * 8) = __builtin_bit_cast(S8, v);
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
};

// The matrix units' operand of rows i0 + lane % 32 and contraction 16 * s + 8 * (lane / 32) + 0..7.
template <typename T, int N, bool ALONG>
__device__ __forceinline__ S8 fragment(const T* lds, int i0, int s) {
  const int lane = threadIdx.x & 63;
  if constexpr (ALONG) {
    const int i = i0 + (lane & 31);
    return *reinterpret_cast<const S8*>(lds + i * kDepth16 + (((2 * s + (lane >> 5)) ^ (lane & 7)) << 3));
  } else {
    const int k4 = 8 * (lane >> 5) + ((lane & 15) >> 2);  // the places repeat after 16
    const int k = 16 * s + k4;
    const int pair = ((i0 >> 4) + ((lane >> 4) & 1)) ^ pair_swap<N>(k4);
    const T* at = lds + k * N + pair * 16 + (lane & 3) * 4;
    using L = __attribute__((address_space(3))) S4;
    const S4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L*)at);
    const S4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L*)(at + 4 * N));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// Waits until at most N of this wavefront's loads are on their way.
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N < 64, "the counter's range");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | ((N >> 4) << 14));
}

// The contraction's stages in a ring of S places: S - 1 on their way while one is multiplied.
// DIRECT: a stage past the end reads nothing (its addresses are outside) and counts all the same.
// Through registers AHEAD stages are on their way, each in registers of its own.
template <typename T, int BM, int BN, int THREADS, bool ALONG_A, bool ALONG_B, bool DIRECT, int S,
          int AHEAD = 1>
struct Ring {
  using SA = Stage<T, BM, ALONG_A, THREADS>;
  using SB = Stage<T, BN, ALONG_B, THREADS>;
  static constexpr int kStage = SA::kElems + SB::kElems;
  static constexpr int kBytes = S * kStage * 2;

  template <typename F>
  static __device__ __forceinline__ void run(const Side<T>& a, const Side<T>& b, int64_t depth,
                                             T* lds, F&& multiply) {
    if constexpr (DIRECT) {
      const T *pa = uniform(a.p), *pb = uniform(b.p);
      int64_t left = depth;
      const int64_t steps = (depth + kDepth16 - 1) / kDepth16;
      uint32_t off_a[SA::kMine], off_b[SB::kMine];
      SA::offsets(a, off_a);
      SB::offsets(b, off_b);
      auto load = [&](T* to) {
        SA::load_lds(pa, off_a, left, to);
        SB::load_lds(pb, off_b, left, to + SA::kElems);
        pa += ALONG_A ? kDepth16 : kDepth16 * a.ld;
        pb += ALONG_B ? kDepth16 : kDepth16 * b.ld;
        left -= kDepth16;
      };
      int now = 0;
#pragma unroll
      for (int s = 0; s < S - 1; ++s) load(lds + s * kStage);
      for (int64_t t = 0; t < steps; ++t) {
        const int next = now == 0 ? S - 1 : now - 1;
        // this stage is in LDS; the later ones may be on their way still
        wait_loads<(S - 2) * (SA::kMine + SB::kMine)>();
        __syncthreads();
        if (S > 2 || t + 1 < steps) load(lds + next * kStage);
        multiply(lds + now * kStage, lds + now * kStage + SA::kElems, t);
        now = now + 1 == S ? 0 : now + 1;
      }
      wait_loads<0>();  // stages past the end
      __syncthreads();
    } else {
      through_registers<T, kDepth16, SA, SB, S, AHEAD>(a, b, depth, lds, multiply);
    }
  }
};

// The bytes of LDS that tile16 needs: the ring, and the tile itself on its way out.
template <typename T, typename C, int BM, int BN, int S>
constexpr int tile16_lds() {
  constexpr int ring = S * (BM + BN) * kDepth16 * 2, out = BM * BN * (int)sizeof(C);
  return ring > out ? ring : out;
}

// A workgroup of WM * WN wavefronts; sums are written as C.
template <typename T, typename C, int BM, int BN, int WM, int WN, bool ALONG_A, bool ALONG_B,
          bool DIRECT, int S>
__device__ __forceinline__ void tile16(Side<T> a, Side<T> b, int64_t depth, unsigned char* lds,
                                       C* c, int64_t ldc) {
  constexpr int THREADS = WM * WN * 64, X = BM / WM / 32, Y = BN / WN / 32;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wi = (wave / WN) * (BM / WM), wj = (wave % WN) * (BN / WN);
  F16x acc[X][Y];
#pragma unroll
  for (int x = 0; x < X; ++x)
#pragma unroll
    for (int y = 0; y < Y; ++y)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.0f;
  constexpr int AHEAD = BM == 128 ? 2 : 1;  // as many registers as there are
  Ring<T, BM, BN, THREADS, ALONG_A, ALONG_B, DIRECT, S, AHEAD>::run(
      a, b, depth, reinterpret_cast<T*>(lds), [&](const T* la, const T* lb, int64_t) {
#pragma unroll
        for (int s = 0; s < kDepth16 / 16; ++s) {
          S8 fa[X], fb[Y];
#pragma unroll
          for (int x = 0; x < X; ++x) fa[x] = fragment<T, BM, ALONG_A>(la, wi + 32 * x, s);
#pragma unroll
          for (int y = 0; y < Y; ++y) fb[y] = fragment<T, BN, ALONG_B>(lb, wj + 32 * y, s);
#pragma unroll
          for (int x = 0; x < X; ++x)
#pragma unroll
            for (int y = 0; y < Y; ++y) acc[x][y] = mma32(T{}, fb[y], fa[x], acc[x][y]);
        }
      });
  // b's rows run along the sums' registers: 4 neighbours of c's row to a lane.  The tile passes
  // through LDS, so that whole rows leave in 16-byte pieces; a row's pieces are exchanged by its
  // number, so that a wavefront's writes, one column of 32 rows, fall on different banks.
  constexpr int V = kVec<C>, kPieces = BN / V;
  C* out = reinterpret_cast<C*>(lds);
#pragma unroll
  for (int x = 0; x < X; ++x) {
    const int i = wi + 32 * x + (lane & 31);
#pragma unroll
    for (int y = 0; y < Y; ++y)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int j = wj + 32 * y + 2 * r + 4 * (lane >> 5);
        typedef C V4 __attribute__((ext_vector_type(4)));
        V4 v;
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = (C)acc[x][y][r + q];
        *reinterpret_cast<V4*>(out + i * BN + (((j / V) ^ (i & (kPieces - 1))) * V + j % V)) = v;
      }
  }
  __syncthreads();
#pragma unroll 4
  for (int at = threadIdx.x; at < BM * kPieces; at += THREADS) {
    const int i = at / kPieces, j = at % kPieces * V;
    if (i >= a.n || j >= b.n) continue;
    store_upto(c + i * ldc + j, load16(out + i * BN + ((j / V) ^ (i & (kPieces - 1))) * V),
               b.n - j);
  }
}

// Few rows: at most BM, by BN, where reading b is the work.  kThin stages, all but one of them
// on their way at any time; the 4 wavefronts share a stage's contraction (16 each) and add up
// their sums at the end, in LDS, in their order.  ``lds`` holds thin_lds<BM, BN>() bytes.
constexpr int kThin = 4;
template <int BM, int BN>
constexpr int thin_lds() {
  constexpr int stages = kThin * (BM + BN) * kDepth16 * 2, sums = 4 * BM * (BN + 4) * 4;
  return stages > sums ? stages : sums;
}

template <typename T, typename C, int BM, int BN, bool ALONG_B, bool DIRECT>
__device__ __forceinline__ void thin16(Side<T> a, Side<T> b, int64_t depth, unsigned char* lds,
                                       C* c, int64_t ldc) {
  constexpr int THREADS = 256, X = BM / 32, Y = BN / 32, P = BN + 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  F16x acc[X][Y];
#pragma unroll
  for (int x = 0; x < X; ++x)
#pragma unroll
    for (int y = 0; y < Y; ++y)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.0f;
  Ring<T, BM, BN, THREADS, true, ALONG_B, DIRECT, kThin, kThin - 1>::run(
      a, b, depth, reinterpret_cast<T*>(lds), [&](const T* la, const T* lb, int64_t) {
        S8 fa[X], fb[Y];
#pragma unroll
        for (int x = 0; x < X; ++x) fa[x] = fragment<T, BM, true>(la, 32 * x, wave);
#pragma unroll
        for (int y = 0; y < Y; ++y) fb[y] = fragment<T, BN, ALONG_B>(lb, 32 * y, wave);
#pragma unroll
        for (int x = 0; x < X; ++x)
#pragma unroll
          for (int y = 0; y < Y; ++y) acc[x][y] = mma32(T{}, fb[y], fa[x], acc[x][y]);
      });
  float* sums = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int x = 0; x < X; ++x)
#pragma unroll
    for (int y = 0; y < Y; ++y)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        sums[(wave * BM + 32 * x + (lane & 31)) * P + 32 * y + 2 * (r & ~3) + 4 * (lane >> 5) +
             (r & 3)] = acc[x][y][r];
  __syncthreads();
  constexpr int V = kVec<C>;
  for (int at = threadIdx.x; at < BM * BN / V; at += THREADS) {
    const int i = at / (BN / V), j = at % (BN / V) * V;
    if (i >= a.n || j >= b.n) continue;
    Pack<C> v;
#pragma unroll
    for (int q = 0; q < V; ++q) {
      float s = sums[i * P + j + q];
#pragma unroll
      for (int w = 1; w < 4; ++w) s += sums[(w * BM + i) * P + j + q];
      v.v[q] = (C)s;
    }
    store_upto(c + i * ldc + j, v, b.n - j);
  }
}

}  // namespace train
}  // namespace purin
