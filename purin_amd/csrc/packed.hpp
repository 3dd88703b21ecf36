// Stages and tiles of products with microscaled 4-bit weights (packed.hip, layer.hip).
//
// Codes go to LDS as they are, 16 bytes (one block of 32) at a time, loaded straight there; a
// lane's fragment is a whole block.  With rows of 16 bits the codes become numbers of the rows'
// type on their way from LDS to the matrix units (v_cvt_scalef32_pk, exact): a quarter of the
// LDS traffic of 16-bit weights, and each is converted once for every wavefront that shares its
// rows.  The order of a contraction is free as long as both operands have the same one: in a
// depth of 64, lanes 0..31 hold the first block, lanes 32..63 the second, and step j of four
// multiplies elements 8 j .. 8 j + 7 of both.
//
// With packed rows the matrix units take the codes and the blocks' scales themselves
// (v_mfma_scale, 32 x 32 x 64), at four times the rate of 16 bits.
#pragma once

#include "expert16.hpp"
#include "micro.hpp"

namespace purin {
namespace train {

typedef int I4 __attribute__((ext_vector_type(4)));
typedef int I8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kOutside = 0x80000000u;  // an offset past every buffer: reads zeros

// 4 bytes a lane from the buffer to ``to`` + 4 * lane in LDS (load_to_lds's notes hold here too).
__device__ __forceinline__ void load_word_to_lds(U4 r, uint32_t at, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane((int)to)), "v"(at), "s"(r)
               : "memory", "m0");
}

// 8 codes of a word as numbers of T.
__device__ __forceinline__ S8 numbers_of(bf16, uint32_t c, float scale) {
  typedef bf16 B2 __attribute__((ext_vector_type(2)));
  const B2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0);
  const B2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1);
  const B2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2);
  const B2 e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3);
  return __builtin_bit_cast(S8, B8{a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]});
}
__device__ __forceinline__ S8 numbers_of(f16, uint32_t c, float scale) {
  typedef f16 H2 __attribute__((ext_vector_type(2)));
  const H2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 0);
  const H2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 1);
  const H2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 2);
  const H2 e = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(c, scale, 3);
  return __builtin_bit_cast(S8, H8{a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]});
}
// The scale of block ``block`` % 4 of a word of four.
__device__ __forceinline__ float scale_of(uint32_t word, int block) {
  return scale_operand((word >> (8 * (block & 3))) & 255u);
}

// A stage of N rows, PIECES pieces of 16 bytes each, in LDS [row][piece] with the pieces of a row
// exchanged by the row's number, so that a read of one piece from neighbouring rows falls on
// different banks.
template <int N, int PIECES, int THREADS>
struct PieceStage {
  static constexpr int kMine = N * PIECES / THREADS;
  static constexpr int kBytes = N * PIECES * 16;
  static_assert(N * PIECES % THREADS == 0, "whole pieces per thread");

  static __device__ __forceinline__ int place(int row, int piece) {
    if constexpr (PIECES >= 8) return row * PIECES + (piece ^ (row & 7));
    else return row * PIECES + (piece ^ ((row >> 3) & (PIECES - 1)));
  }
  // byte offsets of this thread's pieces; ``offset(row)``: the row's, kOutside for none
  template <typename F>
  static __device__ __forceinline__ void offsets(F&& offset, uint32_t (&off)[kMine]) {
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      const int at = m * THREADS + (int)threadIdx.x, row = at / PIECES;
      const int piece = place(row, at % PIECES) % PIECES;
      const uint32_t o = offset(row);
      off[m] = o == kOutside ? kOutside : o + (uint32_t)piece * 16u;
    }
  }
  // ``left``: pieces left of the rows
  static __device__ __forceinline__ void load(const uint8_t* p, const uint32_t (&off)[kMine],
                                              int64_t left, uint32_t to) {
    const U4 r = buffer_at(p);
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      uint32_t at = off[m];
      if (left < PIECES) {
        const int i = m * THREADS + (int)threadIdx.x;
        if (place(i / PIECES, i % PIECES) % PIECES >= left) at = kOutside;
      }
      load_to_lds(r, at, to + (uint32_t)(m * THREADS + wave * 64) * 16u);
    }
  }
  static __device__ __forceinline__ I4 piece(const uint8_t* lds, int row, int p) {
    return *reinterpret_cast<const I4*>(lds + place(row, p) * 16);
  }
};

// Words of four scales of N rows, WORDS of them a row, in LDS [word][row]; every thread of a
// workgroup that is larger loads one that is there already.
template <int N, int WORDS, int THREADS>
struct ScaleStage {
  static constexpr int kMine = (N * WORDS + THREADS - 1) / THREADS;
  static constexpr int kBytes = kMine * THREADS * 4;
  static_assert(N % 64 == 0, "a wavefront's rows have one word number");

  template <typename F>
  static __device__ __forceinline__ void offsets(F&& offset, uint32_t (&off)[kMine]) {
#pragma unroll
    for (int m = 0; m < kMine; ++m) off[m] = offset((m * THREADS + (int)threadIdx.x) % N);
  }
  static __device__ __forceinline__ int word(int m) {
    return (m * THREADS + (int)threadIdx.x) / N % WORDS;
  }
  // the words from number ``first`` on, of ``filled`` / 4 in a row
  static __device__ __forceinline__ void load(const uint8_t* p, const uint32_t (&off)[kMine],
                                              int first, int words, uint32_t to) {
    const U4 r = buffer_at(p);
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      const int w = first + word(m);
      const uint32_t at = w < words ? off[m] + (uint32_t)w * 4u : kOutside;
      load_word_to_lds(r, off[m] == kOutside ? kOutside : at,
                       to + (uint32_t)(m * THREADS + wave * 64) * 4u);
    }
  }
  static __device__ __forceinline__ uint32_t at(const uint8_t* lds, int row, int w) {
    return *reinterpret_cast<const uint32_t*>(lds + (w * N + row) * 4);
  }
};

// ``steps`` stages in a ring of S places of ``bytes``: S - 1 on their way while one is
// multiplied.  load(number, place) issues exactly LOADS loads a wavefront, also past the end.
template <int S, int LOADS, typename L, typename F>
__device__ __forceinline__ void ring(int64_t steps, L&& load, F&& multiply) {
#pragma unroll
  for (int s = 0; s < S - 1; ++s) load(s, s);
  int now = 0;
  for (int64_t t = 0; t < steps; ++t) {
    const int next = now == 0 ? S - 1 : now - 1;
    wait_loads<(S - 2) * LOADS>();  // this stage is in LDS; the later ones may be on their way
    __syncthreads();
    load(t + S - 1, next);
    multiply(t, now);
    now = now + 1 == S ? 0 : now + 1;
  }
  wait_loads<0>();  // stages past the end
  __syncthreads();
}

// Codes and scales of N rows that lie ``pitch`` bytes apart (scales: ``words`` words).
struct Codes {
  const uint8_t *codes, *scales;
  int blocks, words;
  __device__ __forceinline__ Codes(const uint8_t* c, const uint8_t* s, int64_t row, int64_t length)
      : blocks(micro_blocks(length)), words(micro_filled(micro_blocks(length)) / 4) {
    codes = c + row * blocks * 16;
    scales = s + row * words * 4;
  }
};

// ---------------------------------------------------------------------------
// many rows
// ---------------------------------------------------------------------------

// A workgroup's BM x BN tile from rows of 16 bits (16-byte pieces at 16-byte addresses).
template <typename T, int BM, int BN, int WM, int WN, int S>
struct TileHalf {
  static constexpr int THREADS = WM * WN * 64, X = BM / WM / 32, Y = BN / WN / 32;
  using SA = PieceStage<BM, 8, THREADS>;  // a depth of 64
  using SB = PieceStage<BN, 2, THREADS>;
  using SC = ScaleStage<BN, 1, THREADS>;
  static constexpr int kStage = SA::kBytes + SB::kBytes + SC::kBytes;
  static constexpr int kLoads = SA::kMine + SB::kMine + SC::kMine;
  static constexpr int kLds = S * kStage > BM * BN * (int)sizeof(T) ? S * kStage
                                                                    : BM * BN * (int)sizeof(T);

  // a: m rows of ``inner`` elements, lda apart; b: n rows of codes
  static __device__ __forceinline__ void run(const T* a, int64_t lda, int m, int64_t inner,
                                             const Codes& b, int n, unsigned char* lds, T* c,
                                             int64_t ldc) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int wi = (wave / WN) * (BM / WM), wj = (wave % WN) * (BN / WN);
    F16x acc[X][Y];
#pragma unroll
    for (int x = 0; x < X; ++x)
#pragma unroll
      for (int y = 0; y < Y; ++y)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.0f;
    uint32_t off_a[SA::kMine], off_b[SB::kMine], off_c[SC::kMine];
    SA::offsets([&](int r) { return r < m ? (uint32_t)r * (uint32_t)lda * 2u : kOutside; }, off_a);
    SB::offsets([&](int r) { return r < n ? (uint32_t)r * (uint32_t)b.blocks * 16u : kOutside; }, off_b);
    SC::offsets([&](int r) { return r < n ? (uint32_t)r * (uint32_t)b.words * 4u : kOutside; }, off_c);
    const uint8_t *pa = reinterpret_cast<const uint8_t*>(uniform(a)), *pb = uniform(b.codes),
                  *pc = uniform(b.scales);
    const int64_t pieces = (inner + 7) / 8;
    const uint32_t base = lds_address(lds);
    ring<S, kLoads>(
        (inner + 63) / 64,
        [&](int64_t t, int at) {
          const uint32_t to = base + (uint32_t)(at * kStage);
          SA::load(pa + t * 128, off_a, pieces - 8 * t, to);
          SB::load(pb + t * 32, off_b, b.blocks - 2 * t, to + SA::kBytes);
          SC::load(pc, off_c, (int)(t >> 1), b.words, to + SA::kBytes + SB::kBytes);
        },
        [&](int64_t t, int at) {
          const uint8_t* la = lds + at * kStage;
          const uint8_t *lb = la + SA::kBytes, *lc = lb + SB::kBytes;
          I4 codes[Y];
          float scale[Y];
#pragma unroll
          for (int y = 0; y < Y; ++y) {
            const int row = wj + 32 * y + (lane & 31);
            codes[y] = SB::piece(lb, row, half);
            scale[y] = scale_of(SC::at(lc, row, 0), 2 * ((int)t & 1) + half);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            S8 fa[X], fb[Y];
#pragma unroll
            for (int x = 0; x < X; ++x)
              fa[x] = __builtin_bit_cast(S8, SA::piece(la, wi + 32 * x + (lane & 31), 4 * half + j));
#pragma unroll
            for (int y = 0; y < Y; ++y) fb[y] = numbers_of(T{}, (uint32_t)codes[y][j], scale[y]);
#pragma unroll
            for (int x = 0; x < X; ++x)
#pragma unroll
              for (int y = 0; y < Y; ++y) acc[x][y] = mma32(T{}, fb[y], fa[x], acc[x][y]);
          }
        });
    tile_out<T, T, BM, BN, WM, WN>(acc, lds, m, n, c, ldc);
  }
};

// A workgroup's BM x BN tile from packed rows; sums are written as C.
template <typename C, int BM, int BN, int WM, int WN, int S>
struct TileBoth {
  static constexpr int THREADS = WM * WN * 64, X = BM / WM / 32, Y = BN / WN / 32;
  using SA = PieceStage<BM, 8, THREADS>;  // a depth of 256
  using SB = PieceStage<BN, 8, THREADS>;
  using CA = ScaleStage<BM, 2, THREADS>;
  using CB = ScaleStage<BN, 2, THREADS>;
  static constexpr int kStage = SA::kBytes + SB::kBytes + CA::kBytes + CB::kBytes;
  static constexpr int kLoads = SA::kMine + SB::kMine + CA::kMine + CB::kMine;
  static constexpr int kOut = BM * BN * (int)sizeof(C);
  static constexpr int kLds = S * kStage > kOut ? S * kStage : kOut;

  static __device__ __forceinline__ void run(const Codes& a, int m, const Codes& b, int n,
                                             unsigned char* lds, C* c, int64_t ldc) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int wi = (wave / WN) * (BM / WM), wj = (wave % WN) * (BN / WN);
    F16x acc[X][Y];
#pragma unroll
    for (int x = 0; x < X; ++x)
#pragma unroll
      for (int y = 0; y < Y; ++y)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.0f;
    uint32_t off_a[SA::kMine], off_b[SB::kMine], off_ca[CA::kMine], off_cb[CB::kMine];
    const uint32_t pitch = (uint32_t)b.blocks * 16u, row_words = (uint32_t)b.words * 4u;
    SA::offsets([&](int r) { return r < m ? (uint32_t)r * pitch : kOutside; }, off_a);
    SB::offsets([&](int r) { return r < n ? (uint32_t)r * pitch : kOutside; }, off_b);
    CA::offsets([&](int r) { return r < m ? (uint32_t)r * row_words : kOutside; }, off_ca);
    CB::offsets([&](int r) { return r < n ? (uint32_t)r * row_words : kOutside; }, off_cb);
    const uint8_t *pa = uniform(a.codes), *pb = uniform(b.codes), *sa = uniform(a.scales),
                  *sb = uniform(b.scales);
    const uint32_t base = lds_address(lds);
    ring<S, kLoads>(
        (b.blocks + 7) / 8,
        [&](int64_t t, int at) {
          const uint32_t to = base + (uint32_t)(at * kStage);
          SA::load(pa + t * 128, off_a, b.blocks - 8 * t, to);
          SB::load(pb + t * 128, off_b, b.blocks - 8 * t, to + SA::kBytes);
          CA::load(sa, off_ca, (int)(2 * t), b.words, to + SA::kBytes + SB::kBytes);
          CB::load(sb, off_cb, (int)(2 * t), b.words, to + SA::kBytes + SB::kBytes + CA::kBytes);
        },
        [&](int64_t t, int at) {
          const uint8_t* la = lds + at * kStage;
          const uint8_t *lb = la + SA::kBytes, *ca = lb + SB::kBytes, *cb = ca + CA::kBytes;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            // the scales of blocks 4 q + half and 4 q + 2 + half in bytes 0 and 2
            int ka[X], kb[Y];
#pragma unroll
            for (int x = 0; x < X; ++x)
              ka[x] = (int)(CA::at(ca, wi + 32 * x + (lane & 31), q) >> (8 * half));
#pragma unroll
            for (int y = 0; y < Y; ++y)
              kb[y] = (int)(CB::at(cb, wj + 32 * y + (lane & 31), q) >> (8 * half));
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              I8 fa[X], fb[Y];
#pragma unroll
              for (int x = 0; x < X; ++x) {
                const I4 v = SA::piece(la, wi + 32 * x + (lane & 31), 4 * q + 2 * s + half);
                fa[x] = I8{v[0], v[1], v[2], v[3], 0, 0, 0, 0};
              }
#pragma unroll
              for (int y = 0; y < Y; ++y) {
                const I4 v = SB::piece(lb, wj + 32 * y + (lane & 31), 4 * q + 2 * s + half);
                fb[y] = I8{v[0], v[1], v[2], v[3], 0, 0, 0, 0};
              }
#pragma unroll
              for (int x = 0; x < X; ++x)
#pragma unroll
                for (int y = 0; y < Y; ++y)
                  acc[x][y] = s == 0 ? __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                                           fb[y], fa[x], acc[x][y], 4, 4, 0, kb[y], 0, ka[x])
                                     : __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                                           fb[y], fa[x], acc[x][y], 4, 4, 2, kb[y], 2, ka[x]);
            }
          }
        });
    tile_out<C, C, BM, BN, WM, WN>(acc, lds, m, n, c, ldc);
  }
};

// ---------------------------------------------------------------------------
// few rows
// ---------------------------------------------------------------------------

// The sums of BM rows and 64 columns over a contraction that the 4 wavefronts share, a quarter
// of every stage each: acc holds a wavefront's own part.  NA: the rows are the sum of that many
// arrays.  Rows of 16 bits: ``offset(row)`` bytes from the arrays' starts, or kOutside.
template <typename T, int BM, int NA, int S>
struct ThinPacked {
  static constexpr int THREADS = 256, X = BM / 32, Y = 2;
  using SA = PieceStage<BM, 32, THREADS>;  // a depth of 256
  using SB = PieceStage<64, 8, THREADS>;
  using SC = ScaleStage<64, 2, THREADS>;
  static constexpr int kStage = NA * SA::kBytes + SB::kBytes + SC::kBytes;
  static constexpr int kLoads = NA * SA::kMine + SB::kMine + SC::kMine;
  static constexpr int kRing = S * kStage;

  // from block ``first`` on ``blocks`` of them; ``row(j)``: the row of codes of column j, -1 for none
  template <typename FA, typename FB>
  static __device__ __forceinline__ void run(const T* const (&a)[NA], FA&& offset, int64_t inner,
                                             const Codes& b, FB&& row, int64_t first,
                                             int64_t blocks, unsigned char* lds,
                                             F16x (&acc)[X][Y]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    uint32_t off_a[SA::kMine], off_b[SB::kMine], off_c[SC::kMine];
    SA::offsets(offset, off_a);
    SB::offsets([&](int j) { const int r = row(j); return r < 0 ? kOutside : (uint32_t)r * (uint32_t)b.blocks * 16u; }, off_b);
    SC::offsets([&](int j) { const int r = row(j); return r < 0 ? kOutside : (uint32_t)r * (uint32_t)b.words * 4u; }, off_c);
    const uint8_t *pb = uniform(b.codes + first * 16), *pc = uniform(b.scales);
    const uint8_t* pa[NA];
#pragma unroll
    for (int i = 0; i < NA; ++i) pa[i] = reinterpret_cast<const uint8_t*>(uniform(a[i] + first * 32));
    const int64_t pieces = min((inner + 7) / 8 - first * 4, blocks * 4);
    const uint32_t base = lds_address(lds);
    ring<S, kLoads>(
        (blocks + 7) / 8,
        [&](int64_t t, int at) {
          const uint32_t to = base + (uint32_t)(at * kStage);
#pragma unroll
          for (int i = 0; i < NA; ++i)
            SA::load(pa[i] + t * 512, off_a, pieces - 32 * t, to + (uint32_t)(i * SA::kBytes));
          SB::load(pb + t * 128, off_b, blocks - 8 * t, to + (uint32_t)(NA * SA::kBytes));
          SC::load(pc, off_c, (int)(first / 4 + 2 * t), b.words,
                   to + (uint32_t)(NA * SA::kBytes + SB::kBytes));
        },
        [&](int64_t t, int at) {
          const uint8_t* la = lds + at * kStage;
          const uint8_t *lb = la + NA * SA::kBytes, *lc = lb + SB::kBytes;
          I4 codes[Y];
          float scale[Y];
#pragma unroll
          for (int y = 0; y < Y; ++y) {
            const int j = 32 * y + (lane & 31);
            codes[y] = SB::piece(lb, j, 2 * wave + half);
            scale[y] = scale_of(SC::at(lc, j, wave >> 1), 2 * (wave & 1) + half);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            S8 fb[Y];
#pragma unroll
            for (int y = 0; y < Y; ++y) fb[y] = numbers_of(T{}, (uint32_t)codes[y][j], scale[y]);
#pragma unroll
            for (int i = 0; i < NA; ++i)
#pragma unroll
              for (int x = 0; x < X; ++x) {
                const S8 fa = __builtin_bit_cast(
                    S8, SA::piece(la + i * SA::kBytes, 32 * x + (lane & 31), 8 * wave + 4 * half + j));
#pragma unroll
                for (int y = 0; y < Y; ++y) acc[x][y] = mma32(T{}, fb[y], fa, acc[x][y]);
              }
          }
        });
  }
};

// The wavefronts' parts of BM x 64 sums, in LDS: row i, column j of part w at thin_at(w, i, j).
constexpr int kThinPitch = 64 + 4;
template <int BM>
constexpr int kThinSums = 4 * BM * kThinPitch * 4;
template <int BM>
__device__ __forceinline__ void thin_parts(const F16x (&acc)[BM / 32][2], float* sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int x = 0; x < BM / 32; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        sums[(wave * BM + 32 * x + (lane & 31)) * kThinPitch + 32 * y + 2 * (r & ~3) +
             4 * (lane >> 5) + (r & 3)] = acc[x][y][r];
  __syncthreads();
}
// Their sum, in the wavefronts' order.
template <int BM>
__device__ __forceinline__ float thin_sum(const float* sums, int i, int j) {
  float s = sums[i * kThinPitch + j];
#pragma unroll
  for (int w = 1; w < 4; ++w) s += sums[(w * BM + i) * kThinPitch + j];
  return s;
}

// ---------------------------------------------------------------------------
// rows at any address
// ---------------------------------------------------------------------------

// Rows whose 16-byte pieces lie anywhere, to ones at 16 bytes, zeros behind their length.
template <typename T>
static __global__ __launch_bounds__(256) void k_align_rows(const T* __restrict__ a, int64_t lda,
                                                    int64_t inner, Divider by_row, uint32_t pieces,
                                                    int64_t first, T* __restrict__ out) {
  for (uint32_t n = blockIdx.x * 256 + threadIdx.x; n < pieces; n += gridDim.x * 256) {
    const uint32_t in = by_row.quotient(n);
    const int64_t row = first + in, l = (int64_t)(n - in * by_row.d) * 8;
    store16(out + row * by_row.d * 8 + l, load_upto(a + row * lda + l, inner - l));
  }
}

static int64_t whole256(int64_t n) { return (n + 255) / 256 * 256; }
// Bytes of rows that are aligned for the loads.
static int64_t aligned_bytes(int64_t rows, int64_t inner) {
  return whole256(rows * ((inner + 7) / 8) * 16);
}

template <typename T>
static int align_rows(hipStream_t st, const T* a, int64_t lda, int64_t rows, int64_t inner, T* out) {
  const int64_t per = (inner + 7) / 8, most = ((int64_t(1) << 30) - 1) / per;
  const Divider by((uint32_t)per);
  for (int64_t first = 0; first < rows; first += most) {
    const uint32_t pieces = (uint32_t)(std::min(most, rows - first) * per);
    k_align_rows<T><<<grid_of(pieces, 256), dim3(256), 0, st>>>(a, lda, inner, by, pieces, first, out);
    if (int rc = launched("k_align_rows")) return rc;
  }
  return PURIN_CP_OK;
}

}  // namespace train
}  // namespace purin
