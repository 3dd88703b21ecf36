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

#include <type_traits>

#include "expert16.hpp"
#include "micro.hpp"

namespace purin {
namespace train {

typedef int I4 __attribute__((ext_vector_type(4)));
typedef int I8 __attribute__((ext_vector_type(8)));
typedef float F4 __attribute__((ext_vector_type(4)));

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

// A stage of N rows, PIECES pieces of 16 bytes each, in LDS [row][piece].  The pieces of the rows
// that cover the banks together (256 bytes) are exchanged by those rows' number, so that a read of
// one piece from any 16 rows of 16 such sets, as the hardware takes them, falls on different banks.
template <int N, int PIECES, int THREADS>
struct PieceStage {
  static constexpr int kMine = N * PIECES / THREADS;
  static constexpr int kBytes = N * PIECES * 16;
  static_assert(N * PIECES % THREADS == 0, "whole pieces per thread");

  static_assert(PIECES <= 16, "a row is no longer than the banks");
  static __device__ __forceinline__ int place(int row, int piece) {
    return row * PIECES + (piece ^ ((row * PIECES / 16) & (PIECES - 1)));
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

// The scales of N rows for 32 blocks (four stages of 256) at a time, two pieces of 16 bytes a row, in
// LDS [piece][row]; two such chunks.  A load of scales takes a line of the cache a row, however
// little of it is wanted: with a word of four blocks for each half stage the scales brought as much
// from L2 to L1 as the codes.  Rows have whole pieces (words % 4 == 0).
template <int N, int THREADS>
struct ScaleChunks {
  static constexpr int kBytes = 2 * N * 32;
  static_assert(N % THREADS == 0 || THREADS % N == 0, "whole rows per load");
  static constexpr int kMine = N / THREADS > 0 ? N / THREADS : 1;

  template <typename F>
  static __device__ __forceinline__ void offsets(F&& offset, uint32_t (&off)[kMine]) {
#pragma unroll
    for (int m = 0; m < kMine; ++m) off[m] = offset((m * THREADS + (int)threadIdx.x) % N);
  }
  // piece number 2 ``chunk`` + ``piece`` of the rows, of ``pieces``
  static __device__ __forceinline__ void load(const uint8_t* p, const uint32_t (&off)[kMine], int chunk,
                                              int piece, int pieces, uint32_t lds) {
    const U4 r = buffer_at(p);
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int at = 2 * chunk + piece;
    const uint32_t to = lds + (uint32_t)((chunk & 1) * N * 32 + piece * N * 16);
#pragma unroll
    for (int m = 0; m < kMine; ++m)
      if (N >= THREADS || wave * 64 < N)
        load_to_lds(r, at < pieces && off[m] != kOutside ? off[m] + (uint32_t)at * 16u : kOutside,
                    to + (uint32_t)(m * THREADS + wave * 64) * 16u);
  }
  // the two words of stage ``t``
  static __device__ __forceinline__ uint2 at(const uint8_t* lds, int row, int64_t t) {
    return *reinterpret_cast<const uint2*>(lds + (((int)t >> 2) & 1) * N * 32 +
                                           (((int)t & 3) >> 1) * N * 16 + row * 16 + ((int)t & 1) * 8);
  }
};

// ``steps`` stages in a ring of S places of ``bytes``: S - 1 on their way while one is
// multiplied.  load(number, place) issues exactly LOADS loads a wavefront, also past the end (more
// in some stages only make the waits longer).
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
  __device__ __forceinline__ int lines() const { return (blocks + 7) / 8; }
  __device__ __forceinline__ Codes(const uint8_t* c, const uint8_t* s, int64_t row, int64_t length)
      : blocks(micro_blocks(length)), words(micro_filled(micro_blocks(length)) / 4) {
    codes = c + row * blocks * 16;
    scales = s + row * words * 4;
  }
};

// ---------------------------------------------------------------------------
// many rows
// ---------------------------------------------------------------------------

// A workgroup's B x B tile from rows of 16 bits (16-byte pieces at 16-byte addresses), in three
// stages of 64.  Bound by the matrix units as the product of dense weights is, whose time it has with
// half the bytes read: 32768 rows, 16 experts, 2048 x 4096, 256 x 256 tiles: 522-570 us, 0.96-1.05
// PFLOP/s; the units are busy 48 % of the time, 58 % of what the CUs are.
template <typename T, int B, int WN>
struct TileHalf {
  static constexpr int BM = B, BN = B, WM = 2, S = 3;
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

// A workgroup's B x B tile from packed rows; sums are written as C.  CHUNKS: scales by
// ScaleChunks, for rows that have whole pieces of them.  Two stages of 256 (of 128 in four places
// the half lines cost more than the deeper ring gives: 32768 rows, 16 experts, 2048 x 4096 233 us,
// 248).  256 x 256 tiles: 128 x 256 and 128 x 128 ones, two workgroups a CU, read more from L2 than
// their overlap gives (320, 290).  201-245 us in all: 75 of them each tile's first stages and its way
// out (268 MB), in which its CU, with room for one workgroup, multiplies nothing; the contraction
// itself runs at 3.6 PFLOP/s.
template <typename C, int B, int WN, bool CHUNKS>
struct TileBoth {
  static constexpr int BM = B, BN = B, WM = 2;
  static constexpr int THREADS = WM * WN * 64, X = BM / WM / 32, Y = BN / WN / 32;
  using SA = PieceStage<BM, 8, THREADS>;  // a depth of 256
  using SB = PieceStage<BN, 8, THREADS>;
  using CA = std::conditional_t<CHUNKS, ScaleChunks<BM, THREADS>, ScaleStage<BM, 2, THREADS>>;
  using CB = std::conditional_t<CHUNKS, ScaleChunks<BN, THREADS>, ScaleStage<BN, 2, THREADS>>;
  static constexpr int kScales = CA::kBytes + CB::kBytes;
  static constexpr int kStage = SA::kBytes + SB::kBytes + (CHUNKS ? 0 : kScales);
  static constexpr int kOut = BM * BN * (int)sizeof(C);
  static constexpr int kRing = 2 * kStage + (CHUNKS ? kScales : 0);
  static constexpr int kLds = kRing > kOut ? kRing : kOut;

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
    auto load_chunk = [&](int chunk, int piece) {
      if constexpr (CHUNKS) {
        CA::load(sa, off_ca, chunk, piece, b.words / 4, base + 2 * kStage);
        CB::load(sb, off_cb, chunk, piece, b.words / 4, base + 2 * kStage + CA::kBytes);
      }
    };
    load_chunk(0, 0);
    load_chunk(0, 1);
    ring<2, 0>(
        (b.blocks + 7) / 8,
        [&](int64_t t, int at) {
          const uint32_t to = base + (uint32_t)(at * kStage);
          SA::load(pa + t * 128, off_a, b.blocks - 8 * t, to);
          SB::load(pb + t * 128, off_b, b.blocks - 8 * t, to + SA::kBytes);
          if constexpr (CHUNKS) {
            // the next chunk's, whose place the last chunk but one has left
            if ((t & 3) >= 2) load_chunk((int)(t >> 2) + 1, (int)(t & 1));
          } else {
            CA::load(sa, off_ca, (int)(2 * t), b.words, to + SA::kBytes + SB::kBytes);
            CB::load(sb, off_cb, (int)(2 * t), b.words, to + SA::kBytes + SB::kBytes + CA::kBytes);
          }
        },
        [&](int64_t t, int at) {
          const uint8_t* la = lds + at * kStage;
          const uint8_t* lb = la + SA::kBytes;
          const uint8_t* ca = CHUNKS ? lds + 2 * kStage : lb + SB::kBytes;
          const uint8_t* cb = ca + CA::kBytes;
          auto words = [&](auto side, const uint8_t* from, int row) {
            using S = decltype(side);
            if constexpr (CHUNKS) return S::at(from, row, t);
            else return uint2{S::at(from, row, 0), S::at(from, row, 1)};
          };
          uint2 wa[X], wb[Y];
#pragma unroll
          for (int x = 0; x < X; ++x) wa[x] = words(CA{}, ca, wi + 32 * x + (lane & 31));
#pragma unroll
          for (int y = 0; y < Y; ++y) wb[y] = words(CB{}, cb, wj + 32 * y + (lane & 31));
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            // the scales of blocks 4 q + half and 4 q + 2 + half in bytes 0 and 2
            int ka[X], kb[Y];
#pragma unroll
            for (int x = 0; x < X; ++x) ka[x] = (int)((q ? wa[x].y : wa[x].x) >> (8 * half));
#pragma unroll
            for (int y = 0; y < Y; ++y) kb[y] = (int)((q ? wb[y].y : wb[y].x) >> (8 * half));
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

// The sums of BM rows and 64 columns to a wavefront.  A workgroup's four have parts of one
// contraction, or of two, or each columns of its own (``parts`` = 4, 2, 1): the fewer parts, the
// longer the streams, and the more the wavefronts share of the rows.  Every weight is used by one
// wavefront, once: it loads 128 bytes of 64 columns at a time, whole lines by 8 neighbouring lanes,
// keeps two such loads on their way in registers, and brings the pieces to the lanes that multiply
// them by way of 8 KB of LDS of its own.  No wavefront waits for another, and the many in flight
// hide each other.  (Loads straight to the lanes that multiply them take a cycle a lane: 64 experts,
// 4096 x 2816 in 4 bits 112 us.)
// NA: the rows are the sum of that many arrays.

// Rows of 16 bits in pieces of 8: piece k of row r at p + k * step + r * pitch bytes.  A load of
// one piece of 16 rows takes a cycle a row where each is in one piece (step 16), and one for four
// where rows lie side by side (pitch 16).
struct Rows {
  const void* p;
  uint32_t step, pitch;
};
// Two times 32 columns of a tile: starts and how many are there.
struct Columns {
  int64_t first[2];
  int n[2];
};

using Buffer = __amdgpu_buffer_rsrc_t;
__device__ __forceinline__ Buffer buffer_of(const void* p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, 0x7ffffff0, 0x00020000);
}
__device__ __forceinline__ I4 load_piece(Buffer b, uint32_t at, uint32_t uniform_at) {
  return __builtin_bit_cast(I4, __builtin_amdgcn_raw_buffer_load_b128(b, (int)at, (int)uniform_at, 0));
}

__device__ __forceinline__ F4 mma16(bf16, S8 a, S8 b, F4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(B8, a),
                                                 __builtin_bit_cast(B8, b), c, 0, 0, 0);
}
__device__ __forceinline__ F4 mma16(f16, S8 a, S8 b, F4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(H8, a),
                                                __builtin_bit_cast(H8, b), c, 0, 0, 0);
}

// A wavefront's sums: rows 16 x + lane % 16, columns 16 y + 4 (lane / 16) + r.
template <int BM>
struct ThinAcc {
  static constexpr int X = BM / 16;
  F4 v[X][4];
  __device__ __forceinline__ ThinAcc() {
#pragma unroll
    for (int x = 0; x < X; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y) v[x][y] = F4{0, 0, 0, 0};
  }
};

// The wavefronts' BM x 64 sums, in LDS.
constexpr int kThinPitch = 64 + 4;
template <int BM>
constexpr int kThinSums = 4 * BM * kThinPitch * 4;
template <int BM>
__device__ __forceinline__ void thin_parts(const ThinAcc<BM>& acc, float* sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int x = 0; x < BM / 16; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y)
      *reinterpret_cast<F4*>(sums + (wave * BM + 16 * x + (lane & 15)) * kThinPitch + 16 * y +
                             4 * (lane >> 4)) = acc.v[x][y];
  __syncthreads();
}
// Row i, column j (64 to each set of ``parts`` wavefronts): the parts' sum, in their order.
template <int BM>
__device__ __forceinline__ float thin_sum(const float* sums, int parts, int i, int j) {
  const float* at = sums + ((j >> 6) * parts * BM + i) * kThinPitch + (j & 63);
  float s = at[0];
  for (int w = 1; w < parts; ++w) s += at[w * BM * kThinPitch];
  return s;
}

// A lane's rows (16 x + lane % 16 of the tile), and the pieces of them that it multiplies in a
// unit of ``PIECES`` (LANE apart for the lane groups, INSIDE for its own).
template <int X, int NA, int PIECES, int LANE, int INSIDE>
struct RowStream {
  const uint8_t* p[NA];
  uint32_t step, at[X];
  int left;  // pieces from this lane's first on

  // ``row(i)``: the row of tile row i, -1 for none.  ``pieces``: those of the rows up to the end of
  // the wavefront's part.  The loops go on to an even number of lines, with weights of zero, and a
  // row's elements there are the next part's: an infinity among them, times zero, would be NaN.
  template <typename F>
  __device__ __forceinline__ RowStream(const Rows (&a)[NA], F&& row, int pieces)
      : step(a[0].step) {
    const int lane = threadIdx.x & 63, group = lane >> 4;
#pragma unroll
    for (int i = 0; i < NA; ++i) p[i] = uniform((const uint8_t*)a[i].p);
#pragma unroll
    for (int x = 0; x < X; ++x) {
      const int r = row(16 * x + (lane & 15));
      at[x] = r < 0 ? kOutside : (uint32_t)r * a[0].pitch + (uint32_t)(group * LANE) * step;
    }
    left = pieces - group * LANE;
  }
  __device__ __forceinline__ I4 load(int i, int x, int unit, int k) const {
    const bool in = unit * PIECES + k * INSIDE < left;
    return load_piece(buffer_of(p[i] + (int64_t)unit * PIECES * step), in ? at[x] : kOutside,
                      (uint32_t)(k * INSIDE) * step);
  }
};

// Parts of a contraction for a number of 64-column streams of it.  us with 1 | 2 | 4: a layer of one
// token, 8 experts (352 and 256 streams) 62 | 49 | 47; of 64 tokens, 64 experts in 4 bits (2816 and
// 4096) 194 | 190 | 206.  Products in 4 bits, one row to an expert, 2560 columns, contractions of 4096,
// then of 1408:
//   streams      1040              1600              2560              3200              4160              5120
//   4096   44 | 44 | 42      59 | 55 | 57      83 | 75 | 80    100 | 97 | 103   129 | 122 | 132   138 | 139 | 156
//   1408   24 | 24 | 26      32 | 30 | 35      37 | 39 | 48      46 | 51 | 61      57 | 65 | 78      61 | 73 | 92
// Layers of 16 tokens, dense, 4096 long: 4 from 176 streams (63 | 43 | 38) to 1408 (178 | 169 | 153), equal
// from 2048 on (214 | 211 | 208).  The turns lie between the long contractions' and the short ones'.
inline int stream_parts(int64_t streams) { return streams >= 4096 ? 1 : streams >= 1536 ? 2 : 4; }
// A part of the lines ``first`` to ``end``.
__device__ __forceinline__ void share_lines(int first, int end, int part, int parts, int& from,
                                            int& to) {
  const int per = (max(end - first, 0) + parts - 1) / parts;
  from = min(end, first + part * per);
  to = min(end, from + per);
}

// 64 columns' lines of 128 bytes, in two runs of 32 columns, on their way to the wavefront's LDS:
// [column][piece], the pieces exchanged by the column's number.
struct LineStream {
  const uint8_t* p[2];
  uint32_t at;          // this lane's piece of column lane / 8; eight columns are ``step`` bytes
  int step, pieces;     // pieces of 16 bytes, in a column
  int n[2];
  I4 v[2][8];

  __device__ __forceinline__ LineStream(const uint8_t* first, const uint8_t* second, const Columns& c,
                                        int pitch, int count)
      : step(8 * pitch), pieces(count) {
    const int lane = threadIdx.x & 63;
    p[0] = uniform(first);
    p[1] = uniform(second);
    at = (uint32_t)((lane >> 3) * pitch + (lane & 7) * 16);
    n[0] = c.n[0];
    n[1] = c.n[1];
  }
  // line number ``line`` of the columns; from ``to`` on none
  __device__ __forceinline__ void load(int slot, int line, int to) {
    const int lane = threadIdx.x & 63;
    // a column past all of them where the line, or the lane's piece of it, is not there
    const int j = line < to && 8 * line + (lane & 7) < pieces ? lane >> 3 : 64;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[slot][i] = load_piece(buffer_of(p[i >> 2] + (int64_t)line * 128),
                              j + 8 * (i & 3) < n[i >> 2] ? at : kOutside,
                              (uint32_t)(step * (i & 3)));
  }
  __device__ __forceinline__ void store(int slot, uint8_t* lds) const {
    const int lane = threadIdx.x & 63;
    // columns 8 i + lane / 8 have the number lane / 8 in their eight
    uint8_t* to = lds + (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) *reinterpret_cast<I4*>(to + i * 1024) = v[slot][i];
    __builtin_amdgcn_wave_barrier();  // in order within a wavefront; for the compiler
  }
  // piece ``k`` of column 16 y + lane % 16
  static __device__ __forceinline__ I4 piece(const uint8_t* lds, int y, int k) {
    const int j = (threadIdx.x & 15);
    return *reinterpret_cast<const I4*>(lds + (16 * y + j) * 128 + ((k ^ (j & 7)) << 4));
  }
};
constexpr int kLineLds = 4 * 8192;  // a workgroup's

// Microscaled weights: a line is eight blocks, four at a time to the lane groups.  Scales are
// loaded for two lines at once: a load of them takes a line of the cache a column.
template <typename T, int BM, int NA>
struct StreamCodes {
  static constexpr int X = BM / 16;

  // lines ``from`` to ``to``
  template <typename F>
  static __device__ __forceinline__ void run(const Rows (&a)[NA], F&& row, int64_t inner,
                                             const Codes& b, const Columns& c, int from, int to,
                                             uint8_t* lds, ThinAcc<BM>& acc) {
    const int lane = threadIdx.x & 63, group = lane >> 4;
    lds += (threadIdx.x >> 6) * 8192;
    LineStream lines(b.codes + c.first[0] * b.blocks * 16, b.codes + c.first[1] * b.blocks * 16, c,
                     b.blocks * 16, b.blocks);
    // the scales of column 16 y + lane % 16
    const int words = b.words * 4;
    const uint8_t* ps[2] = {uniform(b.scales + c.first[0] * words), uniform(b.scales + c.first[1] * words)};
    uint32_t at_scale[4];
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int j = 16 * (y & 1) + (lane & 15);
      at_scale[y] = j < c.n[y >> 1] ? (uint32_t)(j * words) : kOutside;
    }
    I4 scales_next[4], rows_now[NA][X][4];
    uint32_t scales[4];  // the lane group's of the four units
    // the words of two lines, of which the last row's may end the memory: only those that are there
    auto load_scales = [&](int line) {
      if (line < to && 2 * line + 4 <= b.words) {
#pragma unroll
        for (int y = 0; y < 4; ++y)
          scales_next[y] = load_piece(buffer_of(ps[y >> 1] + line * 8), at_scale[y], 0);
      } else {
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            scales_next[y][k] =
                line < to && 2 * line + k < b.words
                    ? (int)__builtin_amdgcn_raw_buffer_load_b32(buffer_of(ps[y >> 1] + line * 8 + k * 4),
                                                                (int)at_scale[y], 0, 0)
                    : 0;
      }
    };
    load_scales(from);
    lines.load(0, from, to);
    lines.load(1, from + 1, to);
    const RowStream<X, NA, 16, 4, 1> rows(a, row, min((int)((inner + 7) / 8), 32 * to));
    auto load_rows = [&](int j, int unit) {
#pragma unroll
      for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int x = 0; x < X; ++x) rows_now[i][x][j] = rows.load(i, x, unit, j);
    };
#pragma unroll
    for (int j = 0; j < 4; ++j) load_rows(j, 2 * from);
    for (int t = from; t < to; t += 2) {
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        scales[y] = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u)  // past the end the codes are zero, and the words another column's
          if (2 * t + u < 2 * to)
            scales[y] |= (((uint32_t)scales_next[y][u] >> (8 * group)) & 255u) << (8 * u);
      }
      load_scales(t + 2);
#pragma unroll
      for (int s = 0; s < 2; ++s) {  // past the end: zeros
        lines.store(s, lds);
        lines.load(s, t + s + 2, to);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          I4 codes[4];
          float by[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            codes[y] = LineStream::piece(lds, y, 4 * u + group);
            by[y] = scale_of(scales[y], 2 * s + u);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            S8 fb[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) fb[y] = numbers_of(T{}, (uint32_t)codes[y][j], by[y]);
#pragma unroll
            for (int i = 0; i < NA; ++i)
#pragma unroll
              for (int x = 0; x < X; ++x) {
                const S8 fa = __builtin_bit_cast(S8, rows_now[i][x][j]);
#pragma unroll
                for (int y = 0; y < 4; ++y) acc.v[x][y] = mma16(T{}, fb[y], fa, acc.v[x][y]);
              }
            load_rows(j, 2 * (t + s) + u + 1);
          }
        }
        __builtin_amdgcn_wave_barrier();
      }
    }
  }
};

// Dense weights whose contraction is contiguous (``ld`` elements apart, 16-byte pieces at 16-byte
// addresses): a line is 64 of it.
template <typename T, int BM, int NA>
struct StreamDense {
  static constexpr int X = BM / 16;

  template <typename F>
  static __device__ __forceinline__ void run(const Rows (&a)[NA], F&& row, int64_t inner,
                                             const T* w, int64_t ld, const Columns& c, int from, int to,
                                             uint8_t* lds, ThinAcc<BM>& acc) {
    const int lane = threadIdx.x & 63, group = lane >> 4;
    lds += (threadIdx.x >> 6) * 8192;
    const int pieces = (int)((inner + 7) / 8);
    LineStream lines((const uint8_t*)(w + c.first[0] * ld), (const uint8_t*)(w + c.first[1] * ld), c,
                     (int)ld * 2, pieces);
    lines.load(0, from, to);
    lines.load(1, from + 1, to);
    const RowStream<X, NA, 8, 1, 4> rows(a, row, min(pieces, 8 * to));
    I4 rows_now[NA][X][2];
    auto load_rows = [&](int j, int unit) {
#pragma unroll
      for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int x = 0; x < X; ++x) rows_now[i][x][j] = rows.load(i, x, unit, j);
    };
#pragma unroll
    for (int j = 0; j < 2; ++j) load_rows(j, from);
    for (int t = from; t < to; t += 2) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {  // past the end: zeros
        lines.store(s, lds);
        lines.load(s, t + s + 2, to);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          S8 fb[4];
#pragma unroll
          for (int y = 0; y < 4; ++y)
            fb[y] = __builtin_bit_cast(S8, LineStream::piece(lds, y, 4 * j + group));
#pragma unroll
          for (int i = 0; i < NA; ++i)
#pragma unroll
            for (int x = 0; x < X; ++x) {
              const S8 fa = __builtin_bit_cast(S8, rows_now[i][x][j]);
#pragma unroll
              for (int y = 0; y < 4; ++y) acc.v[x][y] = mma16(T{}, fb[y], fa, acc.v[x][y]);
            }
          load_rows(j, t + s + 1);
        }
        __builtin_amdgcn_wave_barrier();
      }
    }
  }
};

// ---------------------------------------------------------------------------
// rows at any address
// ---------------------------------------------------------------------------

// Rows at any address to whole pieces of 8 elements, zeros behind their length.
template <typename T>
__device__ __forceinline__ void align_piece(const T* a, int64_t lda, int64_t inner, int64_t row,
                                            int64_t piece, T* out) {
  store16(out + (row * ((inner + 7) / 8) + piece) * 8,
          load_upto(a + row * lda + piece * 8, inner - piece * 8));
}
template <typename T>
static __global__ __launch_bounds__(256) void k_align_rows(const T* __restrict__ a, int64_t lda,
                                                           int64_t inner, Divider by,
                                                           uint32_t pieces, int64_t first,
                                                           T* __restrict__ out) {
  for (uint32_t n = blockIdx.x * 256 + threadIdx.x; n < pieces; n += gridDim.x * 256) {
    const uint32_t q = by.quotient(n);
    align_piece(a, lda, inner, first + q, n - q * by.d, out);
  }
}

// The same side by side: piece k of row r at out + (k * rows + r) * 16 bytes.  A workgroup turns 32
// rows by 16 pieces, through LDS: small tiles, so that few rows fill the card (768 rows of 4096:
// 64 by 32 7.7 us).
template <typename T>
static __global__ __launch_bounds__(256) void k_turn_rows(const T* __restrict__ a, int64_t lda,
                                                          int64_t inner, int64_t rows,
                                                          int64_t tiles, uint8_t* __restrict__ out) {
  __shared__ __align__(16) uint8_t lds[32 * 16 * 16];
  const int64_t pieces = (inner + 7) / 8;
  const int64_t row = blockIdx.x / tiles * 32, piece = blockIdx.x % tiles * 16;
#pragma unroll
  for (int i = threadIdx.x; i < 32 * 16; i += 256) {
    const int r = i >> 4, k = i & 15;
    if (row + r < rows && piece + k < pieces)
      *reinterpret_cast<S8*>(lds + (r * 16 + (k ^ (r & 15))) * 16) = __builtin_bit_cast(
          S8, load_upto(a + (row + r) * lda + (piece + k) * 8, inner - (piece + k) * 8));
  }
  __syncthreads();
#pragma unroll
  for (int i = threadIdx.x; i < 32 * 16; i += 256) {
    const int k = i >> 5, r = i & 31;
    if (row + r < rows && piece + k < pieces)
      *reinterpret_cast<S8*>(out + ((piece + k) * rows + row + r) * 16) =
          *reinterpret_cast<const S8*>(lds + (r * 16 + (k ^ (r & 15))) * 16);
  }
}

static int64_t whole256(int64_t n) { return (n + 255) / 256 * 256; }
// Bytes of rows that are aligned for the loads.
static int64_t aligned_bytes(int64_t rows, int64_t inner) {
  return whole256(rows * ((inner + 7) / 8) * 16);
}

template <typename T>
static int align_rows(hipStream_t st, const T* a, int64_t lda, int64_t rows, int64_t inner,
                      void* out) {
  const int64_t per = (inner + 7) / 8, most = ((int64_t(1) << 30) - 1) / per;
  const Divider by((uint32_t)per);
  for (int64_t first = 0; first < rows; first += most) {
    const uint32_t pieces = (uint32_t)(std::min(most, rows - first) * per);
    k_align_rows<T><<<grid_of(pieces, 256), dim3(256), 0, st>>>(a, lda, inner, by, pieces, first,
                                                                (T*)out);
    if (int rc = launched("k_align_rows")) return rc;
  }
  return PURIN_CP_OK;
}

template <typename T>
static int turn_rows(hipStream_t st, const T* a, int64_t lda, int64_t rows, int64_t inner, void* out) {
  const int64_t tiles = (inner + 127) / 128, groups = (rows + 31) / 32 * tiles;
  if (groups >= (int64_t(1) << 24))  // fewer than 2^32 threads
    return set_error(PURIN_CP_ERR_UNSUPPORTED, "too many tiles for a launch");
  k_turn_rows<T><<<dim3((unsigned)groups), dim3(256), 0, st>>>(a, lda, inner, rows, tiles, (uint8_t*)out);
  return launched("k_turn_rows");
}

}  // namespace train
}  // namespace purin
