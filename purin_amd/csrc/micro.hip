// Microscaled numbers and the activation between the experts' products (include/purin_train.h:
// pack, unpack, activate, activate_vjp).
//
// 32 neighbours share a power of two 2^s, s from the largest magnitude m among them:
//   4 bits   s = max(floor(log2 m) - 2, -127), element = the nearest of 0 .5 1 1.5 2 3 4 6 (and
//            their negatives) to x / 2^s, ties to the even code, at most 6
//   8 bits   s = max(floor(log2 m), -127), element = x / 2^s in 64ths, to the nearest (ties to
//            even), at most 127
// The scale is held as s + 127, 255 where a neighbour is infinite or NaN (then all 32 are NaN).
// Scaling by powers of two is exact, so an element is rounded once, and both kinds are exact again
// in the type that they came from: four or seven bits beside a power of two not below the one
// that the type itself has there.
//
// All are bound by memory: a thread has 8 neighbours, 4 threads a block, whose largest magnitude
// passes between them without LDS.  Read and written, us and TB/s: 32768 x 2048 bf16 to 4 bits 35
// (4.8); 4099 x 1111 float32 to 8 bits 7 and back 7.5 (3.2, 3.0); 16 x 4096 x 2048 bf16 to 4 bits
// across memory 86-90 (3.8-3.9) and back 58 (5.8, the codes in the cache); the gated activation of
// 49152 x 2816 bf16 with kept rows 94-98, backward 93-97 (5.7-6.0, part of them in the cache), without
// 73-76 and 113-117 (5.5, 6.0).  gelu is bound by its share of a normal distribution, a 32-bit erfcf for
// 16-bit results too: 4099 x 777 float16 10.5 both ways, silu 7 and 6.

#include <algorithm>
#include <type_traits>

#include "micro.hpp"
#include "train.hpp"

namespace purin {
namespace train {

// 8 neighbours as they are in memory; ``n`` of them are there, zeros behind.  They become numbers
// behind the branch, so that several loads are on their way before the first is waited for.
template <typename T>
struct Eight {
  static constexpr int kWords = 8 * sizeof(T) / 4;
  typedef uint32_t Words __attribute__((ext_vector_type(kWords)));
  Words w;
  __device__ __forceinline__ Eight() = default;
  __device__ __forceinline__ Eight(const T* p, int n) {
    constexpr int V = kVec<T>;
    struct All {
      Pack<T> v[8 / V];
    } all;
    if (n >= 8) {
#pragma unroll
      for (int i = 0; i < 8; i += V) all.v[i / V] = load16(p + i);
      w = __builtin_bit_cast(Words, all);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) all.v[i / V].v[i % V] = i < n ? p[i] : (T)0;
      w = __builtin_bit_cast(Words, all);
      asm("" : "+v"(w));  // whole words for both: halves would be taken apart, and waited for, above
    }
  }
  __device__ __forceinline__ typename Elem<T>::Acc operator[](int i) const {
    struct All {
      T v[8];
    };
    return (typename Elem<T>::Acc)__builtin_bit_cast(All, w).v[i];
  }
};
template <typename T>
__device__ __forceinline__ void store8(T* p, int n, const typename Elem<T>::Acc (&v)[8]) {
  constexpr int V = kVec<T>;
  if (n >= 8) {
#pragma unroll
    for (int i = 0; i < 8; i += V) {
      Pack<T> x;
#pragma unroll
      for (int q = 0; q < V; ++q) x.v[q] = (T)v[i + q];
      store16(p + i, x);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (T)v[i];
  }
}

// ---------------------------------------------------------------------------
// to few bits
// ---------------------------------------------------------------------------

// The rows of a tensor (groups, rows, length), its blocks along length.
template <typename T>
struct Strided {
  const T* p;
  int64_t groups, rows, length;
  int64_t sg, sr, sl;
};

// Rows whose neighbours are adjacent.  Thread number n of a group's rows has part n % 4 of block
// n / 4; the scales' blocks are counted, behind the row's last one are only they.
template <typename T, int KIND>
__global__ __launch_bounds__(256) void k_pack(Strided<T> x, Divider by_row, uint32_t pieces,
                                              int64_t first, uint8_t* __restrict__ codes,
                                              uint8_t* __restrict__ scales) {
  const int blocks = micro_blocks(x.length), filled = micro_filled(blocks);
  for (int64_t g = blockIdx.y; g < x.groups; g += gridDim.y)
    for (uint32_t n = blockIdx.x * 256 + threadIdx.x; n < pieces; n += gridDim.x * 256) {
      const uint32_t in = by_row.quotient(n);
      const int at = (int)(n - in * by_row.d), block = at >> 2;
      const int64_t row = first + in, out = g * x.rows + row;
      const int64_t l = (int64_t)at * 8;
      const Eight<T> raw(x.p + g * x.sg + row * x.sr + l,
                         (int)max<int64_t>(0, min<int64_t>(8, x.length - l)));
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = raw[i];
      uint32_t most = magnitude(v[0]);
#pragma unroll
      for (int i = 1; i < 8; ++i) most = max(most, magnitude(v[i]));
      most = quad_max(most);
      const uint32_t s = micro_scale<KIND>(most);
      if ((at & 3) == 0) scales[out * filled + block] = (uint8_t)s;
      if (block < blocks) store_codes<KIND>(codes + (out * blocks * 32 + l) * kMicroBits<KIND> / 8, v, s);
    }
}

// Rows that are adjacent themselves, 8 to a thread, whose neighbours are sl apart: a workgroup
// has 64 rows and 8 blocks, and its codes pass through LDS, so that a row's leave together.
// Neighbouring workgroups have neighbouring rows (the other order: 90 us for 88).
constexpr int kAcross = 64;
template <typename T, int KIND>
__global__ __launch_bounds__(256) void k_pack_across(Strided<T> x, int64_t tiles_r,
                                                     uint8_t* __restrict__ codes,
                                                     uint8_t* __restrict__ scales) {
  constexpr int kRow = 8 * 32 * kMicroBits<KIND> / 8, kPieces = kRow / 16;  // bytes, pieces of 16
  // row 8 a + r at place 8 r + a, its pieces exchanged by a: a wavefront writes 8 places, two blocks
  // of each, and these fall on different banks
  __shared__ __align__(16) uint8_t held[kAcross * kRow];
  auto place = [](int a, int r, int piece) {
    return ((8 * r + a) * kPieces + (piece ^ (KIND == kFp4 ? a & 6 : 2 * a))) * 16;
  };
  __shared__ uint8_t held_scales[kAcross][8];
  const int blocks = micro_blocks(x.length), filled = micro_filled(blocks);
  // lanes: 8 times 8 rows, then the 4 quarters of a block, then the blocks
  const int tid = threadIdx.x, r8 = tid & 7, quarter = (tid >> 3) & 3, block = tid >> 5;
  const int64_t tl = blockIdx.x / tiles_r, tr = blockIdx.x - tl * tiles_r;
  const int64_t row = tr * kAcross, l = (tl * 8 + block) * 32 + quarter * 8;
  const int n = (int)max<int64_t>(0, min<int64_t>(8, x.rows - row - r8 * 8));
  for (int64_t g = blockIdx.y; g < x.groups; g += gridDim.y) {
    Eight<T> v[8];  // [neighbour][row]
    const T* p = x.p + g * x.sg + row + r8 * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = Eight<T>(p + (l + j) * x.sl, l + j < x.length ? n : 0);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      uint32_t most = magnitude(v[0][r]);
#pragma unroll
      for (int j = 1; j < 8; ++j) most = max(most, magnitude(v[j][r]));
      most = max(most, (uint32_t)__shfl_xor((int)most, 8, 64));
      most = max(most, (uint32_t)__shfl_xor((int)most, 16, 64));
      const uint32_t s = micro_scale<KIND>(most);
      float one[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) one[j] = v[j][r];
      const int in = (block * 32 + quarter * 8) * kMicroBits<KIND> / 8;
      store_codes<KIND>(held + place(r8, r, in / 16) + in % 16, one, s);
      if (quarter == 0) held_scales[r8 * 8 + r][block] = (uint8_t)s;
    }
    __syncthreads();
    const int64_t out = g * x.rows + row;
    const int64_t whole = (int64_t)blocks * 32 * kMicroBits<KIND> / 8;  // bytes of a row's codes
    for (int i = tid; i < kAcross * kPieces; i += 256) {
      const int a = i / kPieces % 8, b = i / kPieces / 8, r = 8 * a + b, c = i % kPieces;
      const int64_t at = tl * kRow + c * 16;
      if (row + r < x.rows && at < whole)
        *reinterpret_cast<uint4*>(codes + (out + r) * whole + at) =
            *reinterpret_cast<const uint4*>(held + place(a, b, c));
    }
    for (int i = tid; i < kAcross * 8; i += 256) {
      const int r = i >> 3, b = i & 7;
      if (row + r < x.rows && tl * 8 + b < filled)
        scales[(out + r) * filled + tl * 8 + b] = held_scales[r][b];
    }
    __syncthreads();
  }
}

// Rows of codes to the values they stand for.
template <typename T, int KIND>
__global__ __launch_bounds__(256) void k_unpack(const uint8_t* __restrict__ codes,
                                                const uint8_t* __restrict__ scales, int64_t length,
                                                Divider by_row, uint32_t pieces, int64_t first,
                                                T* __restrict__ out, int64_t ldo) {
  const int blocks = micro_blocks(length), filled = micro_filled(blocks);
  for (uint32_t n = blockIdx.x * 256 + threadIdx.x; n < pieces; n += gridDim.x * 256) {
    const uint32_t in = by_row.quotient(n);
    const int at = (int)(n - in * by_row.d);
    const int64_t row = first + in, l = (int64_t)at * 8;
    float v[8];
    load_codes<KIND>(codes + (row * blocks * 32 + l) * kMicroBits<KIND> / 8,
                     scales[row * filled + (at >> 2)], v);
    store8(out + row * ldo + l, (int)min<int64_t>(8, length - l), v);
  }
}

// ---------------------------------------------------------------------------
// the activation
// ---------------------------------------------------------------------------

// h = f(gate) value, or f(u) without a gate; KEEP: u is packed to 8 bits on its way, each half by
// itself.  Thread number n of the rows has 8 neighbours of h.
template <typename T, bool GATED, bool KEEP>
__global__ __launch_bounds__(256) void k_activate(int act, const T* __restrict__ u, int64_t ldu,
                                                  int64_t hidden, Divider by_row, uint32_t pieces,
                                                  int64_t first, T* __restrict__ out,
                                                  uint8_t* __restrict__ codes,
                                                  uint8_t* __restrict__ scales) {
  using A = typename Elem<T>::Acc;
  const int blocks = micro_blocks(hidden), filled = micro_filled(blocks);
  for (uint32_t n = blockIdx.x * 256 + threadIdx.x; n < pieces; n += gridDim.x * 256) {
    const uint32_t in = by_row.quotient(n);
    const int at = (int)(n - in * by_row.d);
    const int64_t row = first + in, l = (int64_t)at * 8;
    const int some = (int)max<int64_t>(0, min<int64_t>(8, hidden - l));
    A g[8], v[8], h[8];
    const Eight<T> first_half(u + row * ldu + l, some);
    Eight<T> second;
    if constexpr (GATED) second = Eight<T>(u + row * ldu + hidden + l, some);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      g[i] = first_half[i];
      if constexpr (GATED) v[i] = second[i];
      h[i] = activation<T>(act, g[i]);
      if constexpr (GATED) h[i] *= v[i];
    }
    store8(out + row * hidden + l, some, h);
    if constexpr (KEEP) {
#pragma unroll
      for (int half = 0; half < (GATED ? 2 : 1); ++half) {
        const A(&x)[8] = half ? v : g;
        uint32_t most = magnitude(x[0]);
#pragma unroll
        for (int i = 1; i < 8; ++i) most = max(most, magnitude(x[i]));
        most = quad_max(most);
        const uint32_t s = micro_scale<kInt8>(most);
        const int64_t to = row * (GATED ? 2 : 1) + half;
        if ((at & 3) == 0) scales[to * filled + (at >> 2)] = (uint8_t)s;
        if ((at >> 2) < blocks) store_codes<kInt8>(codes + to * blocks * 32 + l, x, s);
      }
    }
  }
}

// g_gate = f'(gate) value g, g_value = f(gate) g; KEPT: gate and value are what the 8 bits stand
// for.
template <typename T, bool GATED, bool KEPT>
__global__ __launch_bounds__(256) void k_activate_vjp(
    int act, const T* __restrict__ u, int64_t ldu, const uint8_t* __restrict__ codes,
    const uint8_t* __restrict__ scales, const T* __restrict__ g_out, int64_t ldg, int64_t hidden,
    Divider by_row, uint32_t pieces, int64_t first, T* __restrict__ g_u) {
  using A = typename Elem<T>::Acc;
  constexpr int kParts = GATED ? 2 : 1;
  const int blocks = micro_blocks(hidden), filled = micro_filled(blocks);
  for (uint32_t n = blockIdx.x * 256 + threadIdx.x; n < pieces; n += gridDim.x * 256) {
    const uint32_t in = by_row.quotient(n);
    const int at = (int)(n - in * by_row.d);
    const int64_t row = first + in, l = (int64_t)at * 8;
    const int some = (int)min<int64_t>(8, hidden - l);
    A x[kParts][8], g[8];
    const Eight<T> raw_g(g_out + row * ldg + l, some);
    if constexpr (KEPT) {
#pragma unroll
      for (int half = 0; half < kParts; ++half) {
        const int64_t from = row * kParts + half;
        load_codes<kInt8>(codes + from * blocks * 32 + l, scales[from * filled + (at >> 2)], x[half]);
      }
    } else {
      Eight<T> raw[kParts];
#pragma unroll
      for (int half = 0; half < kParts; ++half)
        raw[half] = Eight<T>(u + row * ldu + half * hidden + l, some);
#pragma unroll
      for (int half = 0; half < kParts; ++half)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[half][i] = raw[half][i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = raw_g[i];
    A to[kParts][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      A f, slope;
      activation_slope<T>(act, x[0][i], f, slope);
      if constexpr (GATED) {
        to[0][i] = slope * x[1][i] * g[i];
        to[1][i] = f * g[i];
      } else {
        to[0][i] = slope * g[i];
      }
    }
#pragma unroll
    for (int half = 0; half < kParts; ++half)
      store8(g_u + (row * kParts + half) * hidden + l, some, to[half]);
  }
}

// Calls f(first row, pieces, divider) for as many rows at a time as 31 bits hold the pieces of.
template <typename F>
static int by_rows(int64_t rows, int64_t per, F&& f) {
  const int64_t most = std::max<int64_t>(1, ((int64_t(1) << 30) - 1) / per);
  const Divider by((uint32_t)per);
  for (int64_t first = 0; first < rows; first += most)
    if (int rc = f(first, (uint32_t)(std::min(most, rows - first) * per), by)) return rc;
  return PURIN_CP_OK;
}

static int check_kind(int32_t kind) {
  return kind == PURIN_TRAIN_FP4 || kind == PURIN_TRAIN_INT8 ? PURIN_CP_OK
                                                             : refuse("unknown kind");
}
static int check_length(int64_t groups, int64_t rows, int64_t length) {
  if (groups < 0 || rows < 0 || length < 0) return refuse("sizes must not be negative");
  if (length > (int64_t(1) << 30))
    return set_error(PURIN_CP_ERR_UNSUPPORTED, "rows must not be longer than 2^30");
  if (rows >= (int64_t(1) << 40) || groups >= (int64_t(1) << 40))
    return set_error(PURIN_CP_ERR_UNSUPPORTED, "rows and groups must stay below 2^40");
  return PURIN_CP_OK;
}
static int check_activation(int32_t act, int32_t dtype, int64_t rows, int64_t hidden) {
  if (!known_dtype(dtype)) return refuse("unknown dtype");
  if (act < PURIN_TRAIN_RELU || act > PURIN_TRAIN_GELU) return refuse("unknown activation");
  return check_length(1, rows, hidden);
}
static int32_t aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
static const char* const kAlign = "codes must lie at 16 bytes, scales at 4";
static bool codes_ok(const void* codes, const void* scales) {
  return aligned16(codes) && reinterpret_cast<uintptr_t>(scales) % 4 == 0;
}

template <typename T, int KIND>
static int pack(hipStream_t st, const Strided<T>& x, uint8_t* codes, uint8_t* scales) {
  const unsigned gy = (unsigned)std::min<int64_t>(x.groups, 32768);
  if (x.sl == 1 || x.length == 1) {
    return by_rows(x.rows, micro_filled(micro_blocks(x.length)) * 4,
                   [&](int64_t first, uint32_t pieces, const Divider& by) {
                     const unsigned gx = grid_of(pieces, 256).x;
                     const dim3 grid(gx, std::min(gy, std::max(1u, (1u << 23) / gx)));
                     k_pack<T, KIND><<<grid, dim3(256), 0, st>>>(x, by, pieces, first, codes, scales);
                     return launched("k_pack");
                   });
  }
  const int64_t tiles_l = (micro_filled(micro_blocks(x.length)) + 7) / 8;
  const int64_t tiles_r = (x.rows + kAcross - 1) / kAcross, tiles = tiles_l * tiles_r;
  if (tiles >= (int64_t(1) << 24)) return set_error(PURIN_CP_ERR_UNSUPPORTED, "too many tiles for a launch");
  const unsigned most = (unsigned)std::max<int64_t>(1, (int64_t(1) << 23) / tiles);  // threads below 2^32
  k_pack_across<T, KIND><<<dim3((unsigned)tiles, std::min(gy, most)), dim3(256), 0, st>>>(
      x, tiles_r, codes, scales);
  return launched("k_pack_across");
}

}  // namespace train
}  // namespace purin

using namespace purin;
using namespace purin::train;

extern "C" {

int purin_train_pack(void* stream, int32_t dtype, int32_t kind, int64_t groups, int64_t rows,
                     int64_t length, const void* x, int64_t sg, int64_t sr, int64_t sl, void* codes,
                     void* scales) {
  return guarded([&] {
    if (!known_dtype(dtype)) return refuse("unknown dtype");
    if (dtype == PURIN_TRAIN_F64)
      return set_error(PURIN_CP_ERR_UNSUPPORTED, "numbers of 64 bits are not packed");
    if (int rc = check_kind(kind)) return rc;
    if (int rc = check_length(groups, rows, length)) return rc;
    if (sg < 0 || sr < 0 || sl < 0) return refuse("strides must not be negative");
    if (sl != 1 && sr != 1 && length > 1 && rows > 1)
      return refuse("a unit stride is needed along the rows or along their length");
    if (!groups || !rows || !length) return (int)PURIN_CP_OK;
    if (!x || !codes || !scales) return refuse("NULL array");
    if (!codes_ok(codes, scales)) return refuse(kAlign);
    return by_dtype(dtype, [&](auto v) {
      using T = decltype(v);
      if constexpr (sizeof(T) == 8) return (int)PURIN_CP_ERR_UNSUPPORTED;
      else {
        const Strided<T> from{(const T*)x, groups, rows, length, sg, sr, sl};
        return kind == PURIN_TRAIN_FP4
                   ? pack<T, kFp4>((hipStream_t)stream, from, (uint8_t*)codes, (uint8_t*)scales)
                   : pack<T, kInt8>((hipStream_t)stream, from, (uint8_t*)codes, (uint8_t*)scales);
      }
    });
  });
}

int purin_train_unpack(void* stream, int32_t dtype, int32_t kind, int64_t rows, int64_t length,
                       const void* codes, const void* scales, void* out, int64_t ldo) {
  return guarded([&] {
    if (!known_dtype(dtype)) return refuse("unknown dtype");
    if (dtype == PURIN_TRAIN_F64)
      return set_error(PURIN_CP_ERR_UNSUPPORTED, "numbers of 64 bits are not packed");
    if (int rc = check_kind(kind)) return rc;
    if (int rc = check_length(1, rows, length)) return rc;
    if (!rows || !length) return (int)PURIN_CP_OK;
    if (!codes || !scales || !out) return refuse("NULL array");
    if (rows > 1 && ldo < length) return refuse("a row pitch is below the row's length");
    if (!codes_ok(codes, scales)) return refuse(kAlign);
    return by_dtype(dtype, [&](auto v) {
      using T = decltype(v);
      if constexpr (sizeof(T) == 8) return (int)PURIN_CP_ERR_UNSUPPORTED;
      else
        return by_rows(rows, (length + 7) / 8, [&](int64_t first, uint32_t pieces, const Divider& by) {
          auto kernel = kind == PURIN_TRAIN_FP4 ? k_unpack<T, kFp4> : k_unpack<T, kInt8>;
          kernel<<<grid_of(pieces, 256), dim3(256), 0, (hipStream_t)stream>>>(
              (const uint8_t*)codes, (const uint8_t*)scales, length, by, pieces, first, (T*)out, ldo);
          return launched("k_unpack");
        });
    });
  });
}

int purin_train_activate(void* stream, int32_t dtype, int32_t activation, int32_t gated,
                         int64_t rows, int64_t hidden, const void* u, int64_t ldu, void* out,
                         void* codes, void* scales) {
  return guarded([&] {
    if (int rc = check_activation(activation, dtype, rows, hidden)) return rc;
    if (!codes != !scales) return refuse("codes and scales go together");
    if (codes && dtype == PURIN_TRAIN_F64)
      return set_error(PURIN_CP_ERR_UNSUPPORTED, "numbers of 64 bits are not packed");
    if (!rows || !hidden) return (int)PURIN_CP_OK;
    if (!u || !out) return refuse("NULL array");
    if (rows > 1 && ldu < (gated ? 2 : 1) * hidden)
      return refuse("a row pitch is below the row's length");
    if (!codes_ok(codes, scales)) return refuse(kAlign);
    return by_dtype(dtype, [&](auto v) {
      using T = decltype(v);
      auto go = [&](auto kernel, int64_t per) {
        return by_rows(rows, per, [&](int64_t first, uint32_t pieces, const Divider& by) {
          kernel<<<grid_of(pieces, 256), dim3(256), 0, (hipStream_t)stream>>>(
              activation, (const T*)u, ldu, hidden, by, pieces, first, (T*)out, (uint8_t*)codes,
              (uint8_t*)scales);
          return launched("k_activate");
        });
      };
      if constexpr (sizeof(T) != 8)
        if (codes)
          return go(gated ? k_activate<T, true, true> : k_activate<T, false, true>,
                    micro_filled(micro_blocks(hidden)) * 4);
      return go(gated ? k_activate<T, true, false> : k_activate<T, false, false>, (hidden + 7) / 8);
    });
  });
}

int purin_train_activate_vjp(void* stream, int32_t dtype, int32_t activation, int32_t gated,
                             int64_t rows, int64_t hidden, const void* u, int64_t ldu,
                             const void* codes, const void* scales, const void* g, int64_t ldg,
                             void* g_u) {
  return guarded([&] {
    if (int rc = check_activation(activation, dtype, rows, hidden)) return rc;
    if (!codes != !scales) return refuse("codes and scales go together");
    if (codes && dtype == PURIN_TRAIN_F64)
      return set_error(PURIN_CP_ERR_UNSUPPORTED, "numbers of 64 bits are not packed");
    if (!rows || !hidden) return (int)PURIN_CP_OK;
    if ((!u && !codes) || !g || !g_u) return refuse("NULL array");
    if (rows > 1 && ((!codes && ldu < (gated ? 2 : 1) * hidden) || ldg < hidden))
      return refuse("a row pitch is below the row's length");
    if (!codes_ok(codes, scales)) return refuse(kAlign);
    return by_dtype(dtype, [&](auto v) {
      using T = decltype(v);
      auto go = [&](auto kernel) {
        return by_rows(rows, (hidden + 7) / 8, [&](int64_t first, uint32_t pieces, const Divider& by) {
          kernel<<<grid_of(pieces, 256), dim3(256), 0, (hipStream_t)stream>>>(
              activation, (const T*)u, ldu, (const uint8_t*)codes, (const uint8_t*)scales,
              (const T*)g, ldg, hidden, by, pieces, first, (T*)g_u);
          return launched("k_activate_vjp");
        });
      };
      if constexpr (sizeof(T) != 8)
        if (codes) return go(gated ? k_activate_vjp<T, true, true> : k_activate_vjp<T, false, true>);
      return go(gated ? k_activate_vjp<T, true, false> : k_activate_vjp<T, false, false>);
    });
  });
}

}  // extern "C"
