// A whole layer of experts for a few tokens (include/purin_train.h: expert_layer).
//
//   out(t) = sum over t's experts e of  w(t, e) f(x(t) A[e]) B[e]
//
// Every weight of an expert that some token has is read once: that is the work, and the tokens'
// rows are few beside it.  So nothing is sorted: a workgroup has one expert and 64 columns of its
// matrix, finds the tokens that have the expert and takes their rows as those of its tile.  Two
// launches and their sum:
//   up     chooses the tokens' experts (every workgroup for itself), multiplies by A, applies f
//          and the token's weight.  The results keep twice the type's digits, as the sum of two
//          numbers of the type, so that they take part in the second product as they are;
//   down   multiplies them by B, a row of 32-bit sums for each (token, slot);
//   sum    adds a token's rows in the order of its slots.

#include <algorithm>

#include "choose.hpp"
#include "packed.hpp"
#include "tiles.hpp"

namespace purin {
namespace train {

constexpr int kTokens = PURIN_TRAIN_LAYER_TOKENS, kPairs = PURIN_TRAIN_LAYER_PAIRS;

// An expert's matrix: rows of codes, or a dense one whose contraction is contiguous (ld apart)
// or across.
struct Matrices {
  const void* values;
  const uint8_t* scales;
  int64_t se, ld;
};

// The two times 32 columns of a workgroup's tile: starts and how many are there.
struct Columns {
  int64_t first[2];
  int n[2];
};

// ---------------------------------------------------------------------------
// sums of BM rows and 2 x 32 columns
// ---------------------------------------------------------------------------

// Microscaled weights.
template <typename T, int BM, int NA>
struct ThinCodes {
  using Core = ThinPacked<T, BM, NA, BM * NA <= 64 ? 3 : 2>;  // as many as LDS holds
  static constexpr int kRing = Core::kRing;

  template <typename F>
  static __device__ __forceinline__ void run(const T* const (&a)[NA], F&& offset, int64_t inner,
                                             const Matrices& w, int e, int64_t outer,
                                             const Columns& c, unsigned char* lds,
                                             F16x (&acc)[BM / 32][2]) {
    const Codes b((const uint8_t*)w.values, w.scales, e * outer, inner);
    Core::run(a, offset, inner, b,
              [&](int j) {
                const bool second = j >= 32;
                const int in = j & 31;
                return in < (second ? c.n[1] : c.n[0]) ? (int)(second ? c.first[1] : c.first[0]) + in
                                                       : -1;
              },
              0, b.blocks, lds, acc);
  }
};

// Dense weights.
template <typename T, int BM, int NA, bool ALONG, bool DIRECT>
struct ThinDense {
  static constexpr int X = BM / 32, S = 4, AHEAD = 3;
  using SA = PieceStage<BM, 8, 256>;
  using SB = Stage<T, 32, ALONG, 256>;
  static constexpr int kStage = NA * SA::kBytes + 2 * SB::kElems * 2;
  static constexpr int kLoads = NA * SA::kMine + 2 * SB::kMine;
  static constexpr int kRing = (DIRECT ? S : 2) * kStage;

  static __device__ __forceinline__ void multiply(const uint8_t* la, F16x (&acc)[X][2]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T* lb = reinterpret_cast<const T*>(la + NA * SA::kBytes);
    S8 fb[2];
#pragma unroll
    for (int y = 0; y < 2; ++y) fb[y] = fragment<T, 32, ALONG>(lb + y * SB::kElems, 0, wave);
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int x = 0; x < X; ++x) {
        const S8 fa = __builtin_bit_cast(S8, SA::piece(la + i * SA::kBytes, 32 * x + (lane & 31),
                                                       2 * wave + (lane >> 5)));
#pragma unroll
        for (int y = 0; y < 2; ++y) acc[x][y] = mma32(T{}, fb[y], fa, acc[x][y]);
      }
  }

  template <typename F>
  static __device__ __forceinline__ void run(const T* const (&a)[NA], F&& offset, int64_t inner,
                                             const Matrices& w, int e, int64_t, const Columns& c,
                                             unsigned char* lds, F16x (&acc)[X][2]) {
    const T* base = (const T*)w.values + e * w.se;
    Side<T> b[2];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      // columns that are not there: the first ones again, whose sums are dropped
      const int from = !DIRECT && c.n[y] <= 0 ? 0 : y;
      b[y] = {base + (ALONG ? c.first[from] * w.ld : c.first[from]), w.ld, c.n[from],
              c.first[from] > 0};
    }
    uint32_t off_a[SA::kMine], off_b[2][SB::kMine];
    SA::offsets(offset, off_a);
    const int64_t step = ALONG ? kDepth16 : kDepth16 * w.ld;
    if constexpr (DIRECT) {
      const uint8_t* pa[NA];
      const T* pb[2];
#pragma unroll
      for (int i = 0; i < NA; ++i) pa[i] = reinterpret_cast<const uint8_t*>(uniform(a[i]));
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        SB::offsets(b[y], off_b[y]);
        pb[y] = uniform(b[y].p);
      }
      const int64_t pieces = (inner + 7) / 8;
      const uint32_t to = lds_address(lds);
      ring<S, kLoads>(
          (inner + kDepth16 - 1) / kDepth16,
          [&](int64_t t, int at) {
#pragma unroll
            for (int i = 0; i < NA; ++i)
              SA::load(pa[i] + t * 128, off_a, pieces - 8 * t, to + (uint32_t)(at * kStage + i * SA::kBytes));
            T* lb = reinterpret_cast<T*>(lds + at * kStage + NA * SA::kBytes);
#pragma unroll
            for (int y = 0; y < 2; ++y)
              SB::load_lds(pb[y] + t * step, off_b[y], inner - t * kDepth16, lb + y * SB::kElems);
          },
          [&](int64_t, int at) { multiply(lds + at * kStage, acc); });
    } else {
      // through registers, as through_registers does for two operands
      Pack<T> va[AHEAD][NA][SA::kMine], vb[AHEAD][2][SB::kMine];
      auto put = [&](const Pack<T>(&a)[NA][SA::kMine], const Pack<T>(&b)[2][SB::kMine],
                     const uint32_t(&move)[2], const int(&by)[2], unsigned char* to) {
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
          for (int m = 0; m < SA::kMine; ++m)
            *reinterpret_cast<S8*>(to + i * SA::kBytes + (m * 256 + (int)threadIdx.x) * 16) =
                __builtin_bit_cast(S8, a[i][m]);
        T* lb = reinterpret_cast<T*>(to + NA * SA::kBytes);
#pragma unroll
        for (int y = 0; y < 2; ++y) SB::store_settled(move[y], by[y], b[y], lb + y * SB::kElems);
      };
      const int64_t whole = SB::whole(b[0]) && SB::whole(b[1]) ? inner / kDepth16 : 0;
      int64_t t = 0;
      int now = 0;
      if (whole) {
        uint32_t move[2];
        int by[2];
        const T* from[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          move[y] = SB::reach(b[y], off_b[y]);
          by[y] = b[y].n % kVec<T> ? kVec<T> - b[y].n % kVec<T> : 0;
          from[y] = uniform(b[y].p) - SB::lead(b[y]);
        }
        int64_t at = 0;
        // without a condition, so that the waits count on it: past the last whole stage, that
        // one again; rows that are not there read the first
        auto load = [&](int v) {
#pragma unroll
          for (int i = 0; i < NA; ++i)
#pragma unroll
            for (int m = 0; m < SA::kMine; ++m) {
              const uint32_t o = off_a[m] == kOutside ? 0u : off_a[m];
              va[v][i][m] = load16(reinterpret_cast<const T*>(
                  reinterpret_cast<const uint8_t*>(a[i]) + at * 128 + o));
            }
#pragma unroll
          for (int y = 0; y < 2; ++y) SB::load(from[y] + at * step, off_b[y], vb[v][y]);
          if (at + 1 < whole) ++at;
        };
#pragma unroll
        for (int s = 0; s < AHEAD; ++s) load(s);
        put(va[0], vb[0], move, by, lds);
        for (; t < whole; t += AHEAD) {
#pragma unroll
          for (int u = 0; u < AHEAD; ++u) {
            if (t + u >= whole) break;
            __syncthreads();
            load(u);
            multiply(lds + now * kStage, acc);
            if (t + u + 1 < whole)
              put(va[(u + 1) % AHEAD], vb[(u + 1) % AHEAD], move, by, lds + (now ^ 1) * kStage);
            now ^= 1;
          }
        }
        t = whole;
      }
      const uint32_t still[2] = {0, 0};
      const int none[2] = {0, 0};
      for (; t * kDepth16 < inner; ++t) {
        const int64_t left = inner - t * kDepth16;
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
          for (int m = 0; m < SA::kMine; ++m) {
            const int q = m * 256 + (int)threadIdx.x;
            const int first = SA::place(q / 8, q % 8) % 8 * 8;
            va[0][i][m] = off_a[m] == kOutside || first >= left
                              ? zeros16<T>()
                              : load_upto(reinterpret_cast<const T*>(
                                              reinterpret_cast<const uint8_t*>(a[i]) + off_a[m]) +
                                              t * kDepth16,
                                          left - first);
          }
#pragma unroll
        for (int y = 0; y < 2; ++y) SB::load_each(b[y], b[y].p + t * step, left, vb[0][y]);
        put(va[0], vb[0], still, none, lds + now * kStage);
        __syncthreads();
        multiply(lds + now * kStage, acc);
        now ^= 1;
      }
      __syncthreads();
    }
  }
};

// ---------------------------------------------------------------------------
// who has which expert
// ---------------------------------------------------------------------------

struct AnyRow {
  const void* p;
  int32_t dtype;
  int64_t first;
  __device__ __forceinline__ double operator[](int e) const {
    return load_weight<double>(p, dtype, first + e);
  }
};

template <int G, int V>
__device__ __forceinline__ void choose_tokens(const void* weights, int32_t wdtype, int64_t ldw,
                                              int tokens, int experts, int slots, int32_t* ids,
                                              double* chosen) {
  for (int t = threadIdx.x / G; t < tokens; t += 256 / G)
    choose<double, G, V>(AnyRow{weights, wdtype, t * ldw}, experts, slots, (int)threadIdx.x % G,
                         ids + t * slots, chosen + t * slots);
}

// The expert that is number ``group`` among those with a token, -1 past the last, and its
// tokens' pairs (token * slots + slot), in order.  Every wavefront finds the expert by itself.
struct Group {
  uint32_t used[PURIN_TRAIN_MAX_EXPERTS / 32];
  int32_t pair_of[kTokens];
  int32_t list[kTokens];
  int32_t count;
};
__device__ __forceinline__ int find_group(const int32_t* ids, int pairs, int slots, int group,
                                          Group& g) {
  const int tid = threadIdx.x, lane = tid & 63;
  if (tid < PURIN_TRAIN_MAX_EXPERTS / 32) g.used[tid] = 0;
  if (tid < kTokens) g.pair_of[tid] = -1;
  __syncthreads();
  for (int p = tid; p < pairs; p += 256) {
    const int32_t e = ids[p];
    if (e >= 0) atomicOr(&g.used[e >> 5], 1u << (e & 31));
  }
  __syncthreads();
  uint32_t word = lane < PURIN_TRAIN_MAX_EXPERTS / 32 ? g.used[lane] : 0;
  const int n = __popc(word);
  int sum = n;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up(sum, d, 64);
    if (lane >= d) sum += up;
  }
  const uint64_t here = __ballot(lane < 32 && group < sum);
  if (!here) return -1;
  const int at = __ffsll((unsigned long long)here) - 1;
  word = (uint32_t)__shfl((int)word, at, 64);
  for (int skip = group - (__shfl(sum, at, 64) - __popc(word)); skip > 0; --skip) word &= word - 1;
  const int expert = __builtin_amdgcn_readfirstlane(at * 32 + __ffs(word) - 1);
  for (int p = tid; p < pairs; p += 256)
    if (ids[p] == expert) g.pair_of[p / slots] = p;
  __syncthreads();
  if (tid < kTokens) {
    const int32_t pair = g.pair_of[tid];
    const uint64_t have = __ballot(pair >= 0);
    if (pair >= 0) g.list[__popcll(have & ((uint64_t(1) << tid) - 1))] = pair;
    if (tid == 0) g.count = __popcll(have);
  }
  __syncthreads();
  return expert;
}

template <typename T, int BM>
__device__ __forceinline__ void clear(F16x (&acc)[BM / 32][2]) {
#pragma unroll
  for (int x = 0; x < BM / 32; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.0f;
}

template <int BM, typename Core>
constexpr int layer_lds() {
  constexpr int choice = kPairs * 12;
  constexpr int most = Core::kRing > kThinSums<BM> ? Core::kRing : kThinSums<BM>;
  return most > choice ? most : choice;
}

struct Up {
  const void* weights;
  int64_t ldw;
  int32_t wdtype, tokens, experts, slots, act, gated;
  int64_t ldx, width, hidden, pitch, tiles;
};

// Workgroup: expert number blockIdx.x / tiles, columns of tile blockIdx.x % tiles.
template <typename T, int BM, typename Core>
__global__ __launch_bounds__(256) void k_layer_up(Up p, const T* __restrict__ x, Matrices w,
                                                  int32_t* __restrict__ ids_out,
                                                  T* __restrict__ high, T* __restrict__ low) {
  extern __shared__ __align__(16) unsigned char lds16[];
  __shared__ Group group;
  __shared__ float weight_of[kTokens];
  const int tid = threadIdx.x, pairs = p.tokens * p.slots;
  double* chosen = reinterpret_cast<double*>(lds16);
  int32_t* ids = reinterpret_cast<int32_t*>(lds16 + kPairs * 8);
  if (p.experts <= 64)
    choose_tokens<16, 4>(p.weights, p.wdtype, p.ldw, p.tokens, p.experts, p.slots, ids, chosen);
  else if (p.experts <= 256)
    choose_tokens<16, 16>(p.weights, p.wdtype, p.ldw, p.tokens, p.experts, p.slots, ids, chosen);
  else
    choose_tokens<64, 16>(p.weights, p.wdtype, p.ldw, p.tokens, p.experts, p.slots, ids, chosen);
  __syncthreads();
  if (blockIdx.x == 0)
    for (int i = tid; i < pairs; i += 256) ids_out[i] = ids[i];
  const int at = (int)(blockIdx.x / p.tiles), tile = (int)(blockIdx.x - at * p.tiles);
  const int e = find_group(ids, pairs, p.slots, at, group);
  if (e < 0) return;
  const int count = group.count;
  if (tid < count) weight_of[tid] = (float)chosen[group.list[tid]];
  __syncthreads();
  const int wide = p.gated ? 32 : 64;  // columns of h
  const int64_t col = (int64_t)tile * wide, outer = p.gated ? 2 * p.hidden : p.hidden;
  Columns c;
  c.first[0] = col;
  c.n[0] = (int)min<int64_t>(32, p.hidden - col);
  c.first[1] = p.gated ? p.hidden + col : col + 32;
  c.n[1] = p.gated ? c.n[0] : (int)max<int64_t>(0, min<int64_t>(32, p.hidden - col - 32));
  for (int r0 = 0; r0 < count; r0 += BM) {
    F16x acc[BM / 32][2];
    clear<T, BM>(acc);
    const T* const a[1] = {x};
    Core::run(a,
              [&](int r) {
                return r0 + r < count
                           ? (uint32_t)(group.list[r0 + r] / p.slots) * (uint32_t)p.ldx * 2u
                           : kOutside;
              },
              p.hidden ? p.width : 0, w, e, outer, c, lds16, acc);
    float* sums = reinterpret_cast<float*>(lds16);
    thin_parts<BM>(acc, sums);
    for (int i = tid; i < min(BM, count - r0) * (wide / 8); i += 256) {
      const int r = i / (wide / 8), j = i % (wide / 8) * 8;
      if (col + j >= p.pitch) continue;
      Pack<T> hi, lo;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        float h = activation<T>(p.act, thin_sum<BM>(sums, r, j + q));
        if (p.gated) h *= thin_sum<BM>(sums, r, 32 + j + q);
        h = col + j + q < p.hidden ? h * weight_of[r0 + r] : 0.0f;
        hi.v[q] = (T)h;
        const float rest = h - (float)hi.v[q];
        lo.v[q] = (T)(fabsf((float)hi.v[q]) < __builtin_inff() ? rest : 0.0f);
      }
      const int64_t to = group.list[r0 + r] * p.pitch + col + j;
      store16(high + to, hi);
      store16(low + to, lo);
    }
    __syncthreads();
  }
}

struct Down {
  int32_t tokens, slots;
  int64_t hidden, outer, pitch, tiles;
};

template <typename T, int BM, typename Core>
__global__ __launch_bounds__(256) void k_layer_down(Down p, const T* __restrict__ high,
                                                    const T* __restrict__ low, Matrices w,
                                                    const int32_t* __restrict__ ids_in,
                                                    float* __restrict__ parts) {
  extern __shared__ __align__(16) unsigned char lds16[];
  __shared__ Group group;
  const int tid = threadIdx.x, pairs = p.tokens * p.slots;
  int32_t* ids = reinterpret_cast<int32_t*>(lds16);
  for (int i = tid; i < pairs; i += 256) ids[i] = ids_in[i];
  __syncthreads();
  const int at = (int)(blockIdx.x / p.tiles), tile = (int)(blockIdx.x - at * p.tiles);
  const int e = find_group(ids, pairs, p.slots, at, group);
  if (e < 0) return;
  const int64_t col = (int64_t)tile * 64;
  Columns c;
  c.first[0] = col;
  c.n[0] = (int)min<int64_t>(32, p.outer - col);
  c.first[1] = col + 32;
  c.n[1] = (int)max<int64_t>(0, min<int64_t>(32, p.outer - col - 32));
  const int n = (int)min<int64_t>(64, p.outer - col), count = group.count;
  for (int r0 = 0; r0 < count; r0 += BM) {
    F16x acc[BM / 32][2];
    clear<T, BM>(acc);
    const T* const a[2] = {high, low};
    Core::run(a,
              [&](int r) {
                return r0 + r < count ? (uint32_t)group.list[r0 + r] * (uint32_t)p.pitch * 2u
                                      : kOutside;
              },
              p.hidden, w, e, p.outer, c, lds16, acc);
    float* sums = reinterpret_cast<float*>(lds16);
    thin_parts<BM>(acc, sums);
    for (int i = tid; i < min(BM, count - r0) * 16; i += 256) {
      const int r = i >> 4, j = (i & 15) * 4;
      if (j >= n) continue;
      Pack<float> v;
#pragma unroll
      for (int q = 0; q < 4; ++q) v.v[q] = thin_sum<BM>(sums, r, j + q);
      store_upto(parts + group.list[r0 + r] * p.outer + col + j, v, n - j);
    }
    __syncthreads();
  }
}

// A token's rows added up in the order of its slots.
template <typename T>
__global__ __launch_bounds__(256) void k_layer_sum(const float* __restrict__ parts,
                                                   const int32_t* __restrict__ ids, int slots,
                                                   int64_t outer, T* __restrict__ out) {
  const int64_t t = blockIdx.y, j = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (j >= outer) return;
  float sum[4] = {0, 0, 0, 0};
  for (int s = 0; s < slots; ++s) {
    if (ids[t * slots + s] < 0) continue;
    const Pack<float> v = load_upto(parts + (t * slots + s) * outer + j, outer - j);
#pragma unroll
    for (int q = 0; q < 4; ++q) sum[q] += v.v[q];
  }
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (j + q < outer) out[t * outer + j + q] = (T)sum[q];
}

// The workspace's parts, each at 256 bytes.
struct LayerSpace {
  int64_t pitch, ids, high, low, parts, x, bytes;
  LayerSpace(int64_t tokens, int64_t slots, int64_t width, int64_t hidden, int64_t outer) {
    const int64_t pairs = tokens * slots;
    pitch = (hidden + 63) / 64 * 64;
    ids = 0;
    high = ids + whole256(pairs * 4);
    low = high + whole256(pairs * pitch * 2);
    parts = low + whole256(pairs * pitch * 2);
    x = parts + whole256(pairs * outer * 4);
    bytes = x + aligned_bytes(tokens, width);
  }
};

// How an expert's matrices are read.
enum Reading { kCodes, kAlongDirect, kAcrossDirect, kAlong, kAcross };
static Reading reading(const purin_train_matrices& m, int64_t inner, int64_t outer, int64_t half,
                       bool rows_ok, int64_t* ld) {
  if (m.scales) {
    *ld = 0;
    return kCodes;
  }
  const bool along = m.so != 1 && (m.si == 1 || inner <= 1);
  *ld = along ? m.so : m.si;
  const bool direct = rows_ok && direct_ok(m.values, *ld, along ? inner : outer) && m.se % 8 == 0 &&
                      (along || half % 8 == 0);
  return along ? (direct ? kAlongDirect : kAlong) : (direct ? kAcrossDirect : kAcross);
}

template <typename T>
static int layer(hipStream_t st, const Up& shape, int64_t outer, const T* x,
                 const purin_train_matrices& inner, const purin_train_matrices& out_matrices,
                 uint8_t* ws, T* out) {
  Up up = shape;
  const LayerSpace at(up.tokens, up.slots, up.width, up.hidden, outer);
  const int64_t pairs = (int64_t)up.tokens * up.slots, groups = std::min<int64_t>(up.experts, pairs);
  int32_t* ids = (int32_t*)(ws + at.ids);
  T *high = (T*)(ws + at.high), *low = (T*)(ws + at.low);
  float* parts = (float*)(ws + at.parts);
  const int64_t columns = up.gated ? 2 * up.hidden : up.hidden;
  Matrices a{inner.values, (const uint8_t*)inner.scales, inner.se, 0};
  const bool rows_ok = direct_ok(x, up.ldx, up.width);
  const Reading how = reading(inner, up.width, columns, up.hidden, rows_ok, &a.ld);
  if (how == kCodes && up.width && !rows_ok) {
    if (int rc = align_rows<T>(st, x, up.ldx, up.tokens, up.width, (T*)(ws + at.x))) return rc;
    x = (const T*)(ws + at.x);
    up.ldx = (up.width + 7) / 8 * 8;
  }
  up.pitch = at.pitch;
  up.tiles = std::max<int64_t>(1, (up.hidden + (up.gated ? 31 : 63)) / (up.gated ? 32 : 64));
  auto launch_up = [&](auto bm, auto core) {
    constexpr int BM = bm;
    using Core = decltype(core);
    return launch16("k_layer_up", k_layer_up<T, BM, Core>, groups * up.tiles, 1, 1, 256,
                    layer_lds<BM, Core>(), st, up, x, a, ids, high, low);
  };
  auto go_up = [&](auto bm) {
    constexpr int BM = bm;
    switch (how) {
      case kCodes: return launch_up(bm, ThinCodes<T, BM, 1>{});
      case kAlongDirect: return launch_up(bm, ThinDense<T, BM, 1, true, true>{});
      case kAcrossDirect: return launch_up(bm, ThinDense<T, BM, 1, false, true>{});
      case kAlong: return launch_up(bm, ThinDense<T, BM, 1, true, false>{});
      default: return launch_up(bm, ThinDense<T, BM, 1, false, false>{});
    }
  };
  // an expert with more rows than a tile reads its weights again
  const bool tall = up.tokens > 32 && pairs > 16 * up.experts;
  if (int rc = tall ? go_up(i64) : go_up(i32)) return rc;
  Matrices b{out_matrices.values, (const uint8_t*)out_matrices.scales, out_matrices.se, 0};
  const Reading how_b = reading(out_matrices, up.hidden, outer, 8, true, &b.ld);
  const Down down{up.tokens, up.slots, up.hidden, outer, at.pitch, (outer + 63) / 64};
  auto launch_down = [&](auto bm, auto core) {
    constexpr int BM = bm;
    using Core = decltype(core);
    return launch16("k_layer_down", k_layer_down<T, BM, Core>, groups * down.tiles, 1, 1, 256,
                    layer_lds<BM, Core>(), st, down, (const T*)high, (const T*)low, b,
                    (const int32_t*)ids, parts);
  };
  auto go_down = [&](auto bm) {
    constexpr int BM = bm;
    switch (how_b) {
      case kCodes: return launch_down(bm, ThinCodes<T, BM, 2>{});
      case kAlongDirect: return launch_down(bm, ThinDense<T, BM, 2, true, true>{});
      case kAcrossDirect: return launch_down(bm, ThinDense<T, BM, 2, false, true>{});
      case kAlong: return launch_down(bm, ThinDense<T, BM, 2, true, false>{});
      default: return launch_down(bm, ThinDense<T, BM, 2, false, false>{});
    }
  };
  if (int rc = tall ? go_down(i64) : go_down(i32)) return rc;
  k_layer_sum<T><<<dim3((unsigned)((outer + 1023) / 1024), (unsigned)up.tokens), dim3(256), 0, st>>>(
      parts, ids, up.slots, outer, out);
  return launched("k_layer_sum");
}

static int check_layer(int32_t dtype, int64_t tokens, int64_t experts, int64_t slots, int64_t width,
                       int64_t hidden, int64_t outer) {
  if (!known_dtype(dtype)) return refuse("unknown dtype");
  if (dtype_bytes(dtype) != 2)
    return set_error(PURIN_CP_ERR_UNSUPPORTED, "expert_layer takes bfloat16 and float16");
  if (tokens < 0 || width < 0 || hidden < 0 || outer < 0 || experts < 1 || slots < 1)
    return refuse("sizes must not be negative, experts and slots must be positive");
  if (slots > experts) return refuse("slots must not exceed the experts");
  if (experts > PURIN_TRAIN_MAX_EXPERTS)
    return set_error(PURIN_CP_ERR_UNSUPPORTED, "more than 1024 experts");
  if (tokens > kTokens || tokens * slots > kPairs)
    return set_error(PURIN_CP_ERR_UNSUPPORTED,
                     "expert_layer takes at most 64 tokens, and 1024 slots of all of them");
  if (width > (int64_t(1) << 20) || hidden > (int64_t(1) << 19) || outer > (int64_t(1) << 20))
    return set_error(PURIN_CP_ERR_UNSUPPORTED,
                     "width and outer must not exceed 2^20, hidden 2^19");
  return PURIN_CP_OK;
}
static int check_matrices(const purin_train_matrices* m, int64_t inner, int64_t outer) {
  if (!m) return refuse("NULL matrices");
  if (inner && outer && !m->values) return refuse("NULL array");
  if (m->scales) {
    if (reinterpret_cast<uintptr_t>(m->values) % 16 || reinterpret_cast<uintptr_t>(m->scales) % 4)
      return refuse("codes must lie at 16 bytes, scales at 4");
    return PURIN_CP_OK;
  }
  if (m->se < 0 || m->si < 0 || m->so < 0) return refuse("the weight's strides must not be negative");
  if (m->si != 1 && m->so != 1 && inner > 1 && outer > 1)
    return refuse("the weight needs a unit stride along inner or outer");
  return PURIN_CP_OK;
}

}  // namespace train
}  // namespace purin

using namespace purin;
using namespace purin::train;

extern "C" {

int64_t purin_train_expert_layer_workspace_bytes(int32_t dtype, int64_t tokens, int64_t experts,
                                                 int64_t slots, int64_t width, int64_t hidden,
                                                 int64_t outer) {
  int64_t need = -1;
  (void)guarded([&] {
    if (int rc = check_layer(dtype, tokens, experts, slots, width, hidden, outer)) return rc;
    need = tokens && outer ? LayerSpace(tokens, slots, width, hidden, outer).bytes : 0;
    return (int)PURIN_CP_OK;
  });
  return need;
}

int purin_train_expert_layer(void* stream, int32_t dtype, int32_t wdtype, int64_t tokens,
                             int64_t experts, int64_t slots, int64_t width, int64_t hidden,
                             int64_t outer_width, int32_t activation, int32_t gated, const void* x,
                             int64_t ldx, const void* weights, int64_t ldw,
                             const purin_train_matrices* inner, const purin_train_matrices* outer,
                             void* workspace, int64_t workspace_bytes, void* out) {
  return guarded([&] {
    if (int rc = check_layer(dtype, tokens, experts, slots, width, hidden, outer_width)) return rc;
    if (!known_dtype(wdtype)) return refuse("unknown dtype");
    if (activation < PURIN_TRAIN_RELU || activation > PURIN_TRAIN_GELU)
      return refuse("unknown activation");
    if (int rc = check_matrices(inner, width, hidden)) return rc;
    if (int rc = check_matrices(outer, hidden, outer_width)) return rc;
    if (!tokens || !outer_width) return (int)PURIN_CP_OK;
    if ((width && !x) || !weights || !out) return refuse("NULL array");
    if (tokens > 1 && (ldx < width || ldw < experts))
      return refuse("a row pitch is below the row's length");
    if (tokens > 1 && ldx >= (int64_t(1) << 24))
      return set_error(PURIN_CP_ERR_UNSUPPORTED, "ldx must stay below 2^24");
    if (int rc = check_workspace(workspace, workspace_bytes,
                                 purin_train_expert_layer_workspace_bytes(
                                     dtype, tokens, experts, slots, width, hidden, outer_width)))
      return rc;
    const Up up{weights,     ldw, wdtype, (int32_t)tokens, (int32_t)experts, (int32_t)slots, activation,
                gated ? 1 : 0, ldx, width,  hidden,          0,                0};
    uint8_t* ws = (uint8_t*)workspace;
    return dtype == PURIN_TRAIN_BF16
               ? layer<bf16>((hipStream_t)stream, up, outer_width, (const bf16*)x, *inner, *outer, ws,
                             (bf16*)out)
               : layer<f16>((hipStream_t)stream, up, outer_width, (const f16*)x, *inner, *outer, ws,
                            (f16*)out);
  });
}

}  // extern "C"
