// A whole layer of experts for a few tokens (include/purin_train.h: expert_layer).
//
//   out(t) = sum over t's experts e of  w(t, e) f(x(t) A[e]) B[e]
//
// Every weight of an expert that some token has is read once: that is the work, and the tokens'
// rows are few beside it.  Three launches, or four:
//   choose  one workgroup chooses the tokens' experts and sorts the pairs (token, slot) by expert;
//           the others lay out x as the products read it, where it is not so already.  With few
//           pairs the next launch's workgroups do it themselves;
//   up      a workgroup has one expert and 64 columns of A (to 256, by the number of them):
//           multiplies its tokens' rows and applies f.  The results keep twice the type's digits,
//           as the sum of two numbers of the type, so that they take part in the second product as
//           they are;
//   down    the same of B: a row of 32-bit sums, times the token's weight, for each pair.  (The
//           weight before the second product would leave float16's range sooner.);
//   sum     adds a token's rows in the order of its slots.
// Bound by memory.  us and TB/s of weights, bf16: one token, 8 of 64 experts, 2048 x 1408 gated: up 24
// (3.8), down 11 (4.2), sum 4; 24 tokens, 4 of 32, 4096 x 1280 gated: choose 6, up 142-150 (4.3-4.5),
// down 63-67 (4.8-5.1), sum 4.5; 64 tokens, 6 of 64, 4096 x 1408 gated in codes: choose 11, up 99-105
// (3.7-4.0), down 63-66 (3.0), sum 4.5.  The contraction of down is short (44 blocks) for its streams'
// start and end.

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

// ---------------------------------------------------------------------------
// sums of BM rows and 2 x 32 columns
// ---------------------------------------------------------------------------

// The products' cores.  run(): rows a (piece k of row(i)), ``inner`` long, times expert e's matrix
// of ``outer`` columns, of which c are the wavefront's, to sums in LDS (part of its contraction).
// kRing: the LDS that it needs on the way.  First: the same of rows in one array.
template <typename T, int BM, int NA>
struct ThinCodes {
  using First = ThinCodes<T, BM, 1>;
  static constexpr int kRing = kLineLds;
  static constexpr bool kStreams = true;
  template <typename F>
  static __device__ __forceinline__ void run(const Rows (&a)[NA], F&& row, int64_t inner,
                                             const Matrices& w, int e, int64_t outer,
                                             const Columns& c, int part, int parts,
                                             unsigned char* lds) {
    const Codes b((const uint8_t*)w.values, w.scales, e * outer, inner);
    ThinAcc<BM> acc;
    int from, to;
    share_lines(0, c.n[0] > 0 ? b.lines() : 0, part, parts, from, to);
    StreamCodes<T, BM, NA>::run(a, row, inner, b, c, from, to, lds, acc);
    __syncthreads();
    thin_parts<BM>(acc, reinterpret_cast<float*>(lds));
  }
};

template <typename T, int BM, int NA>
struct ThinAlong {
  using First = ThinAlong<T, BM, 1>;
  static constexpr int kRing = kLineLds;
  static constexpr bool kStreams = true;
  template <typename F>
  static __device__ __forceinline__ void run(const Rows (&a)[NA], F&& row, int64_t inner,
                                             const Matrices& w, int e, int64_t, const Columns& c,
                                             int part, int parts, unsigned char* lds) {
    ThinAcc<BM> acc;
    int from, to;
    share_lines(0, c.n[0] > 0 ? (int)((inner + 63) / 64) : 0, part, parts, from, to);
    StreamDense<T, BM, NA>::run(a, row, inner, (const T*)w.values + e * w.se, w.ld, c, from, to, lds, acc);
    __syncthreads();
    thin_parts<BM>(acc, reinterpret_cast<float*>(lds));
  }
};

// Dense weights through LDS: a contraction that runs across memory (transposed by the reads), or
// pieces at any address.  Rows are in one piece each (step 16).
template <typename T, int BM, int NA, bool ALONG, bool DIRECT>
struct ThinDense {
  using First = ThinDense<T, BM, 1, ALONG, DIRECT>;
  static constexpr int X = BM / 32, S = 4, AHEAD = 3;
  using SA = PieceStage<BM, 8, 256>;
  using SB = Stage<T, 32, ALONG, 256>;
  static constexpr int kStage = NA * SA::kBytes + 2 * SB::kElems * 2;
  static constexpr int kLoads = NA * SA::kMine + 2 * SB::kMine;
  static constexpr int kRing = (DIRECT ? S : 2) * kStage;
  static constexpr bool kStreams = false;  // the wavefronts share a tile's columns, always in four

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
  static __device__ __forceinline__ void run(const Rows (&rows)[NA], F&& row, int64_t inner,
                                             const Matrices& w, int e, int64_t, const Columns& c,
                                             int, int, unsigned char* lds) {
    F16x acc[X][2];
#pragma unroll
    for (int x = 0; x < X; ++x)
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[x][y][r] = 0.0f;
    const T* a[NA];
#pragma unroll
    for (int i = 0; i < NA; ++i) a[i] = (const T*)rows[i].p;
    auto offset = [&](int i) {
      const int r = row(i);
      return r < 0 ? kOutside : (uint32_t)r * rows[0].pitch;
    };
    const T* base = (const T*)w.values + e * w.se;
    Side<T> b[2];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      // columns that are not there: the first ones again, whose sums are dropped
      const int from = !DIRECT && c.n[y] <= 0 ? 0 : y;
      b[y] = {base + (ALONG ? c.first[from] * w.ld : c.first[from]), w.ld, c.n[from],
              c.first[from] >= kVec<T>};
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
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float* sums = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int x = 0; x < X; ++x)
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
          *reinterpret_cast<F4*>(sums + (wave * BM + 32 * x + (lane & 31)) * kThinPitch + 32 * y + 2 * r +
                                 4 * (lane >> 5)) =
              F4{acc[x][y][r], acc[x][y][r + 1], acc[x][y][r + 2], acc[x][y][r + 3]};
    __syncthreads();
  }
};

// ---------------------------------------------------------------------------
// who has which expert
// ---------------------------------------------------------------------------

template <typename K>
struct AnyRow {
  const void* p;
  int32_t dtype;
  int64_t first;
  __device__ __forceinline__ K operator[](int e) const { return load_weight<K>(p, dtype, first + e); }
};

template <typename K, int G, int V>
__device__ __forceinline__ void choose_tokens(const void* weights, int32_t wdtype, int64_t ldw,
                                              int tokens, int experts, int slots, int32_t* ids,
                                              K* chosen) {
  for (int t = threadIdx.x / G; t < tokens; t += blockDim.x / G)
    choose<K, G, V>(AnyRow<K>{weights, wdtype, t * ldw}, experts, slots, (int)threadIdx.x % G,
                    ids + t * slots, chosen + t * slots);
}

// The pairs (token * slots + slot) sorted by expert.  Group number g of ``groups`` has expert[g]
// and the places start[g] to start[g + 1]; order, its pairs, in order; place, a pair's place or
// -1; weight, by place.
struct Plan {
  int32_t groups;
  int32_t expert[kPairs], start[kPairs + 1], order[kPairs], place[kPairs];
  float weight[kPairs];
};

// Made by one workgroup of 1024 threads from the choice in LDS.
template <typename K>
__device__ __forceinline__ void make_plan(const int32_t* ids, const K* chosen, int pairs, Plan* plan) {
  __shared__ int32_t first[PURIN_TRAIN_MAX_EXPERTS];  // a place for each expert, then its group's
  __shared__ int32_t wave_rows[16], wave_used[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  first[tid] = 0;
  __syncthreads();
  if (tid < pairs && ids[tid] >= 0) atomicAdd(&first[ids[tid]], 1);
  __syncthreads();
  const int count = first[tid];
  int rows = count, used = count > 0;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int r = __shfl_up(rows, d, 64), u = __shfl_up(used, d, 64);
    if (lane >= d) rows += r, used += u;
  }
  if (lane == 63) wave_rows[wave] = rows, wave_used[wave] = used;
  __syncthreads();
  int before_rows = 0, before_used = 0, all_rows = 0, all_used = 0;
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    if (v < wave) before_rows += wave_rows[v], before_used += wave_used[v];
    all_rows += wave_rows[v], all_used += wave_used[v];
  }
  const int start = before_rows + rows - count, group = before_used + used - 1;
  if (count) plan->expert[group] = tid, plan->start[group] = start;
  if (tid == 0) plan->groups = all_used, plan->start[all_used] = all_rows;
  first[tid] = start;
  __syncthreads();
  // a pair's place: behind the earlier pairs of its expert
  if (tid < pairs) {
    const int e = ids[tid];
    int place = -1;
    if (e >= 0) {
      place = first[e];
      const int4* four = reinterpret_cast<const int4*>(ids);
#pragma unroll 8
      for (int p = 0; p < tid / 4; ++p) {
        const int4 v = four[p];
        place += (v.x == e) + (v.y == e) + (v.z == e) + (v.w == e);
      }
      for (int p = tid & ~3; p < tid; ++p) place += ids[p] == e;
      plan->order[place] = tid;
      plan->weight[place] = (float)chosen[tid];
    }
    plan->place[tid] = place;
  }
}

struct Choose {
  const void* weights;
  int64_t ldw;
  int32_t wdtype, tokens, experts, slots;
  // x's rows, and where they go as whole pieces (NULL: they stay)
  const void* x;
  int64_t ldx, width;
  void* to;
};

// Few pairs: every workgroup of the first product makes the plan for itself, in LDS, which takes
// less than a launch (one token, 8 of 64 experts: 5.7 us for the launch, 2 here).  A layer's us so |
// with the launch, gated bf16: 1 token, 2 of 8 experts, 1024 x 512 17 | 21; 8, 4 of 32, 4096 x 1408 135
// | 143; 16, 8 of 64, 4096 x 1408 346 | 352; 32, 4 of 64, 1024 x 512 57 | 46.  In codes, two workgroups
// to a CU, the plans of one round after another show: 8, 4 of 32 (32 pairs, 1408 workgroups) 63.6 | 64.6;
// 16, 4 of 256, 512 x 256 (64, 512) 28.3 | 28.8; 16, 4 of 64, 1024 x 512 (64, 1024) 44 | 40; 16, 8 of 64
// (128, 1408) 151 | 141.  Between, by pairs times workgroups, gated: 8, 4 of 32, 4096 wide 24576 47.0 | 49.4,
// 32768 64.6 | 65.5, 40960 76.6 | 77.1; 16, 4 of 64, 1024 wide 32768 27.2 | 28.4, 40960 29.7 | 28.6, 49152
// 31.6 | 28.7, 57344 38.0 | 35.3; 16, 8 of 64, 4096 wide 40960 36.5 | 35.9, 49152 37.1 | 36.8, 57344
// 37.8 | 37.6.
constexpr int kOwnPairs = 128, kOwnTokens = 16, kOwnExperts = 256;
constexpr int64_t kOwnCodes = 48 * 1024;  // pairs times workgroups
struct OwnPlan {
  int32_t groups;
  int32_t expert[kOwnPairs], start[kOwnPairs + 1], order[kOwnPairs];
  float chosen[kOwnPairs];
  alignas(16) int32_t ids[kOwnPairs], first[kOwnPairs];  // first: an expert's first pair has it
};
__device__ __forceinline__ void make_own_plan(const Choose& p, OwnPlan& own, Plan* plan) {
  const int tid = threadIdx.x, pairs = p.tokens * p.slots;
  if (p.experts <= 64)
    choose_tokens<float, 16, 4>(p.weights, p.wdtype, p.ldw, p.tokens, p.experts, p.slots, own.ids,
                                own.chosen);
  else
    choose_tokens<float, 16, 16>(p.weights, p.wdtype, p.ldw, p.tokens, p.experts, p.slots, own.ids,
                                 own.chosen);
  if (tid >= pairs && tid < kOwnPairs) own.ids[tid] = -1;
  __syncthreads();
  // four pairs to a read, so that few of their latencies are in a row
  const int fours = (pairs + 3) / 4;
  int e = -1, below = 0, before = 0, all = 0;
  if (tid < kOwnPairs) {
    e = own.ids[tid];
#pragma unroll 4
    for (int q = 0; q < fours; ++q) {
      const int4 v = reinterpret_cast<const int4*>(own.ids)[q];
      all += (v.x >= 0) + (v.y >= 0) + (v.z >= 0) + (v.w >= 0);
      below += (uint32_t(v.x) < uint32_t(e)) + (uint32_t(v.y) < uint32_t(e)) +
               (uint32_t(v.z) < uint32_t(e)) + (uint32_t(v.w) < uint32_t(e));
      before += (v.x == e && 4 * q < tid) + (v.y == e && 4 * q + 1 < tid) +
                (v.z == e && 4 * q + 2 < tid) + (v.w == e && 4 * q + 3 < tid);
    }
    own.first[tid] = e >= 0 && before == 0 ? e : -1;
  }
  __syncthreads();
  const bool writes = blockIdx.x == 0;  // for the later launches
  if (tid < pairs) {
    int group = 0, groups = 0;
#pragma unroll 4
    for (int q = 0; q < fours; ++q) {
      const int4 v = reinterpret_cast<const int4*>(own.first)[q];
      groups += (v.x >= 0) + (v.y >= 0) + (v.z >= 0) + (v.w >= 0);
      group += (uint32_t(v.x) < uint32_t(e)) + (uint32_t(v.y) < uint32_t(e)) +
               (uint32_t(v.z) < uint32_t(e)) + (uint32_t(v.w) < uint32_t(e));
    }
    const bool first = own.first[tid] >= 0;
    const int place = e >= 0 ? below + before : -1;
    if (e >= 0) own.order[place] = tid;
    if (first) own.expert[group] = e, own.start[group] = below;
    if (tid == 0) own.groups = groups, own.start[groups] = all;
    if (writes) {
      plan->place[tid] = place;
      if (e >= 0) plan->weight[place] = own.chosen[tid];
      if (first) plan->expert[group] = e, plan->start[group] = below;
      if (tid == 0) plan->groups = groups, plan->start[groups] = all;
    }
  }
  __syncthreads();
}

template <typename T, typename K>
__global__ __launch_bounds__(1024) void k_layer_choose(Choose p, Plan* __restrict__ plan) {
  if (blockIdx.x) {
    const int64_t per = (p.width + 7) / 8, pieces = per * p.tokens;
    for (int64_t i = (int64_t)(blockIdx.x - 1) * 1024 + threadIdx.x; i < pieces;
         i += (int64_t)(gridDim.x - 1) * 1024)
      align_piece((const T*)p.x, p.ldx, p.width, i / per, i % per, (T*)p.to);
    return;
  }
  __shared__ K chosen[kPairs];
  __shared__ __align__(16) int32_t ids[kPairs];
  if (p.experts <= 64)
    choose_tokens<K, 16, 4>(p.weights, p.wdtype, p.ldw, p.tokens, p.experts, p.slots, ids, chosen);
  else if (p.experts <= 256)
    choose_tokens<K, 16, 16>(p.weights, p.wdtype, p.ldw, p.tokens, p.experts, p.slots, ids, chosen);
  else
    choose_tokens<K, 64, 16>(p.weights, p.wdtype, p.ldw, p.tokens, p.experts, p.slots, ids, chosen);
  __syncthreads();
  make_plan(ids, chosen, p.tokens * p.slots, plan);
}

template <int BM, typename Core>
constexpr int layer_lds() {
  return Core::kRing > kThinSums<BM> ? Core::kRing : kThinSums<BM>;
}
// A wavefront's columns of a tile, ``wide`` to each set of ``parts`` wavefronts, and its part.
// The second 32 of a gated product lie ``hidden`` behind the first.
struct Share {
  Columns c;
  int part;
};
__device__ __forceinline__ Share share_columns(int64_t tile, int parts, int wide, int64_t columns,
                                               bool gated) {
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int64_t col = (tile * (4 / parts) + wave / parts) * wide;
  Share s;
  s.part = wave % parts;
  s.c.first[0] = min(col, columns);
  s.c.n[0] = (int)max<int64_t>(0, min<int64_t>(32, columns - col));
  s.c.first[1] = gated ? columns + s.c.first[0] : min(col + 32, columns);
  s.c.n[1] = gated ? s.c.n[0] : (int)max<int64_t>(0, min<int64_t>(32, columns - col - 32));
  return s;
}

// The group and tile of a workgroup, XCD by XCD (number i is on XCD i % 8): neighbouring tiles,
// which may share lines of memory, run side by side.  The groups shared out are those there are.
__device__ __forceinline__ bool find_item(int64_t tiles, int groups, int& group, int& tile) {
  const int64_t n = groups * tiles, per = (n + 7) / 8, in = blockIdx.x >> 3;
  const int64_t at = (blockIdx.x & 7) * per + in;
  if (in >= per || at >= n) return false;
  group = (int)(at / tiles);
  tile = (int)(at - group * tiles);
  return true;
}

struct Up {
  int32_t slots, act, gated, parts;
  int64_t width, hidden, tiles;
  Rows x;
  uint32_t step, pitch;  // of the hidden rows, by place
};

// Workgroup: group number blockIdx.x / tiles, columns of tile blockIdx.x % tiles.
template <typename T, int BM, typename Core, bool OWN>
__global__ __launch_bounds__(256, 2) void k_layer_up(Up p, Choose choose, Matrices w, Plan* plan,
                                                     uint8_t* __restrict__ high,
                                                     uint8_t* __restrict__ low) {
  extern __shared__ __align__(16) unsigned char lds16[];
  __shared__ std::conditional_t<OWN, OwnPlan, int> made;
  const auto& from = [&]() -> const auto& {
    if constexpr (OWN) {
      make_own_plan(choose, made, plan);
      return made;
    } else {
      return *plan;
    }
  }();
  const int tid = threadIdx.x;
  int at, tile;
  if (!find_item(p.tiles, from.groups, at, tile)) return;
  const int e = __builtin_amdgcn_readfirstlane(from.expert[at]);
  const int start = __builtin_amdgcn_readfirstlane(from.start[at]);
  const int count = __builtin_amdgcn_readfirstlane(from.start[at + 1]) - start;
  const int parts = Core::kStreams ? p.parts : 4, wide = p.gated ? 32 : 64;
  const int64_t col = (int64_t)tile * (4 / parts) * wide;
  const Share own = share_columns(tile, parts, wide, p.hidden, p.gated);
  for (int r0 = 0; r0 < count; r0 += BM) {
    const Rows a[1] = {p.x};
    Core::run(a, [&](int r) { return r0 + r < count ? from.order[start + r0 + r] / p.slots : -1; },
              p.hidden ? p.width : 0, w, e, p.gated ? 2 * p.hidden : p.hidden, own.c, own.part, parts,
              lds16);
    const float* sums = reinterpret_cast<const float*>(lds16);
    const int rows = min(BM, count - r0);
    const int per = 4 / parts * (wide / 8);  // pieces of a row
    for (int i = tid; i < rows * per; i += 256) {
      const int r = i % rows, j = i / rows * 8, place = start + r0 + r;
      if (col + j >= p.hidden) continue;
      const int at = p.gated ? (j >> 5 << 6) + (j & 31) : j;  // of the sums
      Pack<T> hi, lo;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        float h = activation<T>(p.act, thin_sum<BM>(sums, parts, r, at + q));
        if (p.gated) h *= thin_sum<BM>(sums, parts, r, at + 32 + q);
        if (col + j + q >= p.hidden) h = 0.0f;
        hi.v[q] = (T)h;
        const float rest = h - (float)hi.v[q];
        lo.v[q] = (T)(fabsf((float)hi.v[q]) < __builtin_inff() ? rest : 0.0f);
      }
      const int64_t to = (col + j) / 8 * p.step + (int64_t)place * p.pitch;
      store16(reinterpret_cast<T*>(high + to), hi);
      store16(reinterpret_cast<T*>(low + to), lo);
    }
    __syncthreads();
  }
}

struct Down {
  int64_t hidden, outer, tiles;
  uint32_t step, pitch;
  int32_t parts;
};

template <typename T, int BM, typename Core>
__global__ __launch_bounds__(256, 2) void k_layer_down(
    Down p, const uint8_t* __restrict__ high, const uint8_t* __restrict__ low, Matrices w,
    const Plan* __restrict__ plan, float* __restrict__ out) {
  extern __shared__ __align__(16) unsigned char lds16[];
  const int tid = threadIdx.x;
  int at, tile;
  if (!find_item(p.tiles, plan->groups, at, tile)) return;
  const int e = plan->expert[at], start = plan->start[at], count = plan->start[at + 1] - start;
  const int parts = Core::kStreams ? p.parts : 4, wide = 64 * (4 / parts);
  const int64_t col = (int64_t)tile * wide;
  const Share own = share_columns(tile, parts, 64, p.outer, false);
  const int n = (int)min<int64_t>(wide, p.outer - col);
  for (int r0 = 0; r0 < count; r0 += BM) {
    const Rows a[2] = {{high, p.step, p.pitch}, {low, p.step, p.pitch}};
    auto row = [&](int r) { return r0 + r < count ? start + r0 + r : -1; };
    Core::run(a, row, p.hidden, w, e, p.outer, own.c, own.part, parts, lds16);
    const float* sums = reinterpret_cast<const float*>(lds16);
    auto sums_of = [&](auto&& f) {  // f(number in the expert's rows, column, 4 sums)
      for (int i = tid; i < min(BM, count - r0) * (wide / 4); i += 256) {
        const int r = i / (wide / 4), j = i % (wide / 4) * 4;
        if (j >= n) continue;
        F4 v;
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = thin_sum<BM>(sums, parts, r, j + q);
        f(start + r0 + r, j, v);
      }
    };
    bool odd = false;
    sums_of([&](int at, int j, const F4& s) {
      const float weight = plan->weight[at];
      Pack<float> v;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        odd |= !(fabsf(s[q]) < __builtin_inff());
        v.v[q] = s[q] * weight;
      }
      store_upto(out + at * p.outer + col + j, v, n - j);
    });
    // An infinite weight times a low part that is zero, or of the other sign, makes NaN of an
    // infinity.  Where there are such sums, once more with the high parts alone: theirs that are
    // not finite stand.  (Sums of their own for the low parts all the time take more registers than
    // there are.)
    if (__syncthreads_or(odd)) {
      const Rows first[1] = {a[0]};
      Core::First::run(first, row, p.hidden, w, e, p.outer, own.c, own.part, parts, lds16);
      sums_of([&](int at, int j, const F4& s) {
        const float weight = plan->weight[at];
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (j + q < n && !(fabsf(s[q]) < __builtin_inff()))
            out[at * p.outer + col + j + q] = s[q] * weight;
      });
      __syncthreads();
    }
  }
}

// A token's rows added up in the order of its slots.
template <typename T>
__global__ __launch_bounds__(256) void k_layer_sum(const float* __restrict__ parts,
                                                   const Plan* __restrict__ plan, int slots,
                                                   int64_t outer, T* __restrict__ out) {
  const int64_t t = blockIdx.y, j = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (j >= outer) return;
  float sum[4] = {0, 0, 0, 0};
  for (int s = 0; s < slots; ++s) {
    const int64_t place = plan->place[t * slots + s];
    if (place < 0) continue;
    const Pack<float> v = load_upto(parts + place * outer + j, outer - j);
#pragma unroll
    for (int q = 0; q < 4; ++q) sum[q] += v.v[q];
  }
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (j + q < outer) out[t * outer + j + q] = (T)sum[q];
}

// The workspace's parts, each at 256 bytes.
struct LayerSpace {
  int64_t pieces, plan, high, low, parts, x, bytes;
  LayerSpace(int64_t tokens, int64_t slots, int64_t width, int64_t hidden, int64_t outer) {
    const int64_t pairs = tokens * slots;
    pieces = (hidden + 7) / 8;  // of a hidden row
    plan = 0;
    high = plan + whole256(sizeof(Plan));
    low = high + whole256(pairs * pieces * 16);
    parts = low + whole256(pairs * pieces * 16);
    x = parts + whole256(pairs * outer * 4);
    bytes = x + aligned_bytes(tokens, width);
  }
};

// How an expert's matrices are read.
enum Reading { kCodes, kAlongDirect, kAcrossDirect, kAlong, kAcross };
static Reading reading(const purin_train_matrices& m, int64_t inner, int64_t outer, int64_t half,
                       int64_t* ld) {
  if (m.scales) {
    *ld = 0;
    return kCodes;
  }
  const bool along = along_inner(inner, m.si, m.so);
  *ld = along ? m.so : m.si;
  const bool direct = direct_ok(m.values, *ld, along ? inner : outer) && m.se % 8 == 0 &&
                      (along || half % 8 == 0);
  return along ? (direct ? kAlongDirect : kAlong) : (direct ? kAcrossDirect : kAcross);
}
// Calls f with a tile's rows and the core of a reading.
template <typename T, int NA, typename F>
static int by_reading(Reading how, int height, F&& f) {
  if (how == kCodes)
    return height == 16 ? f(i16, ThinCodes<T, 16, NA>{}) : f(i32, ThinCodes<T, 32, NA>{});
  if (how == kAlongDirect)
    return height == 16 ? f(i16, ThinAlong<T, 16, NA>{}) : f(i32, ThinAlong<T, 32, NA>{});
  auto rest = [&](auto bm) {
    constexpr int BM = bm;
    if (how == kAcrossDirect) return f(bm, ThinDense<T, BM, NA, false, true>{});
    if (how == kAlong) return f(bm, ThinDense<T, BM, NA, true, false>{});
    return f(bm, ThinDense<T, BM, NA, false, false>{});
  };
  return height <= 32 ? rest(i32) : rest(i64);
}

struct Shape {
  int64_t tokens, experts, slots, width, hidden, outer;
  int32_t act, gated;
};

template <typename T>
static int layer(hipStream_t st, const Shape& s, const void* weights, int32_t wdtype, int64_t ldw,
                 const T* x, int64_t ldx, const purin_train_matrices& inner,
                 const purin_train_matrices& outer, uint8_t* ws, T* out) {
  const LayerSpace at(s.tokens, s.slots, s.width, s.hidden, s.outer);
  const int64_t pairs = s.tokens * s.slots, groups = std::min(s.experts, pairs);
  if (s.tokens == 1) ldx = 0;  // one row has any pitch
  Plan* plan = (Plan*)(ws + at.plan);
  uint8_t *high = ws + at.high, *low = ws + at.low;
  float* parts = (float*)(ws + at.parts);
  Matrices a{inner.values, (const uint8_t*)inner.scales, inner.se, 0};
  Matrices b{outer.values, (const uint8_t*)outer.scales, outer.se, 0};
  const Reading how_a = reading(inner, s.width, s.gated ? 2 * s.hidden : s.hidden, s.hidden, &a.ld);
  const Reading how_b = reading(outer, s.hidden, s.outer, 8, &b.ld);

  // hidden rows: side by side where the second product streams, else each in one piece
  const bool side = how_b <= kAlongDirect;
  const uint32_t step = side ? (uint32_t)pairs * 16u : 16u, pitch = side ? 16u : (uint32_t)(at.pieces * 16);
  // streams of 64 columns, and the workgroups' tiles of them
  const int64_t wide = s.gated ? 32 : 64, streams_a = std::max<int64_t>(1, (s.hidden + wide - 1) / wide);
  const int64_t streams_b = (s.outer + 63) / 64;
  const int parts_a = how_a <= kAlongDirect ? stream_parts(groups * streams_a) : 4;
  const int parts_b = how_b <= kAlongDirect ? stream_parts(groups * streams_b) : 4;
  auto tiles = [](int64_t streams, int parts) { return (streams * parts + 3) / 4; };
  Up up{(int32_t)s.slots, s.act, s.gated, parts_a, s.width, s.hidden, tiles(streams_a, parts_a),
        {x, 16u, (uint32_t)(ldx * 2)}, step, pitch};
  Choose choose{weights, ldw, wdtype, (int32_t)s.tokens, (int32_t)s.experts, (int32_t)s.slots, x, ldx,
                s.width, nullptr};
  int64_t moves = 0;
  // rows whose pieces lie anywhere move to 16 bytes, but for the core that takes those too
  if (s.width && !direct_ok(x, ldx, s.width) && how_a != kAlong && how_a != kAcross) {
    const int64_t pieces = (s.width + 7) / 8;
    choose.to = ws + at.x;
    up.x = {choose.to, 16u, (uint32_t)pieces * 16u};
    moves = (pieces * s.tokens + 1023) / 1024;
  }
  const bool own = s.tokens <= kOwnTokens && pairs <= kOwnPairs && s.experts <= kOwnExperts &&
                   !moves && wdtype != PURIN_TRAIN_F64 &&
                   (how_a != kCodes || pairs * groups * up.tiles <= kOwnCodes);
  if (!own) {
    const dim3 grid((unsigned)(1 + moves));
    if (wdtype == PURIN_TRAIN_F64)
      k_layer_choose<T, double><<<grid, dim3(1024), 0, st>>>(choose, plan);
    else
      k_layer_choose<T, float><<<grid, dim3(1024), 0, st>>>(choose, plan);
    if (int rc = launched("k_layer_choose")) return rc;
  }

  // Rows of a tile; an expert with more reads its weights again.  64 tokens, 4096 x 1408 gated, us
  // with 16 | 32 rows: 6 of 64 experts in codes 163 | 188, dense 407 | 413; 6 of 32 127 | 127, 245 |
  // 224; 6 of 16 100 | 80, 198 | 133.  32 | 64 through LDS: 6 of 16 155 | 159, 4 of 8 111 | 92.
  const int height = pairs <= 8 * s.experts || s.tokens <= 16 ? 16
                     : pairs <= 24 * s.experts || s.tokens <= 32 ? 32 : 64;
  if (int rc = by_reading<T, 1>(how_a, height, [&](auto bm, auto core) {
        using Core = decltype(core);
        auto kernel = k_layer_up<T, bm, Core, false>;
        // as few tokens have tiles of few rows
        if constexpr (bm == (Core::kStreams ? 16 : 32))
          if (own) kernel = k_layer_up<T, bm, Core, true>;
        return launch16("k_layer_up", kernel, (groups * up.tiles + 7) / 8 * 8, 1, 1, 256,
                        layer_lds<bm, Core>(), st, up, choose, a, plan, high, low);
      }))
    return rc;
  const Down down{s.hidden, s.outer, tiles(streams_b, parts_b), step, pitch, parts_b};
  if (int rc = by_reading<T, 2>(how_b, height, [&](auto bm, auto core) {
        using Core = decltype(core);
        return launch16("k_layer_down", k_layer_down<T, bm, Core>, (groups * down.tiles + 7) / 8 * 8, 1,
                        1, 256, layer_lds<bm, Core>(), st, down, (const uint8_t*)high,
                        (const uint8_t*)low, b, (const Plan*)plan, parts);
      }))
    return rc;
  k_layer_sum<T><<<dim3((unsigned)((s.outer + 1023) / 1024), (unsigned)s.tokens), dim3(256), 0, st>>>(
      parts, plan, (int)s.slots, s.outer, out);
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
  if (std::max({width, hidden, outer}) > PURIN_TRAIN_LAYER_WIDTH || 2 * hidden > PURIN_TRAIN_LAYER_WIDTH)
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
    if (int rc = check_matrices(inner, width, gated ? 2 * hidden : hidden)) return rc;
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
    const Shape s{tokens, experts, slots, width, hidden, outer_width, activation, gated ? 1 : 0};
    uint8_t* ws = (uint8_t*)workspace;
    return dtype == PURIN_TRAIN_BF16
               ? layer<bf16>((hipStream_t)stream, s, weights, wdtype, ldw, (const bf16*)x, ldx, *inner,
                             *outer, ws, (bf16*)out)
               : layer<f16>((hipStream_t)stream, s, weights, wdtype, ldw, (const f16*)x, ldx, *inner,
                            *outer, ws, (f16*)out);
  });
}

}  // extern "C"
