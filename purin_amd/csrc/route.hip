// Tokens to experts and back (include/purin_train.h: route, sort, dispatch, combine and
// their gradients).
//
// With e(t, j) and w(t, j) a token's chosen experts and weights, place(t, j) the pair's row
// among the pairs sorted stably by expert:
//   rows[place(t, j)] = x(t)                     g_x(t) = sum_j g_rows[place(t, j)]
//   out(t) = sum_j w(t, j) rows[place(t, j)]     g_rows[place(t, j)] = w(t, j) g_out(t)
//                                                g_w(t, j) = <g_out(t), rows[place(t, j)]>
// The order is made by counting: every chunk of pairs counts its experts, then every chunk
// places its pairs behind the earlier experts' and the earlier chunks'.  Ranks inside a
// wavefront come from ballots on the expert's bits, so the order is the pairs' own.
//
// Moving rows is bound by memory.  A token's row is read once for all its slots (dispatch), its
// gradient once for both of combine's gradients.  32768 tokens of 4 slots, 4096 bf16: dispatch
// 234 us (5.7 TB/s; part of its writes stay in the 256 MB cache), combine 292 (4.6) and without
// weights 275 (4.9), combine's gradients 481 (5.0).  With few tokens the launches count: choosing
// and sorting 1 token of 64 experts takes 5.6 us, dispatch and combine 3 each.

#include <algorithm>
#include <type_traits>

#include "choose.hpp"
#include "train.hpp"

namespace purin {
namespace train {

constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / 64;
constexpr int64_t kSortChunk = 2048;  // pairs of a workgroup, at least
constexpr int64_t kSortGroups = 256;  // workgroups, at most
// Pairs up to which one workgroup has them all, and no launch counts first (a whole route of 500
// tokens, 6 of 64 experts: 10.1 us for 13.4; 1000 tokens, 8 slots: 15.8 for 13.2).
constexpr int64_t kSortOne = 4096;

struct SortShape {
  int64_t chunk, groups;
};
static SortShape sort_shape(int64_t pairs) {
  if (pairs <= kSortOne)
    return {std::max<int64_t>(1, (pairs + kSortThreads - 1) / kSortThreads) * kSortThreads, 1};
  int64_t chunk = std::max<int64_t>(kSortChunk, (pairs + kSortGroups - 1) / kSortGroups);
  chunk = (chunk + kSortThreads - 1) / kSortThreads * kSortThreads;
  return {chunk, std::max<int64_t>(1, (pairs + chunk - 1) / chunk)};
}

// ---------------------------------------------------------------------------
// choosing a token's experts
// ---------------------------------------------------------------------------

template <typename T, int G, int V>
__global__ __launch_bounds__(256) void k_choose(const T* __restrict__ weights, int64_t ld,
                                                int64_t tokens, int experts, int slots,
                                                int32_t* __restrict__ ids,
                                                T* __restrict__ chosen) {
  const int lane = threadIdx.x % G;
  const int64_t step = (int64_t)gridDim.x * (256 / G);
  for (int64_t t = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G; t < tokens; t += step)
    choose<T, G, V>(weights + t * ld, experts, slots, lane, ids + t * slots, chosen + t * slots);
}

// Calls f with the fewest lanes that hold a token's weights in at most 16 registers each: fewer
// lanes, fewer exchanges.
template <typename F>
static int by_lanes(int experts, F&& f) {
  using std::integral_constant;
  constexpr integral_constant<int, 16> g16;
  if (experts <= 32) return f(g16, integral_constant<int, 2>{});
  if (experts <= 64) return f(g16, integral_constant<int, 4>{});
  if (experts <= 128) return f(g16, integral_constant<int, 8>{});
  if (experts <= 256) return f(g16, g16);
  return f(integral_constant<int, 64>{}, g16);
}

// g_weights(t, e) = g_chosen(t, j) where ids(t, j) = e, 0 elsewhere.  cx threads to a token, its
// experts cx apart; the token's slots are the same addresses in all of them.
template <typename T>
__global__ __launch_bounds__(256) void k_choose_vjp(const int32_t* __restrict__ ids,
                                                    const T* __restrict__ g_chosen,
                                                    int64_t tokens, int experts, int slots, int cx,
                                                    T* __restrict__ g_weights) {
  const int tx = threadIdx.x % cx;
  const int64_t step = (int64_t)gridDim.x * (256 / cx);
  for (int64_t t = (int64_t)blockIdx.x * (256 / cx) + threadIdx.x / cx; t < tokens; t += step)
    for (int e0 = tx; e0 < experts; e0 += 4 * cx) {
      T g[4] = {(T)0, (T)0, (T)0, (T)0};
      for (int j = 0; j < slots; ++j) {
        const int32_t e = ids[t * slots + j];
        const T v = g_chosen[t * slots + j];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (e == e0 + u * cx) g[u] = v;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (e0 + u * cx < experts) g_weights[t * experts + e0 + u * cx] = g[u];
    }
}

// ---------------------------------------------------------------------------
// sorting pairs by expert
// ---------------------------------------------------------------------------

// Experts given by the caller, with -1 for what names none.
template <typename I>
__global__ __launch_bounds__(256) void k_ids(const I* __restrict__ given, int64_t pairs,
                                             int experts, int32_t* __restrict__ ids) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= pairs) return;
  const I e = given[i];
  ids[i] = e >= 0 && e < experts ? (int32_t)e : -1;
}

// counts[g][e]: the pairs of chunk g that go to expert e.
__global__ __launch_bounds__(kSortThreads) void k_sort_count(const int32_t* __restrict__ ids,
                                                             int64_t pairs, int experts,
                                                             int64_t chunk,
                                                             int32_t* __restrict__ counts) {
  __shared__ int32_t hist[PURIN_TRAIN_MAX_EXPERTS];
  for (int e = threadIdx.x; e < experts; e += kSortThreads) hist[e] = 0;
  __syncthreads();
  const int64_t from = (int64_t)blockIdx.x * chunk, to = min(pairs, from + chunk);
  for (int64_t i = from + threadIdx.x; i < to; i += kSortThreads) {
    const int32_t e = ids[i];
    if (e >= 0) atomicAdd(&hist[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += kSortThreads)
    counts[(int64_t)blockIdx.x * experts + e] = hist[e];
}

// Places the pairs of one chunk: expert e's rows begin at the sum of all smaller experts'
// counts; the chunk's first pair of e follows the earlier chunks' pairs of e, a wavefront's
// first the earlier wavefronts'.  LDS: per-wavefront running places [kSortWaves][experts].
__device__ __forceinline__ void place_chunk(const int32_t* ids, int64_t pairs, int experts,
                                            int bits, int64_t chunk, int groups, int group,
                                            const int32_t* counts, int32_t* run, int32_t* offsets,
                                            int32_t* place, int32_t* source) {
  __shared__ int32_t total[PURIN_TRAIN_MAX_EXPERTS];
  __shared__ int32_t before[PURIN_TRAIN_MAX_EXPERTS];
  __shared__ int32_t wave_sum[kSortWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int e = tid; e < experts; e += kSortThreads) total[e] = before[e] = 0;
  for (int i = tid; i < kSortWaves * experts; i += kSortThreads) run[i] = 0;
  __syncthreads();
  const int64_t from = (int64_t)group * chunk, to = min(pairs, from + chunk);
  const int64_t part = chunk / kSortWaves;  // a multiple of 64
  const int64_t wfrom = from + wave * part, wto = min(to, wfrom + part);
  int32_t* mine = run + wave * experts;
  for (int64_t i = wfrom + lane; i < wto; i += 64) {
    const int32_t e = ids[i];
    if (e >= 0) atomicAdd(&mine[e], 1);
  }
  if (groups > 1) {
    const int n = groups * experts;
    for (int i = tid; i < n; i += kSortThreads) {
      const int32_t c = counts[i];
      const int g = i / experts, e = i - g * experts;
      if (c) {
        atomicAdd(&total[e], c);
        if (g < group) atomicAdd(&before[e], c);
      }
    }
  }
  __syncthreads();
  if (groups == 1) {
    for (int e = tid; e < experts; e += kSortThreads) {
      int32_t s = 0;
      for (int w = 0; w < kSortWaves; ++w) s += run[w * experts + e];
      total[e] = s;
    }
    __syncthreads();
  }
  // exclusive sums of the totals over the experts (at most one expert to a thread)
  int32_t mine_total = tid < experts ? total[tid] : 0;
  int32_t sum = mine_total;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int32_t up = __shfl_up(sum, d, 64);
    if (lane >= d) sum += up;
  }
  if (lane == 63) wave_sum[wave] = sum;
  __syncthreads();
  int32_t base = 0, all = 0;
  for (int w = 0; w < kSortWaves; ++w) {
    const int32_t s = wave_sum[w];
    if (w < wave) base += s;
    all += s;
  }
  if (tid < experts) {
    const int32_t first = base + sum - mine_total;
    if (group == 0) {
      offsets[tid] = first;
      if (tid == experts - 1) offsets[experts] = all;
    }
    int32_t next = first + before[tid];
    for (int w = 0; w < kSortWaves; ++w) {
      const int32_t c = run[w * experts + tid];
      run[w * experts + tid] = next;
      next += c;
    }
  }
  __syncthreads();
  volatile int32_t* next = mine;  // this wavefront's alone
  for (int64_t i0 = wfrom; i0 < wto; i0 += 64) {
    const int64_t i = i0 + lane;
    const int32_t e = i < wto ? ids[i] : -1;
    const uint32_t key = e >= 0 ? (uint32_t)e : (uint32_t)experts;
    uint64_t same = ~0ull;
    for (int b = 0; b < bits; ++b) {
      const bool on = (key >> b) & 1u;
      const uint64_t votes = __ballot(on);
      same &= on ? votes : ~votes;
    }
    int32_t p = -1;
    const int rank = __popcll(same & ((1ull << lane) - 1ull));
    if (e >= 0) p = next[e] + rank;
    __builtin_amdgcn_wave_barrier();
    if (e >= 0 && rank == 0) next[e] = p + __popcll(same);
    __builtin_amdgcn_wave_barrier();
    if (i < wto) {
      place[i] = p;
      if (e >= 0) source[p] = (int32_t)i;
    }
  }
  // the rows that no pair has
  for (int64_t i = max<int64_t>(from, all) + tid; i < to; i += kSortThreads) source[i] = -1;
}

__global__ __launch_bounds__(kSortThreads) void k_sort_place(
    const int32_t* __restrict__ ids, int64_t pairs, int experts, int bits, int64_t chunk,
    const int32_t* __restrict__ counts, int32_t* __restrict__ offsets,
    int32_t* __restrict__ place, int32_t* __restrict__ source) {
  extern __shared__ int32_t run[];
  place_chunk(ids, pairs, experts, bits, chunk, (int)gridDim.x, (int)blockIdx.x, counts, run,
              offsets, place, source);
}

// Both parts of a small route in one workgroup.
template <typename T, int G, int V>
__global__ __launch_bounds__(kSortThreads) void k_route(const T* __restrict__ weights, int64_t ld,
                                                        int64_t tokens, int experts, int slots,
                                                        int bits, int64_t chunk, int32_t* ids,
                                                        T* __restrict__ chosen,
                                                        int32_t* __restrict__ offsets,
                                                        int32_t* __restrict__ place,
                                                        int32_t* __restrict__ source) {
  extern __shared__ int32_t run[];
  const int lane = threadIdx.x % G;
  for (int64_t t = threadIdx.x / G; t < tokens; t += kSortThreads / G)
    choose<T, G, V>(weights + t * ld, experts, slots, lane, ids + t * slots, chosen + t * slots);
  __syncthreads();  // the choices are written and seen
  place_chunk(ids, tokens * slots, experts, bits, chunk, 1, 0, nullptr, run, offsets, place,
              source);
}

// Bits of the keys 0 .. experts, the last of which stands for none.
static int key_bits(int experts) {
  int bits = 1;
  while ((1 << bits) <= experts) ++bits;
  return bits;
}
static size_t sort_lds(int experts) { return (size_t)kSortWaves * experts * sizeof(int32_t); }

static int sort_pairs(hipStream_t st, int64_t pairs, int experts, const int32_t* ids, void* ws,
                      int32_t* offsets, int32_t* place, int32_t* source) {
  const SortShape s = sort_shape(pairs);
  const int bits = key_bits(experts);
  if (s.groups > 1) {
    k_sort_count<<<dim3((unsigned)s.groups), dim3(kSortThreads), 0, st>>>(
        ids, pairs, experts, s.chunk, (int32_t*)ws);
    if (int rc = launched("k_sort_count")) return rc;
  }
  const size_t lds = sort_lds(experts);
  if (lds > 32 * 1024)
    if (int rc = raise_lds_cap((const void*)k_sort_place, lds)) return rc;
  k_sort_place<<<dim3((unsigned)s.groups), dim3(kSortThreads), lds, st>>>(
      ids, pairs, experts, bits, s.chunk, (const int32_t*)ws, offsets, place, source);
  return launched("k_sort_place");
}

// ---------------------------------------------------------------------------
// moving rows
// ---------------------------------------------------------------------------

// Threads of a workgroup: cx along a row's 16-byte vectors, 256 / cx tokens.  From 64 on a
// wavefront has one token, whose places and weights are then scalar loads: as vector loads, the
// same address in every lane, they took as long as the rows (8192 tokens of 6 slots, 2048 bf16:
// 70 us for combine, 65 with scalar loads).
static int row_threads(int64_t width, int vec) {
  const int64_t n = (width + vec - 1) / vec;
  int cx = 8;
  while (cx < 256 && cx < n) cx *= 2;
  return cx;
}

// This thread's number among its token's, and its token.
template <bool WIDE>
__device__ __forceinline__ int64_t first_token(int cx, int& tx) {
  tx = threadIdx.x % cx;
  int k = threadIdx.x / cx;
  if constexpr (WIDE) k = __builtin_amdgcn_readfirstlane(k);
  return (int64_t)blockIdx.x * (256 / cx) + k;
}

template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void k_dispatch(const T* __restrict__ x, int64_t ldx,
                                                  int64_t tokens, int slots, int64_t width,
                                                  int cx, int64_t pairs,
                                                  const int32_t* __restrict__ total,
                                                  const int32_t* __restrict__ place,
                                                  T* __restrict__ rows) {
  int tx;
  const int64_t last = max(*total, 0), step = (int64_t)gridDim.x * (256 / cx);
  for (int64_t t = first_token<WIDE>(cx, tx); t < tokens; t += step) {
    const int32_t* at = place + t * slots;
    for (int64_t c = (int64_t)tx * kVec<T>; c < width; c += (int64_t)cx * kVec<T>) {
      const Pack<T> v = load_upto(x + t * ldx + c, width - c);
      for (int j = 0; j < slots; ++j) {
        const int64_t p = at[j];
        if (p >= 0 && p < pairs) store_upto(rows + p * width + c, v, width - c);
      }
      // the rows that no pair has, shared out over the tokens
      for (int64_t p = last + t; p < pairs; p += tokens)
        store_upto(rows + p * width + c, zeros16<T>(), width - c);
    }
  }
}

// How weights are read: none (ones), 32-bit, or by the type given at the call.
enum { kOnes = 0, kFloats = 1, kAny = 2 };
template <typename A, int W>
__device__ __forceinline__ A weight_at(const void* w, int32_t dtype, int64_t i) {
  if constexpr (W == kOnes) return A(1);
  else if constexpr (W == kFloats) return (A) reinterpret_cast<const float*>(w)[i];
  else return load_weight<A>(w, dtype, i);
}

template <typename T, bool WIDE, int W>
__global__ __launch_bounds__(256) void k_combine(const T* __restrict__ rows, int64_t ldr,
                                                 int64_t tokens, int slots, int64_t width, int cx,
                                                 int64_t pairs, const int32_t* __restrict__ place,
                                                 const void* __restrict__ weights, int32_t wdtype,
                                                 T* __restrict__ out) {
  using A = typename Elem<T>::Acc;
  constexpr int B = 4;  // rows in flight
  int tx;
  const int64_t step = (int64_t)gridDim.x * (256 / cx);
  // one 16-byte column: ``load`` reads it of a row
  auto column = [&](int64_t t, auto&& load) {
    Pack<T> r;
    A sum[kVec<T>];
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) sum[i] = A(0);
    for (int j0 = 0; j0 < slots; j0 += B) {
      Pack<T> v[B];
      A w[B];
      int64_t p[B], any = -1;
#pragma unroll
      for (int b = 0; b < B; ++b) {
        // read without a condition, so that one wait covers them all
        const int64_t i = t * slots + min(j0 + b, slots - 1);
        p[b] = place[i];
        w[b] = weight_at<A, W>(weights, wdtype, i);
      }
#pragma unroll
      for (int b = 0; b < B; ++b) {
        if (j0 + b >= slots || p[b] >= pairs) p[b] = -1;
        if (p[b] >= 0) any = p[b];
      }
      if (any < 0) continue;
      // the loads go out together: an empty slot's reads a row that another slot reads
#pragma unroll
      for (int b = 0; b < B; ++b) v[b] = load(p[b] >= 0 ? p[b] : any);
#pragma unroll
      for (int b = 0; b < B; ++b)
        if (p[b] >= 0) {
#pragma unroll
          for (int i = 0; i < kVec<T>; ++i) {
            if constexpr (W == kOnes) sum[i] += (A)v[b].v[i];
            else sum[i] += w[b] * (A)v[b].v[i];
          }
        }
    }
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) r.v[i] = (T)sum[i];
    return r;
  };
  for (int64_t t = first_token<WIDE>(cx, tx); t < tokens; t += step)
    for (int64_t c = (int64_t)tx * kVec<T>; c < width; c += (int64_t)cx * kVec<T>) {
      const int n = (int)min<int64_t>(width - c, kVec<T>);
      if (n == kVec<T>)
        store16(out + t * width + c, column(t, [&](int64_t p) { return load16(rows + p * ldr + c); }));
      else
        store_some(out + t * width + c,
                   column(t, [&](int64_t p) { return load_some(rows + p * ldr + c, n); }), n);
    }
}

// cx threads to a token (a power of two); beyond 64 their parts of a sum meet in LDS.
template <typename T, bool WIDE, int W>
__global__ __launch_bounds__(256) void k_combine_vjp(
    const T* __restrict__ g_out, int64_t ldg, const T* __restrict__ rows, int64_t ldr,
    int64_t tokens, int slots, int64_t width, int cx, int64_t pairs,
    const int32_t* __restrict__ total, const int32_t* __restrict__ place,
    const void* __restrict__ weights, int32_t wdtype, T* __restrict__ g_rows,
    void* __restrict__ g_weights) {
  using A = typename Elem<T>::Acc;
  constexpr int B = 4;  // slots at once
  __shared__ A part[2][4][B];
  int tx, turn = 0;
  const int64_t last = max(*total, 0), step = (int64_t)gridDim.x * (256 / cx);
  // a token's threads stay together, so the exchanges below are whole; with more than a
  // wavefront to a token the workgroup has one
  for (int64_t t = first_token<WIDE>(cx, tx); t < tokens; t += step) {
    for (int j0 = 0; j0 < slots; j0 += B) {
      A w[B], dot[B];
      int64_t at[B];
#pragma unroll
      for (int b = 0; b < B; ++b) {
        const int64_t i = t * slots + min(j0 + b, slots - 1);  // no condition: one wait for all
        at[b] = place[i];
        w[b] = weight_at<A, W>(weights, wdtype, i);
        dot[b] = A(0);
      }
#pragma unroll
      for (int b = 0; b < B; ++b)
        if (j0 + b >= slots || at[b] >= pairs) at[b] = -1;
      int64_t any = -1;
#pragma unroll
      for (int b = 0; b < B; ++b)
        if (at[b] >= 0) any = at[b];
      // one 16-byte column; an empty slot's load is of a row that another slot reads
      auto column = [&](auto&& load, auto&& store, int64_t c) {
        const Pack<T> go = load(g_out + t * ldg + c);
        Pack<T> y[B];
        if (g_weights) {
#pragma unroll
          for (int b = 0; b < B; ++b) y[b] = load(rows + (at[b] >= 0 ? at[b] : any) * ldr + c);
        }
        if (g_rows) {
#pragma unroll
          for (int b = 0; b < B; ++b) {
            if (at[b] < 0) continue;
            Pack<T> r;
#pragma unroll
            for (int i = 0; i < kVec<T>; ++i) r.v[i] = (T)(w[b] * (A)go.v[i]);
            store(g_rows + at[b] * width + c, r);
          }
        }
        if (g_weights) {
#pragma unroll
          for (int b = 0; b < B; ++b) {
            if (at[b] < 0) continue;
#pragma unroll
            for (int i = 0; i < kVec<T>; ++i) dot[b] += (A)go.v[i] * (A)y[b].v[i];
          }
        }
      };
      if (any >= 0)
        for (int64_t c = (int64_t)tx * kVec<T>; c < width; c += (int64_t)cx * kVec<T>) {
          const int n = (int)min<int64_t>(width - c, kVec<T>);
          if (n == kVec<T>)
            column([](const T* p) { return load16(p); },
                   [](T* p, const Pack<T>& v) { store16(p, v); }, c);
          else
            column([n](const T* p) { return load_some(p, n); },
                   [n](T* p, const Pack<T>& v) { store_some(p, v, n); }, c);
        }
      if (g_weights) {
#pragma unroll
        for (int b = 0; b < B; ++b)
          for (int m = min(cx, 64) >> 1; m > 0; m >>= 1) dot[b] += __shfl_xor(dot[b], m, 64);
        if (cx > 64) {
          if (tx % 64 == 0) {
#pragma unroll
            for (int b = 0; b < B; ++b) part[turn][tx / 64][b] = dot[b];
          }
          __syncthreads();
#pragma unroll
          for (int b = 0; b < B; ++b) {
            dot[b] = part[turn][0][b];
            for (int v = 1; v < 4; ++v) dot[b] += part[turn][v][b];
          }
          turn ^= 1;
        }
        if (tx == 0) {
#pragma unroll
          for (int b = 0; b < B; ++b)
            if (j0 + b < slots) store_weight<A>(g_weights, wdtype, t * slots + j0 + b, dot[b]);
        }
      }
    }
    if (g_rows)
      for (int64_t p = last + t; p < pairs; p += tokens)
        for (int64_t c = (int64_t)tx * kVec<T>; c < width; c += (int64_t)cx * kVec<T>)
          store_upto(g_rows + p * width + c, zeros16<T>(), width - c);
  }
}

static int check_pairs(int64_t tokens, int64_t experts, int64_t slots) {
  if (tokens < 0 || experts < 1 || slots < 1)
    return refuse("tokens must not be negative, experts and slots must be positive");
  if (experts > PURIN_TRAIN_MAX_EXPERTS)
    return set_error(PURIN_CP_ERR_UNSUPPORTED, "more than 1024 experts");
  if (tokens >= (int64_t(1) << 31) || tokens * slots >= (int64_t(1) << 31))
    return set_error(PURIN_CP_ERR_UNSUPPORTED, "tokens * slots must stay below 2^31");
  return PURIN_CP_OK;
}

}  // namespace train
}  // namespace purin

using namespace purin;
using namespace purin::train;

extern "C" {

int64_t purin_train_route_workspace_bytes(int64_t tokens, int64_t experts, int64_t slots) {
  int64_t need = -1;
  (void)guarded([&] {
    if (int rc = check_pairs(tokens, experts, slots)) return rc;
    const SortShape s = sort_shape(tokens * slots);
    need = s.groups > 1 ? s.groups * experts * (int64_t)sizeof(int32_t) : 0;
    return (int)PURIN_CP_OK;
  });
  return need;
}

int purin_train_route(void* stream, int32_t dtype, int64_t tokens, int64_t experts, int64_t slots,
                      const void* weights, int64_t ld, void* workspace, int64_t workspace_bytes,
                      int32_t* ids, void* chosen, int32_t* offsets, int32_t* place,
                      int32_t* source) {
  return guarded([&] {
    if (int rc = check_pairs(tokens, experts, slots)) return rc;
    if (!known_dtype(dtype)) return refuse("unknown dtype");
    if (slots > experts) return refuse("slots must not exceed experts");
    if (!offsets || (tokens && (!weights || !ids || !chosen || !place || !source)))
      return refuse("NULL array");
    if (ld < experts && tokens > 1) return refuse("the weights' row pitch is below experts");
    if (int rc = check_workspace(workspace, workspace_bytes,
                                 purin_train_route_workspace_bytes(tokens, experts, slots)))
      return rc;
    hipStream_t st = (hipStream_t)stream;
    const SortShape s = sort_shape(tokens * slots);
    const int bits = key_bits((int)experts);
    // one workgroup for both parts where each of its lane groups has few tokens (four at most):
    // one launch for two (1 token of 64 experts: 5.6 us for 3 and 4 in two launches)
    const bool small = s.groups == 1 && tokens * (experts > 256 ? 64 : 16) <= 4 * kSortThreads;
    if (tokens) {
      const int rc = by_dtype(dtype, [&](auto x) {
        using T = decltype(x);
        return by_lanes((int)experts, [&](auto gg, auto vv) {
          constexpr int G = gg, V = vv;
          if (small) {
            const size_t lds = sort_lds((int)experts);
            if (lds > 32 * 1024)
              if (int e = raise_lds_cap((const void*)k_route<T, G, V>, lds)) return e;
            k_route<T, G, V><<<dim3(1), dim3(kSortThreads), lds, st>>>(
                (const T*)weights, ld, tokens, (int)experts, (int)slots, bits, s.chunk, ids,
                (T*)chosen, offsets, place, source);
            return launched("k_route");
          }
          k_choose<T, G, V><<<grid_of(tokens, 256 / G), dim3(256), 0, st>>>(
              (const T*)weights, ld, tokens, (int)experts, (int)slots, ids, (T*)chosen);
          return launched("k_choose");
        });
      });
      if (rc || small) return rc;
    }
    return sort_pairs(st, tokens * slots, (int)experts, ids, workspace, offsets, place, source);
  });
}

int purin_train_sort(void* stream, int32_t wide, int64_t tokens, int64_t experts, int64_t slots,
                     const void* given, void* workspace, int64_t workspace_bytes, int32_t* ids,
                     int32_t* offsets, int32_t* place, int32_t* source) {
  return guarded([&] {
    if (int rc = check_pairs(tokens, experts, slots)) return rc;
    const int64_t pairs = tokens * slots;
    if (!offsets || (pairs && (!given || !ids || !place || !source))) return refuse("NULL array");
    if (int rc = check_workspace(workspace, workspace_bytes,
                                 purin_train_route_workspace_bytes(tokens, experts, slots)))
      return rc;
    hipStream_t st = (hipStream_t)stream;
    if (pairs) {
      const dim3 grid((unsigned)((pairs + 255) / 256));
      if (wide)
        k_ids<int64_t><<<grid, dim3(256), 0, st>>>((const int64_t*)given, pairs, (int)experts, ids);
      else
        k_ids<int32_t><<<grid, dim3(256), 0, st>>>((const int32_t*)given, pairs, (int)experts, ids);
      if (int rc = launched("k_ids")) return rc;
    }
    return sort_pairs(st, pairs, (int)experts, ids, workspace, offsets, place, source);
  });
}

int purin_train_route_vjp(void* stream, int32_t dtype, int64_t tokens, int64_t experts,
                          int64_t slots, const int32_t* ids, const void* g_chosen,
                          void* g_weights) {
  return guarded([&] {
    if (int rc = check_pairs(tokens, experts, slots)) return rc;
    if (!known_dtype(dtype)) return refuse("unknown dtype");
    if (!tokens) return (int)PURIN_CP_OK;
    if (!ids || !g_chosen || !g_weights) return refuse("NULL array");
    return by_dtype(dtype, [&](auto x) {
      using T = decltype(x);
      int cx = 8;
      while (cx < 64 && cx * 4 < experts) cx *= 2;
      k_choose_vjp<T><<<grid_of(tokens, 256 / cx), dim3(256), 0, (hipStream_t)stream>>>(
          ids, (const T*)g_chosen, tokens, (int)experts, (int)slots, cx, (T*)g_weights);
      return launched("k_choose_vjp");
    });
  });
}

int purin_train_dispatch(void* stream, int32_t dtype, int64_t tokens, int64_t experts,
                         int64_t slots, int64_t width, const void* x, int64_t ldx,
                         const int32_t* offsets, const int32_t* place, void* rows) {
  return guarded([&] {
    if (int rc = check_pairs(tokens, experts, slots)) return rc;
    if (!known_dtype(dtype)) return refuse("unknown dtype");
    if (width < 0) return refuse("width must not be negative");
    if (!tokens || !width) return (int)PURIN_CP_OK;
    if (!x || !offsets || !place || !rows) return refuse("NULL array");
    if (ldx < width && tokens > 1) return refuse("a row pitch is below the width");
    return by_dtype(dtype, [&](auto v) {
      using T = decltype(v);
      const int cx = row_threads(width, kVec<T>);
      auto go = [&](auto kernel) {
        kernel<<<grid_of(tokens, 256 / cx), dim3(256), 0, (hipStream_t)stream>>>(
            (const T*)x, ldx, tokens, (int)slots, width, cx, tokens * slots, offsets + experts,
            place, (T*)rows);
      };
      if (cx >= 64) go(k_dispatch<T, true>);
      else go(k_dispatch<T, false>);
      return launched("k_dispatch");
    });
  });
}

int purin_train_combine(void* stream, int32_t dtype, int32_t wdtype, int64_t tokens,
                        int64_t slots, int64_t width, const void* rows, int64_t ldr,
                        const int32_t* place, const void* weights, void* out) {
  return guarded([&] {
    if (int rc = check_pairs(tokens, 1, slots)) return rc;
    if (!known_dtype(dtype) || (weights && !known_dtype(wdtype))) return refuse("unknown dtype");
    if (width < 0) return refuse("width must not be negative");
    if (!tokens || !width) return (int)PURIN_CP_OK;
    if (!rows || !place || !out) return refuse("NULL array");
    if (ldr < width && tokens * slots > 1) return refuse("a row pitch is below the width");
    return by_dtype(dtype, [&](auto v) {
      using T = decltype(v);
      const int cx = row_threads(width, kVec<T>);
      auto go = [&](auto kernel) {
        kernel<<<grid_of(tokens, 256 / cx), dim3(256), 0, (hipStream_t)stream>>>(
            (const T*)rows, ldr, tokens, (int)slots, width, cx, tokens * slots, place, weights,
            wdtype, (T*)out);
      };
      if (cx < 64) {
        if (weights) go(k_combine<T, false, kAny>);
        else go(k_combine<T, false, kOnes>);
      } else if (!weights) {
        go(k_combine<T, true, kOnes>);
      } else if (wdtype == PURIN_TRAIN_F32) {
        go(k_combine<T, true, kFloats>);
      } else {
        go(k_combine<T, true, kAny>);
      }
      return launched("k_combine");
    });
  });
}

int purin_train_combine_vjp(void* stream, int32_t dtype, int32_t wdtype, int64_t tokens,
                            int64_t experts, int64_t slots, int64_t width, const void* g_out,
                            int64_t ldg, const void* rows, int64_t ldr, const int32_t* offsets,
                            const int32_t* place, const void* weights, void* g_rows,
                            void* g_weights) {
  return guarded([&] {
    if (int rc = check_pairs(tokens, experts, slots)) return rc;
    if (!known_dtype(dtype) || !known_dtype(wdtype)) return refuse("unknown dtype");
    if (width < 0) return refuse("width must not be negative");
    if (!tokens || (!g_rows && !g_weights)) return (int)PURIN_CP_OK;
    if (!offsets || !place || !weights || (width && (!g_out || (g_weights && !rows))))
      return refuse("NULL array");
    if ((ldg < width && tokens > 1) || (g_weights && ldr < width && tokens * slots > 1))
      return refuse("a row pitch is below the width");
    return by_dtype(dtype, [&](auto v) {
      using T = decltype(v);
      // a wavefront to a token; a workgroup where the tokens' wavefronts would leave most of the
      // 256 CUs' room empty
      int cx = row_threads(width, kVec<T>);
      if (cx > 64) cx = cx == 256 && tokens < 2048 ? 256 : 64;
      auto go = [&](auto kernel) {
        kernel<<<grid_of(tokens, 256 / cx), dim3(256), 0, (hipStream_t)stream>>>(
            (const T*)g_out, ldg, (const T*)rows, ldr, tokens, (int)slots, width, cx,
            tokens * slots, offsets + experts, place, weights, wdtype, (T*)g_rows, g_weights);
      };
      if (cx < 64) go(k_combine_vjp<T, false, kAny>);
      else if (wdtype == PURIN_TRAIN_F32) go(k_combine_vjp<T, true, kFloats>);
      else go(k_combine_vjp<T, true, kAny>);
      return launched("k_combine_vjp");
    });
  });
}

}  // extern "C"
