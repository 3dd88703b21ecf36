// Operands' stages through registers: the part that the 16-bit tiles (expert16.hpp) and the 32-
// and 64-bit ones (expert32.hpp) share.
//
// Whole stages load without a condition, so that no load waits for another's: a piece that
// reaches past the operand's rows is read further down and moved into place, one that is past
// them reads some that are there, since what it holds reaches no sum that is kept.  The last,
// partial stage of a contraction loads piece by piece, with zeros behind its end.
#pragma once

#include "train.hpp"

namespace purin {
namespace train {

// A pointer that is the same in all lanes, in scalar registers.
template <typename T>
__device__ __forceinline__ const T* uniform(const T* p) {
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)u);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(u >> 32));
  return reinterpret_cast<const T*>(((uint64_t)hi << 32) | lo);
}

// An operand of a tile: element (i, k) at p + i * ld + k where its contraction is contiguous
// (ALONG), at p + k * ld + i where its rows are; n rows are there.  ``before``: whether those
// that precede them in memory are rows of the same operand.
template <typename T>
struct Side {
  const T* p;
  int64_t ld;
  int n;
  bool before = false;
};

// The elements moved down by ``by`` places (below the full width), zeros behind.
template <typename T>
__device__ __forceinline__ Pack<T> moved(const Pack<T>& v, int by) {
  struct Two {
    uint64_t lo, hi;
  };
  Two x = __builtin_bit_cast(Two, v);
  const int bits = by * (int)sizeof(T) * 8;
  if (bits >= 64) {
    x.lo = x.hi >> (bits - 64);
    x.hi = 0;
  } else if (bits) {
    x.lo = (x.lo >> bits) | (x.hi << (64 - bits));
    x.hi >>= bits;
  }
  return __builtin_bit_cast(Pack<T>, x);
}

// The pieces of one operand of a stage.  Layout says which: kMine a thread, number m being row
// ``row`` (i, or k where the rows are contiguous) from element ``first`` on; piece() is false
// where a thread has no m-th.
template <typename T, int N, int D, bool ALONG, typename Layout>
struct Pieces {
  static constexpr int kMine = Layout::kMine;

  // Whether whole stages may take the way without conditions: a piece that reaches past the
  // rows has a full piece's room before the end; offsets inside a stage fit 32 bits.
  static __device__ __forceinline__ bool whole(const Side<T>& o) {
    return (ALONG || o.before || o.n >= kVec<T>) && o.ld < (int64_t(1) << 21);
  }
  // how far before the stage's first element the loads begin
  static __device__ __forceinline__ int lead(const Side<T>& o) {
    return ALONG ? 0 : max(0, kVec<T> - o.n);
  }
  // byte offsets from there, and the pieces that are moved into place
  static __device__ __forceinline__ uint32_t reach(const Side<T>& o, uint32_t (&off)[kMine]) {
    uint32_t move = 0;
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      int row, first;
      const bool in = Layout::piece(m, row, first);
      if (!in) row = first = 0;
      if constexpr (ALONG) {
        row = min(row, o.n - 1);
      } else {
        if (first >= o.n) first = 0;
        if (first + kVec<T> > o.n) {
          first = o.n - kVec<T>;
          move |= 1u << m;
        }
      }
      off[m] = ((uint32_t)row * (uint32_t)o.ld + (uint32_t)(first + lead(o))) * (uint32_t)sizeof(T);
    }
    return move;
  }
  static __device__ __forceinline__ void load(const T* p, const uint32_t (&off)[kMine],
                                              Pack<T> (&v)[kMine]) {
    // the address space said: a load that might be of LDS would be waited for as one
    typedef T V __attribute__((ext_vector_type(kVec<T>), aligned(sizeof(T))));
    const auto* at = (const __attribute__((address_space(1))) char*)p;
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      const V x = *(const __attribute__((address_space(1))) V*)(at + off[m]);
#pragma unroll
      for (int i = 0; i < kVec<T>; ++i) v[m].v[i] = x[i];
    }
  }
  // any stage, piece by piece
  static __device__ __forceinline__ void load_each(const Side<T>& o, const T* p, int64_t left,
                                                   Pack<T> (&v)[kMine]) {
#pragma unroll
    for (int m = 0; m < kMine; ++m) {
      int row, first;
      const bool in = Layout::piece(m, row, first);
      const int64_t rows = ALONG ? o.n : left, cols = ALONG ? left : o.n;
      if (!in || row >= rows || first >= cols) v[m] = zeros16<T>();
      else v[m] = load_upto(p + row * o.ld + first, cols - first);
    }
  }
};

// All stages of two operands, AHEAD of them on their way, each in registers of its own; a ring of
// S places in LDS.  multiply(a's stage, b's stage, number) follows each.
template <typename T, int D, typename SA, typename SB, int S, int AHEAD, typename F>
__device__ __forceinline__ void through_registers(const Side<T>& a, const Side<T>& b,
                                                  int64_t depth, T* lds, F&& multiply) {
  constexpr int kStage = SA::kElems + SB::kElems;
  const T *pa = uniform(a.p), *pb = uniform(b.p);
  const int64_t step_a = SA::kAlong ? D : D * a.ld, step_b = SB::kAlong ? D : D * b.ld;
  int now = 0;
  int64_t t = 0;
  const int64_t whole = SA::whole(a) && SB::whole(b) ? depth / D : 0;
  if (whole) {
    Pack<T> va[AHEAD][SA::kMine], vb[AHEAD][SB::kMine];
    uint32_t off_a[SA::kMine], off_b[SB::kMine];
    const uint32_t move_a = SA::reach(a, off_a), move_b = SB::reach(b, off_b);
    const int by_a = a.n % kVec<T> ? kVec<T> - a.n % kVec<T> : 0;
    const int by_b = b.n % kVec<T> ? kVec<T> - b.n % kVec<T> : 0;
    // without a condition here too, so that the waits count on it: past the last whole stage,
    // that one again
    int64_t at = 0;
    const T *from_a = pa - SA::lead(a), *from_b = pb - SB::lead(b);
    auto load = [&](int v) {
      SA::load(from_a + at * step_a, off_a, va[v]);
      SB::load(from_b + at * step_b, off_b, vb[v]);
      if (at + 1 < whole) ++at;
    };
    auto put = [&](int v, T* to) {
      SA::store_settled(move_a, by_a, va[v], to);
      SB::store_settled(move_b, by_b, vb[v], to + SA::kElems);
    };
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) load(s);
    put(0, lds);
    for (; t < whole; t += AHEAD) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (t + u >= whole) break;
        const int next = now + 1 == S ? 0 : now + 1;
        __syncthreads();
        load(u);
        multiply(lds + now * kStage, lds + now * kStage + SA::kElems, t + u);
        if (t + u + 1 < whole) put((u + 1) % AHEAD, lds + next * kStage);
        now = next;
      }
    }
    t = whole;
    pa += whole * step_a;
    pb += whole * step_b;
  }
  for (; t * D < depth; ++t) {
    Pack<T> va[SA::kMine], vb[SB::kMine];
    SA::load_each(a, pa, depth - t * D, va);
    SB::load_each(b, pb, depth - t * D, vb);
    pa += step_a;
    pb += step_b;
    SA::store(va, lds + now * kStage);
    SB::store(vb, lds + now * kStage + SA::kElems);
    __syncthreads();
    multiply(lds + now * kStage, lds + now * kStage + SA::kElems, t);
    now = now + 1 == S ? 0 : now + 1;
  }
  __syncthreads();
}

}  // namespace train
}  // namespace purin
