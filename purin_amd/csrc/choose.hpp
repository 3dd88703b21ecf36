// A token's experts from its weights: the largest positive ones, largest first (route.hip,
// layer.hip).
#pragma once

#include "train.hpp"

namespace purin {
namespace train {

// A positive number's bits ascend with it, NaN above infinity; 0 for what is not chosen.
__device__ __forceinline__ uint32_t weight_key(float v) {
  return v != v ? 0x7fc00000u : v > 0.0f ? __builtin_bit_cast(uint32_t, v) : 0u;
}
__device__ __forceinline__ uint64_t weight_key(double v) {
  return v != v ? 0x7ff8000000000000ull : v > 0.0 ? __builtin_bit_cast(uint64_t, v) : 0ull;
}
template <typename T>
struct Key {
  using K = uint32_t;
  static __device__ __forceinline__ K of(T v) { return weight_key((float)v); }
  static __device__ __forceinline__ T value(K k) { return (T)__builtin_bit_cast(float, k); }
};
template <>
struct Key<double> {
  using K = uint64_t;
  static __device__ __forceinline__ K of(double v) { return weight_key(v); }
  static __device__ __forceinline__ double value(K k) { return __builtin_bit_cast(double, k); }
};

// The value of the lane N further on in the 16 (around), without a trip through LDS.
template <int N>
__device__ __forceinline__ uint32_t around16(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + N, 0xf, 0xf, true);
}
template <int N>
__device__ __forceinline__ uint64_t around16(uint64_t v) {
  return ((uint64_t)around16<N>((uint32_t)(v >> 32)) << 32) | around16<N>((uint32_t)v);
}
// The largest value of a group of G lanes (16 or all 64), in all of them.
template <int G, typename K>
__device__ __forceinline__ K group_max(K v) {
  v = max(v, around16<8>(v));
  v = max(v, around16<4>(v));
  v = max(v, around16<2>(v));
  v = max(v, around16<1>(v));
  if constexpr (G == 64) {
    v = max(v, (K)__shfl_xor(v, 16, 64));
    v = max(v, (K)__shfl_xor(v, 32, 64));
  }
  return v;
}

// G lanes to a token, V weights to a lane (expert i * G + lane): slots times, the lanes'
// best by (weight, lowest expert), then the group's.  Bound by that chain: 32768 tokens, 4 of 128
// experts 11 us (13 with the exchanges through LDS), of which reading the weights takes 3.5.
template <typename T, int G, int V, typename R>
__device__ __forceinline__ void choose(const R& row, int experts, int slots, int lane,
                                       int32_t* ids, T* chosen) {
  using K = typename Key<T>::K;
  K key[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = i * G + lane;
    key[i] = e < experts ? Key<T>::of(row[e]) : K(0);
  }
  int32_t my_id = -1;
  K my_key = 0;
  for (int j = 0; j < slots; ++j) {
    K best = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (key[i] > best) {
        best = key[i];
        at = i;
      }
    // the largest weight, then the lowest expert that has it (the largest of the complements)
    const K top = group_max<G>(best);
    const int e = (int)~group_max<G>(best == top ? ~(uint32_t)(at * G + lane) : 0u);
    best = top;
    const int owner = e / G;  // the winner's register, in lane e % G
    if (best != 0 && e % G == lane) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i == owner) key[i] = 0;
    }
    if (j % G == lane) {
      my_id = best != 0 ? e : -1;
      my_key = best;
    }
    if (j % G == G - 1 || j == slots - 1) {  // G slots are written together
      const int base = j - j % G;
      if (base + lane < slots) {
        ids[base + lane] = my_id;
        chosen[base + lane] = my_key ? Key<T>::value(my_key) : (T)0;
      }
    }
  }
}

}  // namespace train
}  // namespace purin
