// Parts that the kernels of microscaled numbers share (micro.hip, packed.hip, layer.hip): blocks,
// scales, elements, and the activation.
#pragma once

#include "train.hpp"

namespace purin {
namespace train {

constexpr int kFp4 = PURIN_TRAIN_FP4, kInt8 = PURIN_TRAIN_INT8;
template <int KIND>
constexpr int kMicroBits = KIND == kFp4 ? 4 : 8;

// Blocks of a row, and the scales that are held for it (whole words).
__host__ __device__ inline int micro_blocks(int64_t length) { return (int)((length + 31) / 32); }
__host__ __device__ inline int micro_filled(int blocks) { return (blocks + 3) & ~3; }

// Division of numbers below 2^31 by one that the host knows: a product and a shift.
struct Divider {
  uint32_t d, m, s;
  explicit Divider(uint32_t by) : d(by), s(0) {
    while ((uint64_t(1) << s) < by) ++s;
    m = (uint32_t)(((uint64_t(1) << 32) * ((uint64_t(1) << s) - by)) / by + 1);
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
};

// The bits of |x| in 32 bits: they ascend with it, infinities and NaN above all numbers.
__device__ __forceinline__ uint32_t magnitude(float x) {
  return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
}
// The largest of four neighbouring lanes, in all of them.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, true));  // 1 0 3 2
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, true));  // 2 3 0 1
}
// A block's scale from its largest magnitude.  A number below the normal ones has a zero here and
// a lower logarithm; the scale's range ends there as well.
template <int KIND>
__device__ __forceinline__ uint32_t micro_scale(uint32_t most) {
  if (most >= 0x7f800000u) return 255u;
  const int e = (int)(most >> 23) - (KIND == kFp4 ? 2 : 0);
  return (uint32_t)max(e, 0);
}
// 2^(scale - 127) as the conversions take it: they read the exponent, 0 as 2^-127 and 255 as NaN.
__device__ __forceinline__ float scale_operand(uint32_t scale) {
  return __builtin_bit_cast(float, scale << 23);
}

// 8 elements, written as 4 or 8 bytes; zeros beside a scale of 255.
template <int KIND>
__device__ __forceinline__ void store_codes(uint8_t* to, const float (&v)[8], uint32_t scale) {
  if constexpr (KIND == kFp4) {
    const float s = scale_operand(scale);
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], s, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], s, 3);
    *reinterpret_cast<uint32_t*>(to) = scale == 255u ? 0u : c;
  } else {
    uint32_t c[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = __builtin_rintf(__builtin_ldexpf(v[i], 133 - (int)scale));
      const int q = (int)fminf(fmaxf(x, -127.0f), 127.0f);
      c[i >> 2] |= ((uint32_t)q & 255u) << (8 * (i & 3));
    }
    *reinterpret_cast<uint2*>(to) = scale == 255u ? uint2{0, 0} : uint2{c[0], c[1]};
  }
}
// What 8 elements stand for.
template <int KIND>
__device__ __forceinline__ void load_codes(const uint8_t* from, uint32_t scale, float (&v)[8]) {
  if constexpr (KIND == kFp4) {
    const uint32_t c = *reinterpret_cast<const uint32_t*>(from);
    const float s = scale_operand(scale);
    typedef float F2 __attribute__((ext_vector_type(2)));
    const F2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0);
    const F2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
    const F2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2);
    const F2 e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3);
    v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1];
    v[4] = d[0], v[5] = d[1], v[6] = e[0], v[7] = e[1];
  } else {
    const uint2 c = *reinterpret_cast<const uint2*>(from);
    // 2^(scale - 133) by way of 64ths of the element, so that no factor leaves the range
    const float s = scale == 255u ? __builtin_nanf("") : __builtin_ldexpf(1.0f, (int)scale - 127);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int q = (int)((i < 4 ? c.x : c.y) << (24 - 8 * (i & 3))) >> 24;
      v[i] = (float)q * 0.015625f * s;
    }
  }
}

// f(u) for T's sums.  16-bit results take the reciprocal and exponential instructions, whose
// errors of a few 2^-24 are far below their rounding.
template <typename T>
__device__ __forceinline__ typename Elem<T>::Acc logistic(typename Elem<T>::Acc u) {
  if constexpr (sizeof(T) == 8) return 1.0 / (1.0 + exp(-u));
  else if constexpr (sizeof(T) == 4) return 1.0f / (1.0f + expf(-u));
  else return __builtin_amdgcn_rcpf(1.0f + __expf(-u));
}
template <typename A>
__device__ __forceinline__ A normal_share(A u) {  // of a normal distribution below u
  if constexpr (sizeof(A) == 8) return 0.5 * erfc(-u * 0.70710678118654752440);
  else return 0.5f * erfcf(-u * 0.70710678f);
}
template <typename T>
__device__ __forceinline__ typename Elem<T>::Acc activation(int act, typename Elem<T>::Acc u) {
  using A = typename Elem<T>::Acc;
  if (act == PURIN_TRAIN_RELU) return u > (A)0 || u != u ? u : (A)0;
  if (act == PURIN_TRAIN_SILU) return u * logistic<T>(u);
  return u * normal_share(u);
}
// f(u) and its derivative.
template <typename T>
__device__ __forceinline__ void activation_slope(int act, typename Elem<T>::Acc u,
                                                 typename Elem<T>::Acc& f,
                                                 typename Elem<T>::Acc& slope) {
  using A = typename Elem<T>::Acc;
  if (act == PURIN_TRAIN_RELU) {
    f = u > (A)0 || u != u ? u : (A)0;
    slope = u > (A)0 ? (A)1 : u != u ? u : (A)0;
  } else if (act == PURIN_TRAIN_SILU) {
    const A s = logistic<T>(u);
    f = u * s;
    slope = s * ((A)1 + u * ((A)1 - s));
  } else {
    const A p = normal_share(u);
    f = u * p;
    A density;
    if constexpr (sizeof(A) == 8) density = 0.39894228040143267794 * exp(-0.5 * u * u);
    else density = 0.39894228f * expf(-0.5f * u * u);
    slope = p + u * density;
  }
}

}  // namespace train
}  // namespace purin
