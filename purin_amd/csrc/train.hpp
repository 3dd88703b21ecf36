// Shared parts of the operators around the projection layer (include/purin_train.h):
// element types and their arithmetic, and vectors of 16 bytes at any address.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "../../include/purin_cp.h"
#include "../../include/purin_train.h"

namespace purin {

int set_error(int code, const std::string& msg);  // plan.hip
int hip_check(hipError_t e, const char* what);    // plan.hip
int raise_lds_cap(const void* kernel, size_t bytes);  // plan.hip

namespace train {

using bf16 = __bf16;
using f16 = _Float16;

// The type sums are held in, and the widest vector of one load: 16 bytes, read
// and written at the element's alignment (the memory pipeline takes it; an
// aligned row costs nothing for it and an odd one stays at full width).
template <typename T>
struct Elem {
  using Acc = float;
};
template <>
struct Elem<double> {
  using Acc = double;
};
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

template <typename T>
struct alignas(sizeof(T)) Pack {
  T v[kVec<T>];
};

template <typename T>
__device__ __forceinline__ Pack<T> load16(const T* p) {
  typedef T V __attribute__((ext_vector_type(kVec<T>), aligned(sizeof(T))));
  const V x = *reinterpret_cast<const V*>(p);
  Pack<T> r;
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) r.v[i] = x[i];
  return r;
}
template <typename T>
__device__ __forceinline__ void store16(T* p, const Pack<T>& r) {
  typedef T V __attribute__((ext_vector_type(kVec<T>), aligned(sizeof(T))));
  V x;
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) x[i] = r.v[i];
  *reinterpret_cast<V*>(p) = x;
}
// The first n elements of a vector (n below the full width), zeros behind them.
template <typename T>
__device__ __forceinline__ Pack<T> load_some(const T* p, int n) {
  Pack<T> r;
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) r.v[i] = i < n ? p[i] : (T)0;
  return r;
}
template <typename T>
__device__ __forceinline__ void store_some(T* p, const Pack<T>& r, int n) {
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i)
    if (i < n) p[i] = r.v[i];
}
template <typename T>
__device__ __forceinline__ Pack<T> load_upto(const T* p, int64_t n) {
  return n >= kVec<T> ? load16(p) : load_some(p, (int)n);
}
template <typename T>
__device__ __forceinline__ void store_upto(T* p, const Pack<T>& r, int64_t n) {
  if (n >= kVec<T>) store16(p, r);
  else store_some(p, r, (int)n);
}
template <typename T>
__device__ __forceinline__ Pack<T> zeros16() {
  Pack<T> r;
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) r.v[i] = (T)0;
  return r;
}

// A weight of any type as the sums' type.
template <typename A>
__device__ __forceinline__ A load_weight(const void* w, int32_t dtype, int64_t i) {
  switch (dtype) {
    case PURIN_TRAIN_F32: return (A) reinterpret_cast<const float*>(w)[i];
    case PURIN_TRAIN_F64: return (A) reinterpret_cast<const double*>(w)[i];
    case PURIN_TRAIN_BF16: return (A)(float)reinterpret_cast<const bf16*>(w)[i];
    default: return (A)(float)reinterpret_cast<const f16*>(w)[i];
  }
}
template <typename A>
__device__ __forceinline__ void store_weight(void* w, int32_t dtype, int64_t i, A v) {
  switch (dtype) {
    case PURIN_TRAIN_F32: reinterpret_cast<float*>(w)[i] = (float)v; break;
    case PURIN_TRAIN_F64: reinterpret_cast<double*>(w)[i] = (double)v; break;
    case PURIN_TRAIN_BF16: reinterpret_cast<bf16*>(w)[i] = (bf16)(float)v; break;
    default: reinterpret_cast<f16*>(w)[i] = (f16)(float)v; break;
  }
}

inline bool known_dtype(int32_t d) { return d >= PURIN_TRAIN_F32 && d <= PURIN_TRAIN_F16; }
inline int64_t dtype_bytes(int32_t d) {
  return d == PURIN_TRAIN_F64 ? 8 : d == PURIN_TRAIN_F32 ? 4 : 2;
}
inline int refuse(const std::string& msg) { return set_error(PURIN_CP_ERR_ARG, msg); }
inline int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? PURIN_CP_OK : hip_check(e, what);
}
// Workgroups for n items, ``per`` to a workgroup; the kernels' loops take what is left beyond
// 2^20 (a launch holds fewer than 2^32 threads).
inline dim3 grid_of(int64_t n, int64_t per) {
  const int64_t g = (n + per - 1) / per;
  return dim3((unsigned)(g < (1 << 20) ? g : (1 << 20)));
}
inline int check_workspace(const void* ws, int64_t have, int64_t need) {
  if (need <= 0) return PURIN_CP_OK;
  if (!ws || have < need)
    return refuse("workspace too small: the call needs " + std::to_string(need) + " bytes, " +
                  std::to_string(ws ? have : 0) + " given");
  if (reinterpret_cast<uintptr_t>(ws) % 256 != 0)
    return refuse("workspace must be 256-byte aligned");
  return PURIN_CP_OK;
}

// Calls f with a value of the element type of a known dtype.
template <typename F>
int by_dtype(int32_t dtype, F&& f) {
  switch (dtype) {
    case PURIN_TRAIN_F32: return f(float{});
    case PURIN_TRAIN_F64: return f(double{});
    case PURIN_TRAIN_BF16: return f(bf16{});
    default: return f(f16{});
  }
}

// What an entry point returns for an exception on the host (memory for a message
// or a table): nothing may leave the C boundary.
template <typename F>
int guarded(F&& f) noexcept {
  try {
    return f();
  } catch (...) {
    return PURIN_CP_ERR_NOMEM;
  }
}

}  // namespace train
}  // namespace purin
