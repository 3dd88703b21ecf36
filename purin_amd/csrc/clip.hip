// The global norm of a list of gradients, their scaling to a largest norm, and the norm's gradient
// (include/purin_train.h: clip, norm_vjp).
//
//   norm = sqrt(sum over tensors and elements of g^2),  out = g * min(1, largest / norm)
//   d norm / d g = g / norm, taken as 0 where the norm is 0
//
// Two passes over the gradients, both bound by memory (10^9 bf16 elements in 290 tensors: 428 and
// 750 us, 5.1 TB/s together; 50,000 in 14: 4 and 4 us, and two launches).  The first leaves one sum of squares
// per workgroup; every workgroup of the second adds those sums up again, in the same order, so
// that no launch stands between the passes and the result does not depend on which workgroup
// came first.  Squares are summed in 64 bits: those of 32-bit and bfloat16 numbers leave the
// 32-bit range on both sides.  The tensors' addresses travel with the launch (kTable tensors
// each), so nothing is uploaded and nothing is kept.

#include <algorithm>
#include <vector>

#include "train.hpp"

namespace purin {
namespace train {

constexpr int kTable = 96;            // tensors of one launch: its arguments stay under 4 KiB
constexpr int kClipThreads = 512;
constexpr int64_t kSums = 2048;       // workgroups of a list's first pass, beyond one a launch
constexpr int64_t kClipChunk = 16384; // elements of a workgroup's piece: it takes every
                                      // gridDim-th piece of the launch's tensors

struct ClipTable {
  const void* in[kTable];
  void* out[kTable];
  int64_t count[kTable];
  int32_t first[kTable + 1];  // a tensor's first piece
  uint8_t dtype[kTable];
  int32_t tensors;
};
static_assert(sizeof(ClipTable) < 3800, "launch arguments");

// The tensor of a piece: the last whose first piece is not behind it.
__device__ __forceinline__ int tensor_of(const ClipTable& t, int32_t piece) {
  int lo = 0, hi = t.tensors - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= piece) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// The sum of one value per thread, in every thread, in an order of its own.
__device__ __forceinline__ double sum_all(double v, double* buf) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m, 64);
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < kClipThreads / 64; ++w) s += buf[w];
  return s;
}

template <typename T>
__device__ double squares(const T* p, int64_t n) {
  constexpr int V = kVec<T>, U = 4;
  double s[V];
#pragma unroll
  for (int i = 0; i < V; ++i) s[i] = 0.0;
  const int64_t step = (int64_t)kClipThreads * V;
  int64_t i = (int64_t)threadIdx.x * V;
  for (; i + (U - 1) * step + V <= n; i += U * step) {
    Pack<T> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load16(p + i + u * step);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const double x = (double)v[u].v[k];
        s[k] += x * x;
      }
  }
  for (; i < n; i += step) {
    const Pack<T> v = load_upto(p + i, n - i);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const double x = (double)v.v[k];
      s[k] += x * x;
    }
  }
  double all = 0.0;
#pragma unroll
  for (int k = 0; k < V; ++k) all += s[k];
  return all;
}

__global__ __launch_bounds__(kClipThreads) void k_squares(ClipTable t, double* __restrict__ sums) {
  __shared__ double buf[kClipThreads / 64];
  double s = 0.0;
  const int32_t pieces = t.first[t.tensors];
  for (int32_t piece = (int32_t)blockIdx.x; piece < pieces; piece += (int32_t)gridDim.x) {
    const int k = tensor_of(t, piece);
    const int64_t at = (int64_t)(piece - t.first[k]) * kClipChunk;
    const int64_t n = min(kClipChunk, t.count[k] - at);
    switch (t.dtype[k]) {
      case PURIN_TRAIN_F32: s += squares((const float*)t.in[k] + at, n); break;
      case PURIN_TRAIN_F64: s += squares((const double*)t.in[k] + at, n); break;
      case PURIN_TRAIN_BF16: s += squares((const bf16*)t.in[k] + at, n); break;
      default: s += squares((const f16*)t.in[k] + at, n); break;
    }
  }
  s = sum_all(s, buf);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

template <typename A, typename T>
__device__ void scale(const T* in, T* out, int64_t n, double factor) {
  constexpr int V = kVec<T>, U = 4;
  const A f = (A)factor;
  const int64_t step = (int64_t)kClipThreads * V;
  int64_t i = (int64_t)threadIdx.x * V;
  for (; i + (U - 1) * step + V <= n; i += U * step) {
    Pack<T> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load16(in + i + u * step);
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int k = 0; k < V; ++k) v[u].v[k] = (T)((A)v[u].v[k] * f);
      store16(out + i + u * step, v[u]);
    }
  }
  for (; i < n; i += step) {
    Pack<T> v = load_upto(in + i, n - i);
#pragma unroll
    for (int k = 0; k < V; ++k) v.v[k] = (T)((A)v.v[k] * f);
    store_upto(out + i, v, n - i);
  }
}

template <typename A>
__device__ __forceinline__ void scale_piece(const ClipTable& t, int k, int64_t at, int64_t n,
                                            double factor) {
  switch (t.dtype[k]) {
    case PURIN_TRAIN_F32: scale<A>((const float*)t.in[k] + at, (float*)t.out[k] + at, n, factor); break;
    case PURIN_TRAIN_F64: scale<double>((const double*)t.in[k] + at, (double*)t.out[k] + at, n, factor); break;
    case PURIN_TRAIN_BF16: scale<A>((const bf16*)t.in[k] + at, (bf16*)t.out[k] + at, n, factor); break;
    default: scale<A>((const f16*)t.in[k] + at, (f16*)t.out[k] + at, n, factor); break;
  }
}

// A factor that 32 bits hold with fewer bits, or not at all, multiplies in 64.
__device__ __forceinline__ void scale_by(const ClipTable& t, int k, int64_t at, int64_t n,
                                         double factor) {
  const double size = fabs(factor);
  if (size < 0x1p-100 || size > 0x1p100) scale_piece<double>(t, k, at, n, factor);
  else scale_piece<float>(t, k, at, n, factor);
}

// The norm from the first pass's sums; the first workgroup of the list's first launch
// writes it.  ``largest`` < 0: nothing else.
__global__ __launch_bounds__(kClipThreads) void k_scale(ClipTable t,
                                                        const double* __restrict__ sums,
                                                        int32_t n_sums, double largest,
                                                        int32_t norm_dtype,
                                                        void* __restrict__ norm_out) {
  __shared__ double buf[kClipThreads / 64];
  double s = 0.0;
  for (int32_t i = threadIdx.x; i < n_sums; i += kClipThreads) s += sums[i];
  const double norm = sqrt(sum_all(s, buf));
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0)
    store_weight<double>(norm_out, norm_dtype, 0, norm);
  if (largest < 0.0) return;
  // a NaN norm compares false and scales by NaN; an infinite one scales by zero
  const bool whole = norm <= largest;
  const double factor = whole ? 1.0 : largest / norm;
  const int32_t pieces = t.first[t.tensors];
  for (int32_t piece = (int32_t)blockIdx.x; piece < pieces; piece += (int32_t)gridDim.x) {
    const int k = tensor_of(t, piece);
    if (whole && t.in[k] == t.out[k]) continue;  // already what it should be
    const int64_t at = (int64_t)(piece - t.first[k]) * kClipChunk;
    const int64_t n = min(kClipChunk, t.count[k] - at);
    scale_by(t, k, at, n, factor);
  }
}

__device__ __forceinline__ double scalar_at(const void* p, int32_t dtype) {
  return dtype == PURIN_TRAIN_F64 ? *(const double*)p : (double)*(const float*)p;
}

// out = in * g_norm / norm.  Bound by memory, as the second pass above (10^9 bf16 elements in 290
// tensors: 755 us, 5.3 TB/s).
__global__ __launch_bounds__(kClipThreads) void k_norm_vjp(ClipTable t, int32_t norm_dtype,
                                                           const void* __restrict__ norm,
                                                           const void* __restrict__ g_norm) {
  const double length = scalar_at(norm, norm_dtype);
  const double factor = length == 0.0 ? 0.0 : scalar_at(g_norm, norm_dtype) / length;
  const int32_t pieces = t.first[t.tensors];
  for (int32_t piece = (int32_t)blockIdx.x; piece < pieces; piece += (int32_t)gridDim.x) {
    const int k = tensor_of(t, piece);
    const int64_t at = (int64_t)(piece - t.first[k]) * kClipChunk;
    scale_by(t, k, at, min(kClipChunk, t.count[k] - at), factor);
  }
}

// Outputs may stand in for their own inputs, and may overlap nothing else.
static int check_overlap(int64_t count, const purin_train_tensor* tensors) {
  struct Span {
    uintptr_t from, to;
    int64_t tensor;
    bool out;
  };
  std::vector<Span> spans;
  spans.reserve(2 * count);
  for (int64_t i = 0; i < count; ++i) {
    const purin_train_tensor& t = tensors[i];
    if (!t.count) continue;
    const uintptr_t n = (uintptr_t)(t.count * dtype_bytes(t.dtype));
    spans.push_back({(uintptr_t)t.out, (uintptr_t)t.out + n, i, true});
    if (t.in != t.out) spans.push_back({(uintptr_t)t.in, (uintptr_t)t.in + n, i, false});
  }
  std::sort(spans.begin(), spans.end(),
            [](const Span& a, const Span& b) { return a.from < b.from; });
  // the furthest end of any span so far, and of any output so far
  uintptr_t any = 0, outs = 0;
  for (const Span& s : spans) {
    if (s.from < (s.out ? any : outs))
      return refuse("tensor " + std::to_string(s.tensor) +
                    (s.out ? ": its output overlaps another tensor" : ": an output overlaps it"));
    any = std::max(any, s.to);
    if (s.out) outs = std::max(outs, s.to);
  }
  return PURIN_CP_OK;
}

static int64_t pieces_of(int64_t count) { return (count + kClipChunk - 1) / kClipChunk; }

// The tensors from..to - 1 of a list, which one launch takes.
struct Launch {
  int64_t from, to, pieces;
};
static int launches_of(int64_t count, const purin_train_tensor* tensors,
                       std::vector<Launch>& launches) {
  for (int64_t i = 0; i < count;) {
    const int64_t to = std::min<int64_t>(count, i + kTable);
    Launch l{i, to, 0};
    for (int64_t k = i; k < to; ++k) l.pieces += pieces_of(tensors[k].count);
    if (l.pieces >= (int64_t(1) << 31)) return refuse("too many elements");
    launches.push_back(l);
    i = to;
  }
  return PURIN_CP_OK;
}
static ClipTable table_of(const purin_train_tensor* tensors, const Launch& l) {
  ClipTable t{};
  int32_t first = 0;
  for (int64_t k = l.from; k < l.to; ++k) {
    const int j = (int)(k - l.from);
    t.in[j] = tensors[k].in;
    t.out[j] = tensors[k].out;
    t.count[j] = tensors[k].count;
    t.dtype[j] = (uint8_t)tensors[k].dtype;
    t.first[j] = first;
    first += (int32_t)pieces_of(tensors[k].count);
  }
  t.tensors = (int32_t)(l.to - l.from);
  t.first[t.tensors] = first;
  return t;
}

static int clip(hipStream_t st, int64_t count, const purin_train_tensor* tensors, double largest,
                double* sums, int32_t norm_dtype, void* norm) {
  std::vector<Launch> launches;
  if (int rc = launches_of(count, tensors, launches)) return rc;
  int64_t pieces = 0;
  for (const Launch& l : launches) pieces += l.pieces;
  if (launches.empty()) launches.push_back({0, 0, 0});
  // the first pass's workgroups, shared out by the launches' pieces
  int64_t n_sums = 0;
  for (const Launch& l : launches) {
    if (!l.pieces) continue;
    const int64_t share = 1 + (int64_t)((double)(kSums - 1) * l.pieces / std::max<int64_t>(pieces, 1));
    const int64_t groups = std::min(l.pieces, share);
    k_squares<<<dim3((unsigned)groups), dim3(kClipThreads), 0, st>>>(table_of(tensors, l),
                                                                       sums + n_sums);
    if (int rc = launched("k_squares")) return rc;
    n_sums += groups;
  }
  bool first = true;
  for (const Launch& l : launches) {
    if (!first && (largest < 0.0 || !l.pieces)) continue;
    const int64_t groups = largest < 0.0 ? 1 : std::min<int64_t>(std::max<int64_t>(l.pieces, 1), kSums);
    k_scale<<<dim3((unsigned)groups), dim3(kClipThreads), 0, st>>>(
        table_of(tensors, l), sums, (int32_t)n_sums, largest, norm_dtype, first ? norm : nullptr);
    if (int rc = launched("k_scale")) return rc;
    first = false;
  }
  return PURIN_CP_OK;
}

static int norm_vjp(hipStream_t st, int64_t count, const purin_train_tensor* tensors,
                    int32_t norm_dtype, const void* norm, const void* g_norm) {
  std::vector<Launch> launches;
  if (int rc = launches_of(count, tensors, launches)) return rc;
  for (const Launch& l : launches) {
    if (!l.pieces) continue;
    k_norm_vjp<<<dim3((unsigned)std::min(l.pieces, kSums)), dim3(kClipThreads), 0, st>>>(
        table_of(tensors, l), norm_dtype, norm, g_norm);
    if (int rc = launched("k_norm_vjp")) return rc;
  }
  return PURIN_CP_OK;
}

// A list whose outputs are written where ``writes``.
static int check_list(int64_t count, const purin_train_tensor* tensors, bool writes) {
  if (count < 0) return refuse("count must not be negative");
  if (count && !tensors) return refuse("NULL tensors");
  for (int64_t i = 0; i < count; ++i) {
    const purin_train_tensor& t = tensors[i];
    if (!known_dtype(t.dtype)) return refuse("unknown dtype");
    if (t.count < 0 || t.count >= (int64_t(1) << 44)) return refuse("a tensor's count is out of range");
    if (t.count && (!t.in || (writes && !t.out))) return refuse("NULL tensor");
  }
  return writes ? check_overlap(count, tensors) : (int)PURIN_CP_OK;
}

}  // namespace train
}  // namespace purin

using namespace purin;
using namespace purin::train;

extern "C" {

int64_t purin_train_clip_workspace_bytes(int64_t tensors) {
  int64_t need = -1;
  (void)guarded([&] {
    if (tensors < 0) return refuse("tensors must not be negative");
    // one sum per workgroup of the first pass: kSums, and one for each launch's rounding up
    need = (kSums + (tensors + kTable - 1) / kTable) * (int64_t)sizeof(double);
    return (int)PURIN_CP_OK;
  });
  return need;
}

int purin_train_clip(void* stream, int64_t count, const purin_train_tensor* tensors,
                     double largest, void* workspace, int64_t workspace_bytes,
                     int32_t norm_dtype, void* norm) {
  return guarded([&] {
    if (count < 0) return refuse("count must not be negative");
    if (!norm) return refuse("NULL norm");
    if (norm_dtype != PURIN_TRAIN_F32 && norm_dtype != PURIN_TRAIN_F64)
      return refuse("the norm is F32 or F64");
    if (largest != largest) return refuse("largest must be a number");
    if (int rc = check_workspace(workspace, workspace_bytes,
                                 purin_train_clip_workspace_bytes(count)))
      return rc;
    if (int rc = check_list(count, tensors, largest >= 0.0)) return rc;
    return clip((hipStream_t)stream, count, tensors, largest, (double*)workspace, norm_dtype,
                norm);
  });
}

int purin_train_norm_vjp(void* stream, int64_t count, const purin_train_tensor* tensors,
                         int32_t norm_dtype, const void* norm, const void* g_norm) {
  return guarded([&] {
    if (!norm || !g_norm) return refuse("NULL norm");
    if (norm_dtype != PURIN_TRAIN_F32 && norm_dtype != PURIN_TRAIN_F64)
      return refuse("the norm is F32 or F64");
    if (int rc = check_list(count, tensors, true)) return rc;
    return norm_vjp((hipStream_t)stream, count, tensors, norm_dtype, norm, g_norm);
  });
}

}  // extern "C"
