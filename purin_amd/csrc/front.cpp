// The torch front end of include/purin_train.h: argument checks, outputs from torch's allocator,
// the current stream, and the gradients as autograd nodes in C++.  A small call's time is the
// host's: the same front end over ctypes and Python autograd functions took 213 us for a training
// step of route, dispatch and combine whose kernels run for 20.
//
// No kernel is here; libpurin_cp.so, which this links to, holds them and knows nothing of torch.

#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <algorithm>
#include <numeric>
#include <optional>
#include <sstream>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/purin_cp.h"
#include "../../include/purin_train.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

// An error code and message of the library; Python sees purin_amd._lib.PurinError.
struct LibraryError : std::exception {
  int code;
  std::string message;
  explicit LibraryError(int c) : code(c), message(purin_cp_last_error()) {}
  LibraryError(int c, std::string m) : code(c), message(std::move(m)) {}
  const char* what() const noexcept override { return message.c_str(); }
};

void check(int code) {
  if (code != PURIN_CP_OK) throw LibraryError(code);
}
int64_t bytes(int64_t need) {
  if (need < 0) throw LibraryError(PURIN_CP_ERR_ARG);
  return need;
}

template <typename... A>
[[noreturn]] void refuse(const A&... parts) {
  std::ostringstream s;
  (s << ... << parts);
  throw py::value_error(s.str());
}

int32_t code_of(const Tensor& t, const char* name) {
  if (!t.is_cuda()) refuse(name, " must be a tensor on the GPU");
  switch (t.scalar_type()) {
    case at::kFloat: return PURIN_TRAIN_F32;
    case at::kDouble: return PURIN_TRAIN_F64;
    case at::kBFloat16: return PURIN_TRAIN_BF16;
    case at::kHalf: return PURIN_TRAIN_F16;
    default: refuse(name, " must be float32, float64, bfloat16 or float16; got ", t.scalar_type());
  }
}

void same_device(const Tensor& a, const Tensor& b, const char* name) {
  if (a.device() != b.device()) refuse(name, " must be on ", a.device(), "; got ", b.device());
}

// The numbers themselves in memory, where torch holds their negatives and a mark (the imaginary
// part of a conjugate).
Tensor numbers(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

// A matrix with adjacent elements in a row and rows that do not overlap.
Tensor matrix(const Tensor& given) {
  const Tensor t = numbers(given);
  if ((t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1)))
    return t.contiguous();
  return t;
}

// Forward-mode differentiation passes these operators by: a result without a tangent would read as
// one whose tangent is zero.
void without_tangent(const Tensor& t) {
  if (t.defined() && t._fw_grad(0).defined())
    throw LibraryError(PURIN_CP_ERR_UNSUPPORTED,
                       "forward-mode differentiation is not supported: a tensor has a tangent");
}
// A trace would hold the allocations of a call and not its kernels.
void outside_traces() {
  if (torch::jit::tracer::isTracing() ||
      c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY))
    throw LibraryError(PURIN_CP_ERR_UNSUPPORTED, "the operator cannot be traced");
}

// The device made current, and its current stream, for one entry point.
struct Call {
  c10::DeviceGuard guard;
  void* stream;
  explicit Call(const Tensor& t)
      : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {
    outside_traces();
  }
};

// A call's scratch: the caller's, or new memory, which the allocator gives to nothing else
// before the stream's kernels are done with it.
struct Workspace {
  Tensor held;
  void* at = nullptr;
  int64_t size = 0;
  Workspace(const std::optional<Tensor>& given, int64_t need, const Tensor& like) {
    if (given) {
      // a broadcast or strided tensor has fewer bytes in one piece than it has elements
      if (!given->is_cuda() || given->layout() != at::kStrided || !given->is_contiguous())
        refuse("workspace must be a contiguous device tensor");
      same_device(like, *given, "workspace");
      held = *given;
    } else if (bytes(need)) {
      held = at::empty({need}, like.options().dtype(at::kByte).requires_grad(false));
    } else {
      return;
    }
    at = held.data_ptr();
    size = (int64_t)held.nbytes();
  }
};

bool wants_grad(const Tensor& t) { return t.requires_grad() && at::GradMode::is_enabled(); }

// Gradients of gradients are not there: with a graph wanted of the backward pass, what it
// returns raises in its own.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list some;
  for (Tensor& g : grads)
    if (g.defined()) some.push_back(g.detach().requires_grad_());
  if (some.empty()) return grads;
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "this operator is differentiable once", (int64_t)some.size());
  some = (*node)(std::move(some));
  size_t k = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = some[k++];
  return grads;
}

// -- routing ------------------------------------------------------------------------------

struct Index {
  Tensor ids, offsets, place, source;
};

Index new_index(int64_t tokens, int64_t count, int64_t slots, const Tensor& like) {
  const int64_t pairs = tokens * slots;
  const auto o = like.options().dtype(at::kInt).requires_grad(false);
  return {at::empty({tokens, slots}, o), at::empty({count + 1}, o), at::empty({tokens, slots}, o),
          at::empty({pairs}, o)};
}

int32_t* ints(const Tensor& t) { return (int32_t*)t.data_ptr(); }

Tensor run_route(const Tensor& weights, int64_t slots, const std::optional<Tensor>& workspace,
                 Index* index) {
  const Tensor w = matrix(weights);
  const int64_t tokens = w.size(0), count = w.size(1);
  const Call call(w);
  const Workspace ws(workspace, purin_train_route_workspace_bytes(tokens, count, slots), w);
  *index = new_index(tokens, count, slots, w);
  Tensor chosen = at::empty({tokens, slots}, w.options().requires_grad(false));
  check(purin_train_route(call.stream, code_of(w, "weights"), tokens, count, slots, w.data_ptr(),
                          w.stride(0), ws.at, ws.size, ints(index->ids), chosen.data_ptr(),
                          ints(index->offsets), ints(index->place), ints(index->source)));
  return chosen;
}

struct RouteFn : torch::autograd::Function<RouteFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& weights, int64_t slots,
                        const std::optional<Tensor>& workspace, Index* index) {
    Tensor chosen = run_route(weights, slots, workspace, index);
    ctx->save_for_backward({index->ids});
    ctx->saved_data["count"] = weights.size(1);
    return chosen;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    without_tangent(grads[0]);
    const Tensor ids = ctx->get_saved_variables()[0], g = numbers(grads[0]).contiguous();
    const int64_t count = ctx->saved_data["count"].toInt();
    const Call call(g);
    Tensor out = at::empty({ids.size(0), count}, g.options().requires_grad(false));
    check(purin_train_route_vjp(call.stream, code_of(g, "gradient"), ids.size(0), count,
                                ids.size(1), ints(ids), g.data_ptr(), out.data_ptr()));
    return once({out, Tensor(), Tensor(), Tensor()});
  }
};

using Routed = std::tuple<int64_t, int64_t, int64_t, Tensor, Tensor, Tensor, Tensor, Tensor>;

Routed route(const Tensor& weights, int64_t slots, const std::optional<Tensor>& workspace) {
  code_of(weights, "weights");
  if (weights.dim() != 2) refuse("weights must have two dimensions; got shape ", weights.sizes());
  const int64_t count = weights.size(1);
  if (slots < 1) refuse("slots must be a positive integer; got ", slots);
  if (count < 1 || slots > count) refuse("slots must not exceed the ", count, " experts; got ", slots);
  without_tangent(weights);
  Index index;
  Tensor chosen = wants_grad(weights) ? RouteFn::apply(weights, slots, workspace, &index)
                                      : run_route(weights, slots, workspace, &index);
  return {weights.size(0), count, slots, index.ids, chosen, index.offsets, index.place, index.source};
}

Routed route_experts(const Tensor& experts, int64_t count, const std::optional<Tensor>& weights,
                     const std::optional<Tensor>& workspace) {
  if (!experts.is_cuda()) refuse("experts must be a tensor on the GPU");
  if ((experts.scalar_type() != at::kInt && experts.scalar_type() != at::kLong) ||
      experts.dim() != 2)
    refuse("experts must be an int32 or int64 tensor (tokens, slots); got ", experts.scalar_type(),
           " ", experts.sizes());
  const int64_t tokens = experts.size(0), slots = experts.size(1);
  if (slots < 1) refuse("experts must have a slot");
  if (count < 1) refuse("count must be a positive integer; got ", count);
  if (weights) {
    code_of(*weights, "weights");
    same_device(experts, *weights, "weights");
    if (weights->sizes() != experts.sizes())
      refuse("weights must have shape ", experts.sizes(), "; got ", weights->sizes());
  }
  const Tensor given = experts.contiguous();
  const Call call(given);
  const Workspace ws(workspace, purin_train_route_workspace_bytes(tokens, count, slots), given);
  const Index x = new_index(tokens, count, slots, given);
  check(purin_train_sort(call.stream, given.scalar_type() == at::kLong, tokens, count, slots,
                         given.data_ptr(), ws.at, ws.size, ints(x.ids), ints(x.offsets),
                         ints(x.place), ints(x.source)));
  return {tokens, count, slots, x.ids, weights ? *weights : Tensor(), x.offsets, x.place, x.source};
}

// -- rows ---------------------------------------------------------------------------------

// A routing's order of rows, as the kernels read it.  The tensors are a caller's by now, who may
// have replaced them.
struct Order {
  Tensor place, offsets;
  Order(const Tensor& p, const Tensor& o) {
    check(p, 2, "routing.place", "(tokens, slots)");
    check(o, 1, "routing.offsets", "(experts + 1)");
    if (p.size(1) < 1) refuse("routing.place must have a slot");
    if (o.size(0) < 2) refuse("routing.offsets must have an expert");
    same_device(p, o, "routing.offsets");
    place = p.contiguous();
    offsets = o.contiguous();
  }
  static void check(const Tensor& t, int64_t dim, const char* name, const char* shape) {
    if (!t.is_cuda() || t.layout() != at::kStrided || t.scalar_type() != at::kInt || t.dim() != dim)
      refuse(name, " must be an int32 tensor ", shape, " on the GPU; got ", t.scalar_type(), " ",
             t.sizes(), " on ", t.device());
  }
};

Tensor run_combine(const Tensor& given, const Tensor& place, const Tensor* weights) {
  const Tensor rows = matrix(given);
  const Call call(rows);
  Tensor out = at::empty({place.size(0), rows.size(1)}, rows.options().requires_grad(false));
  check(purin_train_combine(call.stream, code_of(rows, "rows"),
                            weights ? code_of(*weights, "weights") : 0, place.size(0),
                            place.size(1), rows.size(1), rows.data_ptr(), rows.stride(0),
                            ints(place), weights ? weights->data_ptr() : nullptr, out.data_ptr()));
  return out;
}

Tensor run_dispatch(const Tensor& given, const Tensor& place, const Tensor& offsets) {
  const Tensor x = matrix(given);
  const Call call(x);
  Tensor rows = at::empty({place.numel(), x.size(1)}, x.options().requires_grad(false));
  check(purin_train_dispatch(call.stream, code_of(x, "x"), place.size(0), offsets.numel() - 1,
                             place.size(1), x.size(1), x.data_ptr(), x.stride(0), ints(offsets),
                             ints(place), rows.data_ptr()));
  return rows;
}

struct DispatchFn : torch::autograd::Function<DispatchFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& place,
                        const Tensor& offsets) {
    ctx->save_for_backward({place});
    return run_dispatch(x, place, offsets);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    without_tangent(grads[0]);
    return once({run_combine(grads[0], ctx->get_saved_variables()[0], nullptr), Tensor(), Tensor()});
  }
};

Tensor dispatch(const Tensor& x, const Tensor& place_given, const Tensor& offsets_given) {
  code_of(x, "x");
  const Order order(place_given, offsets_given);
  const Tensor &place = order.place, &offsets = order.offsets;
  same_device(place, x, "x");
  if (x.dim() != 2 || x.size(0) != place.size(0))
    refuse("x must have shape (", place.size(0), ", width); got ", x.sizes());
  without_tangent(x);
  return wants_grad(x) ? DispatchFn::apply(x, place, offsets) : run_dispatch(x, place, offsets);
}

struct CombineFn : torch::autograd::Function<CombineFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& weights,
                        const Tensor& place, const Tensor& offsets) {
    ctx->save_for_backward({rows, weights, place, offsets});
    const Tensor w = numbers(weights).contiguous();
    return run_combine(rows, place, &w);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    for (const Tensor& t : {saved[0], saved[1], grads[0]}) without_tangent(t);
    const Tensor rows = matrix(saved[0]), w = numbers(saved[1]).contiguous(), g = matrix(grads[0]);
    const Tensor &place = saved[2], &offsets = saved[3];
    const Call call(g);
    Tensor g_rows, g_weights;
    if (ctx->needs_input_grad(0))
      g_rows = at::empty(rows.sizes(), rows.options().requires_grad(false));
    if (ctx->needs_input_grad(1))
      g_weights = at::empty(w.sizes(), w.options().requires_grad(false));
    check(purin_train_combine_vjp(
        call.stream, code_of(g, "gradient"), code_of(w, "weights"), place.size(0),
        offsets.numel() - 1, place.size(1), g.size(1), g.data_ptr(), g.stride(0), rows.data_ptr(),
        rows.stride(0), ints(offsets), ints(place), w.data_ptr(),
        g_rows.defined() ? g_rows.data_ptr() : nullptr,
        g_weights.defined() ? g_weights.data_ptr() : nullptr));
    return once({g_rows, g_weights, Tensor(), Tensor()});
  }
};

Tensor combine(const Tensor& rows, const Tensor& weights, const Tensor& place_given,
               const Tensor& offsets_given) {
  code_of(rows, "rows");
  const Order order(place_given, offsets_given);
  const Tensor &place = order.place, &offsets = order.offsets;
  same_device(place, rows, "rows");
  if (rows.dim() != 2 || rows.size(0) != place.numel())
    refuse("rows must have shape (", place.numel(), ", width); got ", rows.sizes());
  code_of(weights, "weights");
  same_device(rows, weights, "weights");
  if (weights.sizes() != place.sizes())
    refuse("weights must have shape ", place.sizes(), "; got ", weights.sizes());
  without_tangent(rows);
  without_tangent(weights);
  if (wants_grad(rows) || wants_grad(weights)) return CombineFn::apply(rows, weights, place, offsets);
  const Tensor w = numbers(weights).contiguous();
  return run_combine(rows, place, &w);
}

// -- the experts' products ------------------------------------------------------------------

// A weight with a unit stride along inner or outer and no overlap inside a matrix; a broadcast
// over the experts stays one.
Tensor weight_strides(const Tensor& given) {
  const Tensor w = numbers(given);
  const int64_t inner = w.size(1), outer = w.size(2), si = w.stride(1), so = w.stride(2);
  if ((so == 1 || outer <= 1) && (si >= outer || inner <= 1)) return w;
  if ((si == 1 || inner <= 1) && (so >= inner || outer <= 1)) return w;
  return w.contiguous();
}

Tensor run_product(const Tensor& rows, const Tensor& w, const Tensor& offsets) {
  const Tensor a = matrix(rows);
  const int32_t code = code_of(a, "rows");
  const int64_t p = a.size(0), inner = a.size(1), outer = w.size(2), experts = w.size(0);
  const Call call(a);
  const Workspace ws(
      std::nullopt, purin_train_expert_product_workspace_bytes(code, p, inner, outer, experts), a);
  Tensor out = at::empty({p, outer}, a.options().requires_grad(false));
  check(purin_train_expert_product(call.stream, code, p, inner, outer, experts, a.data_ptr(),
                                   a.stride(0), w.data_ptr(), w.stride(0), w.stride(1), w.stride(2),
                                   ints(offsets), ws.at, ws.size, out.data_ptr(), outer));
  return out;
}

Tensor run_weights_vjp(const Tensor& a, const Tensor& g, const Tensor& offsets, int64_t experts) {
  const int32_t code = code_of(a, "rows");
  const int64_t p = a.size(0), inner = a.size(1), outer = g.size(1);
  const Call call(a);
  const Workspace ws(
      std::nullopt, purin_train_expert_weights_vjp_workspace_bytes(code, p, inner, outer, experts),
      a);
  Tensor out = at::empty({experts, inner, outer}, a.options().requires_grad(false));
  check(purin_train_expert_weights_vjp(call.stream, code, p, inner, outer, experts, a.data_ptr(),
                                       a.stride(0), g.data_ptr(), g.stride(0), ints(offsets), ws.at,
                                       ws.size, out.data_ptr()));
  return out;
}

// -- microscaled numbers --------------------------------------------------------------------

int64_t micro_blocks(int64_t length) { return (length + 31) / 32; }
int64_t micro_row_bytes(int32_t kind, int64_t length) {
  return micro_blocks(length) * (kind == PURIN_TRAIN_FP4 ? 16 : 32);
}
int64_t micro_scales(int64_t length) { return (micro_blocks(length) + 3) / 4 * 4; }

// Packed rows of a length: codes and scales, as they are in memory.
struct Packed {
  Tensor codes, scales;
  Packed() = default;
  Packed(std::vector<int64_t> lead, int32_t kind, int64_t length, const Tensor& like) {
    const auto o = like.options().dtype(at::kByte).requires_grad(false);
    lead.push_back(micro_row_bytes(kind, length));
    codes = at::empty(lead, o);
    lead.back() = micro_scales(length);
    scales = at::empty(lead, o);
  }
};

// A Microscaled's fields, which a caller may have made: ``lead`` is its shape without the axis
// that the blocks lie along.
Packed check_packed(const Tensor& codes, const Tensor& scales, int32_t kind,
                    const std::vector<int64_t>& shape, int64_t axis, const char* name) {
  const int64_t dims = (int64_t)shape.size();
  if (dims < 1 || axis < -dims || axis >= dims)
    refuse(name, " must be a Microscaled with an axis of its shape; got axis ", axis);
  std::vector<int64_t> lead = shape;
  const int64_t length = lead[axis < 0 ? axis + dims : axis];
  lead.erase(lead.begin() + (axis < 0 ? axis + dims : axis));
  lead.push_back(0);
  for (int i = 0; i < 2; ++i) {
    const Tensor& t = i ? scales : codes;
    const char* part = i ? "scales" : "codes";
    lead.back() = i ? micro_scales(length) : micro_row_bytes(kind, length);
    if (!t.is_cuda() || t.layout() != at::kStrided || t.scalar_type() != at::kByte || t.sizes() != at::IntArrayRef(lead))
      refuse(name, ".", part, " must be a uint8 tensor ", at::IntArrayRef(lead), " on the GPU; got ",
             t.scalar_type(), " ", t.sizes(), " on ", t.device());
  }
  same_device(codes, scales, name);
  Packed p;
  p.codes = codes.contiguous();
  p.scales = scales.contiguous();
  return p;
}

// Rows along the last dimension of ``t``, which has at most three.
Packed run_pack(const Tensor& given, int32_t kind) {
  Tensor t = numbers(given);
  const std::vector<int64_t> lead(t.sizes().begin(), t.sizes().end() - 1);
  while (t.dim() < 3) t = t.unsqueeze(0);
  if (t.stride(2) != 1 && t.size(2) > 1 && t.stride(1) != 1 && t.size(1) > 1) t = t.contiguous();
  int64_t groups = t.size(0), rows = t.size(1), sg = t.stride(0), sr = t.stride(1);
  const int64_t length = t.size(2), sl = length > 1 ? t.stride(2) : 1;
  if (rows == 1 && sl == 1) std::swap(groups, rows), std::swap(sg, sr);
  if (rows > 1 && sg == rows * sr) {
    rows *= groups;
    groups = 1;
  }
  const Call call(t);
  Packed p(lead, kind, length, t);
  check(purin_train_pack(call.stream, code_of(t, "tensor"), kind, groups, rows, length, t.data_ptr(),
                         sg, sr, sl, p.codes.data_ptr(), p.scales.data_ptr()));
  return p;
}

// The values of packed rows, (lead..., length) contiguous.
Tensor run_unpack(const Packed& p, int32_t kind, int64_t length, at::ScalarType dtype) {
  const Call call(p.codes);
  std::vector<int64_t> sizes(p.codes.sizes().begin(), p.codes.sizes().end());
  int64_t rows = 1;
  for (size_t i = 0; i + 1 < sizes.size(); ++i) rows *= sizes[i];
  sizes.back() = length;
  Tensor out = at::empty(sizes, p.codes.options().dtype(dtype));
  check(purin_train_unpack(call.stream, code_of(out, "dtype"), kind, rows, length,
                           p.codes.data_ptr(), p.scales.data_ptr(), out.data_ptr(), length));
  return out;
}

std::tuple<Tensor, Tensor> pack(const Tensor& t, int32_t kind, int64_t axis) {
  if (code_of(t, "tensor") == PURIN_TRAIN_F64)
    refuse("tensor must be float32, bfloat16 or float16 to be packed; got float64");
  if (t.layout() != at::kStrided) refuse("tensor must be dense");
  if (t.dim() < 1 || axis < -t.dim() || axis >= t.dim())
    refuse("axis must be one of the tensor's ", t.dim(), " dimensions; got ", axis);
  without_tangent(t);
  if (wants_grad(t))
    throw LibraryError(PURIN_CP_ERR_UNSUPPORTED, "pack has no gradient: give it a detached tensor");
  const Tensor moved = t.movedim(axis, -1);
  if (moved.dim() <= 3) {
    const Packed p = run_pack(moved, kind);
    return {p.codes, p.scales};
  }
  std::vector<int64_t> lead(moved.sizes().begin(), moved.sizes().end() - 1);
  const Packed p = run_pack(moved.flatten(0, -3), kind);
  lead.push_back(p.codes.size(-1));
  const Tensor codes = p.codes.view(lead);
  lead.back() = p.scales.size(-1);
  return {codes, p.scales.view(lead)};
}

Tensor unpack(const Tensor& codes, const Tensor& scales, int32_t kind,
              const std::vector<int64_t>& shape, int64_t axis, at::ScalarType dtype) {
  const Packed p = check_packed(codes, scales, kind, shape, axis, "packed");
  if (dtype != at::kFloat && dtype != at::kBFloat16 && dtype != at::kHalf)
    refuse("dtype must be float32, bfloat16 or float16; got ", dtype);
  const int64_t length = shape[axis < 0 ? axis + (int64_t)shape.size() : axis];
  return run_unpack(p, kind, length, dtype).movedim(-1, axis);
}

// -- the products' graph --------------------------------------------------------------------

struct ProductFn : torch::autograd::Function<ProductFn> {
  // ``saved``: what the weights' gradient reads of rows is kept in 8 bits
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& weight,
                        const Tensor& offsets, bool saved) {
    Packed kept;
    if (saved && weight.requires_grad()) kept = run_pack(rows.detach(), PURIN_TRAIN_INT8);
    ctx->saved_data["saved"] = saved;
    ctx->save_for_backward({saved ? Tensor() : rows, weight, offsets, kept.codes, kept.scales});
    return run_product(rows, weight_strides(weight), offsets);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    for (const Tensor& t : {saved[0], saved[1], grads[0]}) without_tangent(t);
    const Tensor w = weight_strides(saved[1]), g = matrix(grads[0]);
    const Tensor& offsets = saved[2];
    Tensor g_rows, g_weight;
    if (ctx->needs_input_grad(0)) g_rows = run_product(g, w.transpose(1, 2), offsets);
    if (ctx->needs_input_grad(1)) {
      Packed kept;
      kept.codes = saved[3];
      kept.scales = saved[4];
      const Tensor a = ctx->saved_data["saved"].toBool()
                           ? run_unpack(kept, PURIN_TRAIN_INT8, w.size(1), w.scalar_type())
                           : matrix(saved[0]);
      if (w.stride(2) == 1 || w.size(2) <= 1)
        g_weight = run_weights_vjp(a, g, offsets, w.size(0));
      else  // the weight's own order: (a^T g)^T = g^T a
        g_weight = run_weights_vjp(g, a, offsets, w.size(0)).transpose(1, 2);
    }
    return once({g_rows, g_weight, Tensor(), Tensor()});
  }
};

void check_offsets(const Tensor& rows, const Tensor& offsets, int64_t experts) {
  if (offsets.scalar_type() != at::kInt || offsets.dim() != 1 || offsets.size(0) != experts + 1)
    refuse("offsets must be a Routing or an int32 tensor of ", experts + 1, " entries");
  same_device(rows, offsets, "offsets");
}

Tensor expert_product(const Tensor& rows, const Tensor& weight, const Tensor& offsets, bool saved) {
  code_of(rows, "rows");
  code_of(weight, "weight");
  if (rows.scalar_type() != weight.scalar_type())
    refuse("rows and weight must have one type; got ", rows.scalar_type(), " and ",
           weight.scalar_type());
  if (rows.dim() != 2 || weight.dim() != 3 || rows.size(1) != weight.size(1))
    refuse("rows must have shape (rows, inner) and weight (experts, inner, outer); got ",
           rows.sizes(), " and ", weight.sizes());
  same_device(rows, weight, "weight");
  check_offsets(rows, offsets, weight.size(0));
  if (saved && rows.scalar_type() == at::kDouble) refuse("rows of float64 are not kept in 8 bits");
  without_tangent(rows);
  without_tangent(weight);
  const Tensor at = offsets.contiguous();
  return wants_grad(rows) || wants_grad(weight) ? ProductFn::apply(rows, weight, at, saved)
                                                : run_product(rows, weight_strides(weight), at);
}

// Weights of (experts, inner, outer) in FP4, blocks along inner.
struct PackedWeight {
  Packed p;
  int64_t experts, inner, outer;
  PackedWeight(const Tensor& codes, const Tensor& scales, int32_t kind,
               const std::vector<int64_t>& shape, int64_t axis, const char* name) {
    if (kind != PURIN_TRAIN_FP4 || shape.size() != 3 || (axis != 1 && axis != -2))
      refuse(name, " must be packed as \"fp4\", of shape (experts, inner, outer) along axis 1; got ",
             at::IntArrayRef(shape), " along axis ", axis);
    p = check_packed(codes, scales, kind, shape, axis, name);
    experts = shape[0];
    inner = shape[1];
    outer = shape[2];
    if (experts < 1) refuse(name, " must have an expert");
  }
};

Tensor run_product_packed(const Tensor& rows, const Packed* packed_rows, int32_t code,
                          const Packed& w, const Tensor& offsets, int64_t inner, int64_t outer,
                          const at::TensorOptions& options) {
  const Call call(rows);
  const int64_t p = rows.size(0), experts = w.codes.size(0);
  // the library knows packed rows by their scales, which empty ones lack
  if (packed_rows && (!p || !inner || !outer)) return at::zeros({p, outer}, options);
  const Workspace ws(std::nullopt,
                     purin_train_expert_product_packed_workspace_bytes(
                         code, packed_rows != nullptr, p, inner, outer, experts),
                     rows);
  Tensor out = at::empty({p, outer}, options);
  check(purin_train_expert_product_packed(
      call.stream, code, p, inner, outer, experts, rows.data_ptr(), packed_rows ? 0 : rows.stride(0),
      packed_rows ? packed_rows->scales.data_ptr() : nullptr, w.codes.data_ptr(),
      w.scales.data_ptr(), ints(offsets), ws.at, ws.size, out.data_ptr(), outer));
  return out;
}

// Rows of 32 bits: beside the weights as numbers of 32 bits, for the length of the call.
Tensor run_rows_packed(const Tensor& rows, const Packed& w, const Tensor& offsets, int64_t outer) {
  const Tensor a = matrix(rows);
  if (a.scalar_type() == at::kFloat)
    return run_product(a, run_unpack(w, PURIN_TRAIN_FP4, a.size(1), at::kFloat).transpose(1, 2), offsets);
  return run_product_packed(a, nullptr, code_of(a, "rows"), w, offsets, a.size(1), outer,
                            a.options().requires_grad(false));
}

struct PackedProductFn : torch::autograd::Function<PackedProductFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& codes,
                        const Tensor& scales, const Tensor& offsets, int64_t outer) {
    ctx->save_for_backward({codes, scales, offsets});
    ctx->saved_data["inner"] = rows.size(1);
    Packed w;
    w.codes = codes;
    w.scales = scales;
    return run_rows_packed(rows, w, offsets, outer);
  }
  // the weights unpacked, (experts, outer, inner): the contraction runs across their blocks
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    without_tangent(grads[0]);
    Packed w;
    w.codes = saved[0];
    w.scales = saved[1];
    const Tensor g = matrix(grads[0]);
    const Tensor full = run_unpack(w, PURIN_TRAIN_FP4, ctx->saved_data["inner"].toInt(), g.scalar_type());
    return once({run_product(g, full, saved[2]), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor expert_product_packed(const Tensor& rows, const Tensor& codes, const Tensor& scales,
                             int32_t kind, const std::vector<int64_t>& shape, int64_t axis,
                             const Tensor& offsets) {
  const PackedWeight w(codes, scales, kind, shape, axis, "weight");
  const int32_t code = code_of(rows, "rows");
  if (rows.dim() != 2 || rows.size(1) != w.inner)
    refuse("rows must have shape (rows, ", w.inner, "); got ", rows.sizes());
  if (code == PURIN_TRAIN_F64) refuse("rows must be float32, bfloat16 or float16 beside packed weights");
  same_device(rows, w.p.codes, "weight");
  check_offsets(rows, offsets, w.experts);
  without_tangent(rows);
  const Tensor at = offsets.contiguous();
  return wants_grad(rows) ? PackedProductFn::apply(rows, w.p.codes, w.p.scales, at, w.outer)
                          : run_rows_packed(rows, w.p, at, w.outer);
}

Tensor expert_product_both(const Tensor& rows_codes, const Tensor& rows_scales, int32_t rows_kind,
                           const std::vector<int64_t>& rows_shape, int64_t rows_axis,
                           at::ScalarType dtype, const Tensor& codes, const Tensor& scales,
                           int32_t kind, const std::vector<int64_t>& shape, int64_t axis,
                           const Tensor& offsets) {
  const PackedWeight w(codes, scales, kind, shape, axis, "weight");
  if (rows_kind != PURIN_TRAIN_FP4 || rows_shape.size() != 2 || (rows_axis != 1 && rows_axis != -1) ||
      rows_shape[1] != w.inner)
    refuse("packed rows must be \"fp4\", of shape (rows, ", w.inner, ") along axis 1; got ",
           at::IntArrayRef(rows_shape), " along axis ", rows_axis);
  const Packed a = check_packed(rows_codes, rows_scales, rows_kind, rows_shape, rows_axis, "rows");
  same_device(a.codes, w.p.codes, "weight");
  check_offsets(a.codes, offsets, w.experts);
  const int32_t code = dtype == at::kFloat      ? PURIN_TRAIN_F32
                       : dtype == at::kBFloat16 ? PURIN_TRAIN_BF16
                       : dtype == at::kHalf     ? PURIN_TRAIN_F16
                                                : -1;
  if (code < 0) refuse("packed rows must be of float32, bfloat16 or float16; got ", dtype);
  return run_product_packed(a.codes, &a, code, w.p, offsets.contiguous(), w.inner, w.outer,
                            a.codes.options().dtype(dtype));
}

// -- the activation -------------------------------------------------------------------------

Tensor run_activate(const Tensor& given, int32_t act, bool gated, Packed* kept) {
  const Tensor u = matrix(given);
  const int64_t rows = u.size(0), hidden = gated ? u.size(1) / 2 : u.size(1);
  const Call call(u);
  Tensor out = at::empty({rows, hidden}, u.options().requires_grad(false));
  if (kept) *kept = Packed({rows, gated ? 2 : 1}, PURIN_TRAIN_INT8, hidden, u);
  check(purin_train_activate(call.stream, code_of(u, "rows"), act, gated, rows, hidden, u.data_ptr(),
                             u.stride(0), out.data_ptr(), kept ? kept->codes.data_ptr() : nullptr,
                             kept ? kept->scales.data_ptr() : nullptr));
  return out;
}

struct ActivateFn : torch::autograd::Function<ActivateFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& u, int64_t act, bool gated, bool saved) {
    Packed kept;
    Tensor out = run_activate(u, (int32_t)act, gated, saved ? &kept : nullptr);
    ctx->save_for_backward({saved ? Tensor() : u, kept.codes, kept.scales});
    ctx->saved_data["act"] = act;
    ctx->saved_data["gated"] = gated;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    for (const Tensor& t : {saved[0], grads[0]}) without_tangent(t);
    const bool gated = ctx->saved_data["gated"].toBool(), packed = saved[1].defined();
    const Tensor g = matrix(grads[0]);
    const Tensor u = packed ? Tensor() : matrix(saved[0]);
    const Call call(g);
    const int64_t rows = g.size(0), hidden = g.size(1);
    Tensor out = at::empty({rows, gated ? 2 * hidden : hidden}, g.options().requires_grad(false));
    check(purin_train_activate_vjp(
        call.stream, code_of(g, "gradient"), (int32_t)ctx->saved_data["act"].toInt(), gated, rows,
        hidden, packed ? nullptr : u.data_ptr(), packed ? 0 : u.stride(0),
        packed ? saved[1].data_ptr() : nullptr, packed ? saved[2].data_ptr() : nullptr, g.data_ptr(),
        g.stride(0), out.data_ptr()));
    return once({out, Tensor(), Tensor(), Tensor()});
  }
};

Tensor activate(const Tensor& rows, int64_t act, bool gated, bool saved) {
  const int32_t code = code_of(rows, "rows");
  if (rows.dim() != 2 || (gated && rows.size(1) % 2))
    refuse("rows must have two dimensions, with a gate an even number of columns; got ", rows.sizes());
  if (saved && code == PURIN_TRAIN_F64) refuse("rows of float64 are not kept in 8 bits");
  without_tangent(rows);
  return wants_grad(rows) ? ActivateFn::apply(rows, act, gated, saved)
                          : run_activate(rows, (int32_t)act, gated, nullptr);
}

// -- a whole layer --------------------------------------------------------------------------

// A weight as the library reads it; ``held`` keeps what it points to.
using MicroFields = std::tuple<Tensor, Tensor, int32_t, std::vector<int64_t>, int64_t>;
struct LayerWeight {
  purin_train_matrices m{};
  Tensor held;
  Packed packed;
  int64_t experts, inner, outer;
  LayerWeight(const std::optional<Tensor>& dense, const std::optional<MicroFields>& fields,
              const Tensor& x, const char* name) {
    if (dense) {
      code_of(*dense, name);
      if (dense->dim() != 3 || dense->size(0) < 1 || dense->scalar_type() != x.scalar_type())
        refuse(name, " must have shape (experts, inner, outer) and type ", x.scalar_type(), "; got ",
               dense->sizes(), " and ", dense->scalar_type());
      same_device(x, *dense, name);
      without_tangent(*dense);
      held = weight_strides(*dense);
      experts = held.size(0), inner = held.size(1), outer = held.size(2);
      m = {held.data_ptr(), nullptr, held.stride(0), held.stride(1), held.stride(2)};
    } else {
      const auto& [codes, scales, kind, shape, axis] = *fields;
      const PackedWeight w(codes, scales, kind, shape, axis, name);
      same_device(x, w.p.codes, name);
      packed = w.p;
      experts = w.experts, inner = w.inner, outer = w.outer;
      m = {packed.codes.data_ptr(), packed.scales.data_ptr(), 0, 0, 0};
    }
  }
};

// None where the kernels do not take the call (types, sizes, a gradient wanted), after its checks.
std::optional<Tensor> expert_layer(const Tensor& x, const Tensor& weights, int64_t slots,
                                   const std::optional<Tensor>& inner,
                                   const std::optional<MicroFields>& inner_packed,
                                   const std::optional<Tensor>& outer,
                                   const std::optional<MicroFields>& outer_packed, int32_t act,
                                   const std::optional<Tensor>& workspace) {
  const int32_t code = code_of(x, "x"), wcode = code_of(weights, "weights");
  if (x.dim() != 2 || weights.dim() != 2 || weights.size(0) != x.size(0))
    refuse("x must have shape (tokens, width) and weights (tokens, experts); got ", x.sizes(), " and ",
           weights.sizes());
  same_device(x, weights, "weights");
  if (code == PURIN_TRAIN_F64 && (inner_packed || outer_packed))
    refuse("x must be float32, bfloat16 or float16 beside packed weights");
  const LayerWeight a(inner, inner_packed, x, "inner"), b(outer, outer_packed, x, "outer");
  const int64_t tokens = x.size(0), experts = weights.size(1), hidden = b.inner;
  if (a.experts != experts || b.experts != experts)
    refuse("inner and outer must have the weights' ", experts, " experts; got ", a.experts, " and ",
           b.experts);
  if (a.inner != x.size(1)) refuse("inner must have ", x.size(1), " rows to an expert; got ", a.inner);
  if (a.outer != hidden && a.outer != 2 * hidden)
    refuse("inner must have ", hidden, " or, with a gate, ", 2 * hidden, " columns; got ", a.outer);
  if (slots < 1 || slots > experts)
    refuse("slots must be from 1 to the ", experts, " experts; got ", slots);
  without_tangent(x);
  without_tangent(weights);
  const bool graph = wants_grad(x) || wants_grad(weights) || (inner && wants_grad(*inner)) ||
                     (outer && wants_grad(*outer));
  if (graph || (code != PURIN_TRAIN_BF16 && code != PURIN_TRAIN_F16) ||
      tokens > PURIN_TRAIN_LAYER_TOKENS || tokens * slots > PURIN_TRAIN_LAYER_PAIRS ||
      std::max({a.inner, 2 * hidden, b.outer}) > PURIN_TRAIN_LAYER_WIDTH)
    return std::nullopt;
  const at::NoGradGuard no_grad;
  Tensor rows = matrix(x);
  if (rows.size(0) > 1 && rows.stride(0) >= (1 << 24)) rows = rows.contiguous();
  const Tensor w = matrix(weights);
  const Call call(rows);
  const Workspace ws(workspace,
                     purin_train_expert_layer_workspace_bytes(code, tokens, experts, slots,
                                                              a.inner, hidden, b.outer),
                     rows);
  Tensor out = at::empty({tokens, b.outer}, rows.options());
  check(purin_train_expert_layer(call.stream, code, wcode, tokens, experts, slots, a.inner, hidden,
                                 b.outer, act, a.outer != hidden, rows.data_ptr(), rows.stride(0),
                                 w.data_ptr(), w.stride(0), &a.m, &b.m, ws.at, ws.size,
                                 out.data_ptr()));
  return out;
}

// -- the global norm ------------------------------------------------------------------------

using Tensors = std::vector<std::optional<Tensor>>;

// A tensor's (stride, size) pairs from the smallest stride on, without sizes of one.
std::vector<std::pair<int64_t, int64_t>> steps_of(const Tensor& t) {
  std::vector<std::pair<int64_t, int64_t>> s;
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1) s.emplace_back(t.stride(d), t.size(d));
  std::sort(s.begin(), s.end());
  return s;
}
// Whether the elements fill one span of memory, each once, in whatever order.
bool dense(const Tensor& t) {
  if (t.is_contiguous()) return true;
  int64_t need = 1;
  for (const auto& [stride, size] : steps_of(t)) {
    if (stride != need) return false;
    need *= size;
  }
  return true;
}
// Whether some element may share its place with another.
bool overlaps_itself(const Tensor& t) {
  int64_t need = 1;
  for (const auto& [stride, size] : steps_of(t)) {
    if (stride < need) return true;
    need += stride * (size - 1);
  }
  return false;
}

// The bytes of a tensor's elements: ``from`` + the sum of steps (bytes) times indexes, ``size``
// bytes from each such address on, all below ``to``.
struct Bytes {
  int64_t from, to, size;
  std::vector<std::pair<int64_t, int64_t>> steps;
  explicit Bytes(const Tensor& t) : from((int64_t)t.data_ptr()), size((int64_t)t.element_size()) {
    to = from + size;
    for (const auto& [stride, n] : steps_of(t)) {
      if (!stride) continue;
      steps.emplace_back(stride * size, n);
      to += stride * size * (n - 1);
    }
  }
};

// Whether two tensors may have a byte in common: whether some sum of a's steps less b's, each
// ``c`` times a whole number between ``low`` and ``high``, is the distance of two such elements.
// From the largest step on, only numbers that the smaller steps can make up for are tried, and
// none where the distance is no multiple of what the steps left have in common.  Views of one
// tensor have steps in common, which count as one, and take a few trials; beyond ``left`` trials
// the answer is yes.
struct Shared {
  struct Term {
    int64_t c, low, high;
    int64_t least, most, common;  // of the sums of this term and those behind it
  };
  std::vector<Term> terms;
  int64_t left = 1 << 16;

  static int64_t down(int64_t a, int64_t b) { return a / b - (a % b < 0); }  // b > 0
  bool within(size_t i, int64_t low, int64_t high) {
    if (i == terms.size()) return low <= 0 && 0 <= high;
    const Term& t = terms[i];
    if (down(high, t.common) * t.common < low) return false;
    if (--left < 0) return true;
    const bool more = i + 1 < terms.size();
    const int64_t least = more ? terms[i + 1].least : 0, most = more ? terms[i + 1].most : 0;
    const int64_t first = std::max(t.low, -down(-(low - most), t.c));
    const int64_t last = std::min(t.high, down(high - least, t.c));
    for (int64_t z = first; z <= last; ++z)
      if (within(i + 1, low - t.c * z, high - t.c * z)) return true;
    return false;
  }
  bool operator()(const Bytes& a, const Bytes& b) {
    if (a.from >= b.to || b.from >= a.to) return false;
    for (const auto& [c, n] : a.steps) terms.push_back({c, 0, n - 1, 0, 0, 0});
    for (const auto& [c, n] : b.steps) {
      const auto same = [c = c](const Term& t) { return t.c == c; };
      const auto at = std::find_if(terms.begin(), terms.end(), same);
      if (at == terms.end()) terms.push_back({c, 1 - n, 0, 0, 0, 0});
      else at->low -= n - 1;
    }
    std::sort(terms.begin(), terms.end(), [](const Term& x, const Term& y) { return x.c > y.c; });
    int64_t least = 0, most = 0, common = 0;
    for (size_t i = terms.size(); i-- > 0;) {
      Term& t = terms[i];
      t.least = least += t.c * t.low;
      t.most = most += t.c * t.high;
      t.common = common = std::gcd(common, t.c);
    }
    const int64_t apart = a.from - b.from;
    return within(0, 1 - a.size - apart, b.size - 1 - apart);
  }
};

// One tensor of a list that is read, or written (``out``); ``copied``: by way of a copy, so that
// the library does not see its place.
struct Use {
  size_t tensor;
  bool out, copied;
  Bytes bytes;
};
// Refuses an output that shares memory with another tensor's output or gradient, where one of the
// two is copied (the library looks at the others).
void check_overlap(std::vector<Use> uses) {
  std::sort(uses.begin(), uses.end(),
            [](const Use& a, const Use& b) { return a.bytes.from < b.bytes.from; });
  for (size_t i = 0; i < uses.size(); ++i)
    for (size_t j = i + 1; j < uses.size() && uses[j].bytes.from < uses[i].bytes.to; ++j) {
      const Use &a = uses[i], &b = uses[j];
      if (a.tensor == b.tensor || !(a.out || b.out) || !(a.copied || b.copied)) continue;
      if (Shared()(a.bytes, b.bytes))
        throw LibraryError(PURIN_CP_ERR_ARG, "tensor " + std::to_string((a.out ? a : b).tensor) +
                                                 ": its output overlaps another tensor");
    }
}

int32_t gradient_code(const Tensor& t, const char* name, size_t i) {
  const std::string each = std::string(name) + "[" + std::to_string(i) + "]";
  if (t.layout() != at::kStrided) refuse(each, " must be a dense tensor");
  without_tangent(t);
  return code_of(t, each.c_str());
}

struct List {
  std::vector<purin_train_tensor> table;
  std::vector<std::pair<Tensor, Tensor>> held;  // the copies' owners among them
  bool wide = false;
  void add(const Tensor& in, const Tensor& out, int32_t code) {
    if (!held.empty() && held[0].first.device() != in.device())
      refuse("gradients must be on one device; got ", held[0].first.device(), " and ", in.device());
    if (out.device() != in.device()) refuse("out must be on ", in.device(), "; got ", out.device());
    wide = wide || code == PURIN_TRAIN_F64;
    table.push_back({in.data_ptr(), out.data_ptr(), in.numel(), code, 0});
    held.emplace_back(in, out);
  }
  Tensor run(double largest, const std::optional<Tensor>& workspace) {
    const auto dtype = wide ? at::kDouble : at::kFloat;
    Tensor norm = at::empty({}, held.empty() ? at::TensorOptions().device(at::kCUDA).dtype(dtype)
                                             : held[0].first.options().dtype(dtype));
    const int64_t n = (int64_t)table.size();
    const Call call(norm);
    const Workspace ws(workspace, purin_train_clip_workspace_bytes(n), norm);
    check(purin_train_clip(call.stream, n, table.data(), largest, ws.at, ws.size,
                           wide ? PURIN_TRAIN_F64 : PURIN_TRAIN_F32, norm.data_ptr()));
    return norm;
  }
};

// A gradient whose elements fill one span of memory, in whatever order.
Tensor span(const Tensor& t) {
  const Tensor g = numbers(t);
  return dense(g) ? g : g.contiguous();
}

Tensor run_norm(at::TensorList gradients, const std::optional<Tensor>& workspace) {
  List list;
  for (const Tensor& given : gradients) {
    const Tensor g = span(given);
    list.add(g, g, code_of(g, "gradient"));
  }
  return list.run(-1.0, workspace);
}

struct NormFn : torch::autograd::Function<NormFn> {
  static Tensor forward(AutogradContext* ctx, at::TensorList gradients,
                        const std::optional<Tensor>& workspace) {
    const Tensor norm = run_norm(gradients, workspace);
    variable_list saved = gradients.vec();
    saved.push_back(norm);
    ctx->save_for_backward(std::move(saved));
    return norm;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list saved = ctx->get_saved_variables();
    for (const Tensor& t : saved) without_tangent(t);
    without_tangent(grads[0]);
    const Tensor norm = saved.back(), g_norm = numbers(grads[0]);
    saved.pop_back();
    variable_list out(saved.size() + 1), held;  // the workspace has no gradient
    std::vector<purin_train_tensor> table;
    for (size_t i = 0; i < saved.size(); ++i) {
      if (!ctx->needs_input_grad(i)) continue;
      const Tensor g = span(saved[i]);
      out[i] = at::empty_strided(g.sizes(), g.strides(), g.options().requires_grad(false));
      table.push_back({g.data_ptr(), out[i].data_ptr(), g.numel(), code_of(g, "gradient"), 0});
      held.push_back(g);
    }
    const Call call(norm);
    check(purin_train_norm_vjp(call.stream, (int64_t)table.size(), table.data(),
                               code_of(norm, "norm"), norm.data_ptr(), g_norm.data_ptr()));
    return once(std::move(out));
  }
};

Tensor gradient_norm(const Tensors& gradients, const std::optional<Tensor>& workspace) {
  variable_list given;
  bool graph = false;
  for (size_t i = 0; i < gradients.size(); ++i) {
    if (!gradients[i]) continue;
    gradient_code(*gradients[i], "gradients", i);
    given.push_back(*gradients[i]);
    graph = graph || wants_grad(*gradients[i]);
  }
  if (graph) return NormFn::apply(at::TensorList(given), workspace);
  const at::NoGradGuard no_grad;
  return run_norm(given, workspace);
}

Tensor clip_gradients(const Tensors& gradients, double largest, const std::optional<Tensors>& out,
                      const std::optional<Tensor>& workspace) {
  if (!(largest >= 0.0)) refuse("largest must not be negative; got ", largest);
  const at::NoGradGuard no_grad;
  const Tensors& outs = out ? *out : gradients;
  if (outs.size() != gradients.size())
    refuse("out must hold ", gradients.size(), " tensors; got ", outs.size());
  List list;
  std::vector<std::pair<Tensor, Tensor>> back;
  std::vector<char> copied(gradients.size(), 0);
  for (size_t i = 0; i < gradients.size(); ++i) {
    if (gradients[i].has_value() != outs[i].has_value())
      refuse("out[", i, "] must be None exactly where the gradient is");
    if (!gradients[i]) continue;
    const Tensor &g = *gradients[i], &o = *outs[i];
    const int32_t code = gradient_code(g, "gradients", i);
    const bool in_place = o.is_same(g);
    if (!in_place) {
      gradient_code(o, "out", i);
      if (o.sizes() != g.sizes() || o.scalar_type() != g.scalar_type())
        refuse("out[", i, "] must have shape ", g.sizes(), " and type ", g.scalar_type(), "; got ",
               o.sizes(), " and ", o.scalar_type());
    }
    if (!o.is_contiguous() && overlaps_itself(o))
      refuse("out[", i, "] (or the gradient in place) has elements that share memory");
    // in place the marks of g and out are one, and a factor changes no sign
    if (in_place ? dense(g)
                 : g.is_contiguous() && o.is_contiguous() && !g.is_neg() && !o.is_neg()) {
      list.add(g, o, code);
    } else {  // any other order goes through a copy in order
      copied[i] = 1;
      const Tensor c = at::empty(o.sizes(), o.options().requires_grad(false));
      list.add(numbers(g).contiguous(), c, code);
      back.emplace_back(o, c);
    }
  }
  if (!back.empty()) {
    std::vector<Use> uses;
    for (size_t i = 0; i < gradients.size(); ++i) {
      if (!gradients[i] || !gradients[i]->numel()) continue;
      const bool by_copy = copied[i];
      uses.push_back({i, true, by_copy, Bytes(*outs[i])});
      if (!outs[i]->is_same(*gradients[i])) uses.push_back({i, false, by_copy, Bytes(*gradients[i])});
    }
    check_overlap(std::move(uses));
  }
  const Tensor norm = list.run(largest, workspace);
  for (auto& [o, c] : back) o.copy_(c);
  // autograd's check for tensors that changed after they were saved
  for (const auto& o : outs)
    if (o && !o->is_inference()) o->unsafeGetTensorImpl()->bump_version();
  return norm;
}

}  // namespace

PYBIND11_MODULE(_front, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const LibraryError& e) {
      const py::object type = py::module_::import("purin_amd._lib").attr("PurinError");
      PyErr_SetObject(type.ptr(), type(e.code, e.message).ptr());
    }
  });
  m.def("route", &route);
  m.def("route_experts", &route_experts);
  m.def("dispatch", &dispatch);
  m.def("combine", &combine);
  m.def("expert_product", &expert_product);
  m.def("pack", &pack);
  m.def("unpack", &unpack);
  m.def("expert_product_packed", &expert_product_packed);
  m.def("expert_product_both", &expert_product_both);
  m.def("activate", &activate);
  m.def("expert_layer", &expert_layer);
  m.def("gradient_norm", &gradient_norm);
  m.def("clip_gradients", &clip_gradients);
}
