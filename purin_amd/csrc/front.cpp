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

struct ProductFn : torch::autograd::Function<ProductFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& weight,
                        const Tensor& offsets) {
    ctx->save_for_backward({rows, weight, offsets});
    return run_product(rows, weight_strides(weight), offsets);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    for (const Tensor& t : {saved[0], saved[1], grads[0]}) without_tangent(t);
    const Tensor a = matrix(saved[0]), w = weight_strides(saved[1]), g = matrix(grads[0]);
    const Tensor& offsets = saved[2];
    Tensor g_rows, g_weight;
    if (ctx->needs_input_grad(0)) g_rows = run_product(g, w.transpose(1, 2), offsets);
    if (ctx->needs_input_grad(1)) {
      if (w.stride(2) == 1 || w.size(2) <= 1)
        g_weight = run_weights_vjp(a, g, offsets, w.size(0));
      else  // the weight's own order: (a^T g)^T = g^T a
        g_weight = run_weights_vjp(g, a, offsets, w.size(0)).transpose(1, 2);
    }
    return once({g_rows, g_weight, Tensor()});
  }
};

Tensor expert_product(const Tensor& rows, const Tensor& weight, const Tensor& offsets) {
  code_of(rows, "rows");
  code_of(weight, "weight");
  if (rows.scalar_type() != weight.scalar_type())
    refuse("rows and weight must have one type; got ", rows.scalar_type(), " and ",
           weight.scalar_type());
  if (rows.dim() != 2 || weight.dim() != 3 || rows.size(1) != weight.size(1))
    refuse("rows must have shape (rows, inner) and weight (experts, inner, outer); got ",
           rows.sizes(), " and ", weight.sizes());
  if (offsets.scalar_type() != at::kInt || offsets.dim() != 1 ||
      offsets.size(0) != weight.size(0) + 1)
    refuse("offsets must be a Routing or an int32 tensor of ", weight.size(0) + 1, " entries");
  same_device(rows, weight, "weight");
  same_device(rows, offsets, "offsets");
  without_tangent(rows);
  without_tangent(weight);
  const Tensor at = offsets.contiguous();
  return wants_grad(rows) || wants_grad(weight) ? ProductFn::apply(rows, weight, at)
                                                : run_product(rows, weight_strides(weight), at);
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
  m.def("gradient_norm", &gradient_norm);
  m.def("clip_gradients", &clip_gradients);
}
