"""Tokens to experts and back, around a projection layer that gives the routing weights.

A projection onto a routing polytope (a token's weights over the experts sum to one, an
expert's load stays within its capacity) gives weights ``(tokens, experts)`` that are mostly
exactly zero; a softmax gives weights that are all positive.  From either:

    routing = route(weights, slots)              # each token's experts, and the order of rows
    rows = dispatch(x, routing)                  # the tokens' rows, sorted by expert
    rows = expert_product(rows, w, routing)      # every expert's rows times its matrix
    out = combine(rows, routing)                 # back to the tokens, weights applied

Every call runs in the HIP library (``include/purin_train.h``) on the current stream of its
tensors' device, waits for nothing and keeps nothing; all are differentiable with torch
autograd, once.  The reference ends at the projection layer and has no counterpart.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
from torch.autograd.function import once_differentiable

from purin_amd import _lib

_CODES = {torch.float32: _lib.F32, torch.float64: _lib.F64, torch.bfloat16: _lib.BF16,
          torch.float16: _lib.F16}


def _float_code(t, name):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a tensor on the GPU")
    code = _CODES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be float32, float64, bfloat16 or float16; got {t.dtype}")
    return code


def _matrix(t, name):
    """``t`` (2-D) with adjacent elements in a row and rows that do not overlap, and its code."""
    code = _float_code(t, name)
    if t.ndim != 2:
        raise ValueError(f"{name} must have two dimensions; got shape {tuple(t.shape)}")
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t, code


def _same_device(a, b, name):
    if a.device != b.device:
        raise ValueError(f"{name} must be on {a.device}; got {b.device}")


def _call(name, device, *args):
    """One entry point on the device's current stream."""
    lib = _lib.load()
    stream = torch.cuda.current_stream(device).cuda_stream
    if device.index == torch.cuda.current_device():
        code = getattr(lib, name)(stream, *args)
    else:
        with torch.cuda.device(device):
            code = getattr(lib, name)(stream, *args)
    if code:
        _lib.check(code)


def _workspace(given, need, device):
    """(tensor or None, address, bytes) of a call's scratch: the caller's, or new memory that the
    allocator gives to nothing else before the stream's kernels are done with it."""
    if need < 0:
        _lib.check(_lib.ERR_ARG)
    if given is not None:
        if not isinstance(given, torch.Tensor) or not given.is_cuda:
            raise ValueError("workspace must be a device tensor")
        return given, given.data_ptr(), given.numel() * given.element_size()
    if need == 0:
        return None, None, 0
    t = torch.empty(need, dtype=torch.uint8, device=device)
    return t, t.data_ptr(), need


@dataclass(eq=False)
class Routing:
    """Where each token's rows go.

    ``experts`` (tokens, slots) int32, -1 where a slot is empty; ``weights`` (tokens, slots), 0
    there, connected to autograd where the weights given to ``route`` are; ``offsets``
    (count + 1) int32, each expert's first row and the rows' number last; ``place``
    (tokens, slots) int32, a slot's row, -1 where it is empty; ``source`` (tokens * slots) int32,
    the slot (token * slots + slot) of each row, -1 from ``offsets[count]`` on.
    """

    tokens: int
    count: int
    slots: int
    experts: torch.Tensor
    weights: torch.Tensor | None
    offsets: torch.Tensor
    place: torch.Tensor
    source: torch.Tensor

    @property
    def rows(self):
        """Rows of the sorted buffers: one for each slot."""
        return self.tokens * self.slots


def _index_tensors(tokens, count, slots, device):
    pairs = tokens * slots
    whole = torch.empty(3 * pairs + count + 1, dtype=torch.int32, device=device)
    ids, place, source, offsets = whole.split((pairs, pairs, pairs, count + 1))
    return ids.view(tokens, slots), place.view(tokens, slots), source, offsets


def _slots(slots):
    if isinstance(slots, bool) or not isinstance(slots, int) or slots < 1:
        raise ValueError(f"slots must be a positive integer; got {slots!r}")
    return slots


def route_workspace_bytes(tokens, count, slots):
    """Bytes of a caller's workspace for ``route`` or ``route_experts`` (256-byte aligned)."""
    n = int(_lib.load().purin_train_route_workspace_bytes(tokens, count, slots))
    if n < 0:
        _lib.check(_lib.ERR_ARG)
    return n


def _route(weights, slots, workspace):
    w, code = _matrix(weights, "weights")
    tokens, count = w.shape
    need = _lib.load().purin_train_route_workspace_bytes(tokens, count, slots)
    _, ws, ws_bytes = _workspace(workspace, need, w.device)
    ids, place, source, offsets = _index_tensors(tokens, count, slots, w.device)
    chosen = torch.empty((tokens, slots), dtype=w.dtype, device=w.device)
    _call("purin_train_route", w.device, code, tokens, count, slots, w.data_ptr(), w.stride(0),
          ws, ws_bytes, ids.data_ptr(), chosen.data_ptr(), offsets.data_ptr(), place.data_ptr(),
          source.data_ptr())
    return chosen, (ids, offsets, place, source)


class _RouteFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weights, slots, workspace, index):
        chosen, parts = _route(weights, slots, workspace)
        index.extend(parts)
        ctx.ids = parts[0]
        ctx.count = weights.shape[1]
        return chosen

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        ids, count = ctx.ids, ctx.count
        tokens, slots = ids.shape
        g = g.contiguous()
        g_weights = torch.empty((tokens, count), dtype=g.dtype, device=g.device)
        _call("purin_train_route_vjp", g.device, _CODES[g.dtype], tokens, count, slots,
              ids.data_ptr(), g.data_ptr(), g_weights.data_ptr())
        return g_weights, None, None, None


def route(weights, slots, *, workspace=None):
    """The experts of every token's ``slots`` largest positive weights, and the order of rows.

    ``weights`` (tokens, experts), any floating type, at most 1024 experts.  Zero and negative
    weights choose nothing, so that a token may have fewer experts than slots, or none; ties go
    to the lowest expert; NaN counts as larger than any number.  ``workspace``: a device tensor
    of ``route_workspace_bytes(tokens, experts, slots)`` bytes (new memory otherwise).
    """
    _float_code(weights, "weights")
    if weights.ndim != 2:
        raise ValueError(f"weights must have two dimensions; got shape {tuple(weights.shape)}")
    tokens, count = weights.shape
    slots = _slots(slots)
    if count < 1 or slots > count:
        raise ValueError(f"slots must not exceed the {count} experts; got {slots}")
    if weights.requires_grad and torch.is_grad_enabled():
        index = []
        chosen = _RouteFn.apply(weights, slots, workspace, index)
    else:
        chosen, index = _route(weights, slots, workspace)
    ids, offsets, place, source = index
    return Routing(tokens, count, slots, ids, chosen, offsets, place, source)


def route_experts(experts, count, *, weights=None, workspace=None):
    """The order of rows for experts that are given: ``experts`` (tokens, slots), int32 or int64,
    of ``count`` experts.  A value outside [0, count) leaves its slot empty; a token may name an
    expert more than once.  ``weights`` (tokens, slots) are kept for ``combine``."""
    if not isinstance(experts, torch.Tensor) or not experts.is_cuda:
        raise ValueError("experts must be a tensor on the GPU")
    if experts.dtype not in (torch.int32, torch.int64) or experts.ndim != 2:
        raise ValueError("experts must be an int32 or int64 tensor (tokens, slots); got "
                         f"{experts.dtype} {tuple(experts.shape)}")
    tokens, slots = experts.shape
    _slots(slots)
    if isinstance(count, bool) or not isinstance(count, int) or count < 1:
        raise ValueError(f"count must be a positive integer; got {count!r}")
    if weights is not None:
        _float_code(weights, "weights")
        _same_device(experts, weights, "weights")
        if tuple(weights.shape) != (tokens, slots):
            raise ValueError(f"weights must have shape {(tokens, slots)}; got "
                             f"{tuple(weights.shape)}")
    given = experts.contiguous()
    device = given.device
    need = _lib.load().purin_train_route_workspace_bytes(tokens, count, slots)
    _, ws, ws_bytes = _workspace(workspace, need, device)
    ids, place, source, offsets = _index_tensors(tokens, count, slots, device)
    _call("purin_train_sort", device, int(given.dtype == torch.int64), tokens, count, slots,
          given.data_ptr(), ws, ws_bytes, ids.data_ptr(), offsets.data_ptr(), place.data_ptr(),
          source.data_ptr())
    return Routing(tokens, count, slots, ids, weights, offsets, place, source)


def _routing(routing):
    if not isinstance(routing, Routing):
        raise ValueError("routing must be what route() or route_experts() returns")
    return routing


def _combine(rows, code, routing, weights):
    out = torch.empty((routing.tokens, rows.shape[1]), dtype=rows.dtype, device=rows.device)
    wcode, wptr = (0, None) if weights is None else (_CODES[weights.dtype], weights.data_ptr())
    _call("purin_train_combine", rows.device, code, wcode, routing.tokens, routing.slots,
          rows.shape[1], rows.data_ptr(), rows.stride(0), routing.place.data_ptr(), wptr,
          out.data_ptr())
    return out


def _dispatch(x, code, routing):
    rows = torch.empty((routing.rows, x.shape[1]), dtype=x.dtype, device=x.device)
    _call("purin_train_dispatch", x.device, code, routing.tokens, routing.count, routing.slots,
          x.shape[1], x.data_ptr(), x.stride(0), routing.offsets.data_ptr(),
          routing.place.data_ptr(), rows.data_ptr())
    return rows


class _DispatchFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, routing):
        ctx.routing = routing
        return _dispatch(*_matrix(x, "x"), routing)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        return _combine(*_matrix(g, "gradient"), ctx.routing, None), None


def dispatch(x, routing):
    """The tokens' rows sorted by expert: ``x`` (tokens, width) to (tokens * slots, width), a
    row for each slot that has an expert, zeros behind them."""
    _routing(routing)
    code = _float_code(x, "x")
    _same_device(routing.place, x, "x")
    if x.ndim != 2 or x.shape[0] != routing.tokens:
        raise ValueError(f"x must have shape ({routing.tokens}, width); got {tuple(x.shape)}")
    if x.requires_grad and torch.is_grad_enabled():
        return _DispatchFn.apply(x, routing)
    return _dispatch(_matrix(x, "x")[0], code, routing)


class _CombineFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, routing):
        r, code = _matrix(rows, "rows")
        w = weights.contiguous()
        ctx.routing = routing
        ctx.save_for_backward(r, w)
        return _combine(r, code, routing, w)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        rows, weights = ctx.saved_tensors
        routing = ctx.routing
        g, code = _matrix(g, "gradient")
        need_rows, need_weights = ctx.needs_input_grad[:2]
        g_rows = torch.empty(rows.shape, dtype=rows.dtype, device=g.device) if need_rows else None
        g_weights = torch.empty_like(weights) if need_weights else None
        _call("purin_train_combine_vjp", g.device, code, _CODES[weights.dtype], routing.tokens,
              routing.count, routing.slots, g.shape[1], g.data_ptr(), g.stride(0),
              rows.data_ptr(), rows.stride(0), routing.offsets.data_ptr(),
              routing.place.data_ptr(), weights.data_ptr(),
              g_rows.data_ptr() if need_rows else None,
              g_weights.data_ptr() if need_weights else None)
        return g_rows, g_weights, None


def combine(rows, routing, weights=None):
    """Each token's sum of its slots' rows times their weights: ``rows`` (tokens * slots, width)
    to (tokens, width); zeros for a token without experts.  ``weights`` (tokens, slots), of any
    floating type: ``routing.weights`` where they are not given."""
    _routing(routing)
    code = _float_code(rows, "rows")
    _same_device(routing.place, rows, "rows")
    if rows.ndim != 2 or rows.shape[0] != routing.rows:
        raise ValueError(f"rows must have shape ({routing.rows}, width); got {tuple(rows.shape)}")
    weights = routing.weights if weights is None else weights
    if weights is None:
        raise ValueError("the routing holds no weights: give them")
    _float_code(weights, "weights")
    _same_device(rows, weights, "weights")
    if tuple(weights.shape) != (routing.tokens, routing.slots):
        raise ValueError(f"weights must have shape {(routing.tokens, routing.slots)}; got "
                         f"{tuple(weights.shape)}")
    if (rows.requires_grad or weights.requires_grad) and torch.is_grad_enabled():
        return _CombineFn.apply(rows, weights, routing)
    return _combine(_matrix(rows, "rows")[0], code, routing, weights.contiguous())


def _weight_strides(w):
    """``w`` (experts, inner, outer) with a unit stride along inner or outer and no negative
    or overlapping order inside a matrix; a broadcast over the experts stays one."""
    _, inner, outer = w.shape
    _, si, so = w.stride()
    if (so == 1 or outer <= 1) and (si >= outer or inner <= 1):
        return w
    if (si == 1 or inner <= 1) and (so >= inner or outer <= 1):
        return w
    return w.contiguous()


def _product(a, weight, offsets):
    """a(p) weight[e(p)], any of the two orders of weight."""
    code = _CODES[a.dtype]
    p, inner = a.shape
    experts, _, outer = weight.shape
    need = _lib.load().purin_train_expert_product_workspace_bytes(code, p, inner, outer, experts)
    _, ws, ws_bytes = _workspace(None, need, a.device)
    out = torch.empty((p, outer), dtype=a.dtype, device=a.device)
    _call("purin_train_expert_product", a.device, code, p, inner, outer, experts, a.data_ptr(),
          a.stride(0), weight.data_ptr(), *weight.stride(), offsets.data_ptr(), ws, ws_bytes,
          out.data_ptr(), outer)
    return out


def _product_weights_vjp(a, g, offsets, experts):
    code = _CODES[a.dtype]
    p, inner = a.shape
    outer = g.shape[1]
    need = _lib.load().purin_train_expert_weights_vjp_workspace_bytes(code, p, inner, outer,
                                                                      experts)
    _, ws, ws_bytes = _workspace(None, need, a.device)
    g_weight = torch.empty((experts, inner, outer), dtype=a.dtype, device=a.device)
    _call("purin_train_expert_weights_vjp", a.device, code, p, inner, outer, experts,
          a.data_ptr(), a.stride(0), g.data_ptr(), g.stride(0), offsets.data_ptr(), ws, ws_bytes,
          g_weight.data_ptr())
    return g_weight


class _ProductFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weight, offsets):
        a, _ = _matrix(rows, "rows")
        w = _weight_strides(weight)
        ctx.save_for_backward(a, w, offsets)
        return _product(a, w, offsets)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        a, w, offsets = ctx.saved_tensors
        g, _ = _matrix(g, "gradient")
        g_rows = g_weight = None
        if ctx.needs_input_grad[0]:
            g_rows = _product(g, w.transpose(1, 2), offsets)
        if ctx.needs_input_grad[1]:
            experts, inner, outer = w.shape
            if w.stride(2) == 1 or outer <= 1:
                g_weight = _product_weights_vjp(a, g, offsets, experts)
            else:  # the weight's own order: (a^T g)^T = g^T a
                g_weight = _product_weights_vjp(g, a, offsets, experts).transpose(1, 2)
        return g_rows, g_weight, None


def expert_product(rows, weight, offsets):
    """Every expert's rows times its matrix: ``rows`` (rows, inner) sorted by expert, ``weight``
    (experts, inner, outer) in either order of its last two dimensions in memory, to
    (rows, outer), zeros behind the last expert's rows.

    ``offsets``: a ``Routing``, or (experts + 1) int32 on the GPU: each expert's first row and
    the rows' number last, ascending from 0 and at most ``rows``.
    """
    if isinstance(offsets, Routing):
        offsets = offsets.offsets
    _float_code(rows, "rows")
    _float_code(weight, "weight")
    if rows.dtype != weight.dtype:
        raise ValueError(f"rows and weight must have one type; got {rows.dtype} and "
                         f"{weight.dtype}")
    if rows.ndim != 2 or weight.ndim != 3 or rows.shape[1] != weight.shape[1]:
        raise ValueError("rows must have shape (rows, inner) and weight (experts, inner, outer); "
                         f"got {tuple(rows.shape)} and {tuple(weight.shape)}")
    if (not isinstance(offsets, torch.Tensor) or offsets.dtype != torch.int32
            or tuple(offsets.shape) != (weight.shape[0] + 1,)):
        raise ValueError(f"offsets must be a Routing or an int32 tensor of {weight.shape[0] + 1} "
                         "entries")
    _same_device(rows, weight, "weight")
    _same_device(rows, offsets, "offsets")
    offsets = offsets.contiguous()
    if (rows.requires_grad or weight.requires_grad) and torch.is_grad_enabled():
        return _ProductFn.apply(rows, weight, offsets)
    return _product(_matrix(rows, "rows")[0], _weight_strides(weight), offsets)
