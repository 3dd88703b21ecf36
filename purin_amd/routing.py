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
autograd, once and in reverse.  The reference ends at the projection layer and has no counterpart.

Arguments are checked in ``csrc/front.cpp``, which also holds the autograd nodes: a wrong one
raises ``ValueError``, what the library cannot do ``PurinError`` (forward-mode tangents and
tracing among it, where a result would miss its derivative or its kernels).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from purin_amd import _lib

_lib.load()
from purin_amd import _front  # noqa: E402  (linked to the library, which is built with it)
from purin_amd.microscaled import Microscaled, fields, kept  # noqa: E402


@dataclass(eq=False)
class Routing:
    """Where each token's rows go.

    ``experts`` (tokens, slots) int32, -1 where a slot is empty; ``weights`` (tokens, slots), 0
    there, connected to autograd where the weights given to ``route`` are; ``offsets``
    (count + 1) int32, each expert's first row and the rows' number last; ``place``
    (tokens, slots) int32, a slot's row, -1 where it is empty; ``source`` (tokens * slots) int32,
    the slot (token * slots + slot) of each row, -1 from ``offsets[count]`` on.  ``place`` and
    ``offsets`` are what the calls below read: their types and shapes are checked there, their
    values are not (rows outside the buffer are passed over).
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


def route_workspace_bytes(tokens, count, slots):
    """Bytes of a caller's workspace for ``route`` or ``route_experts`` (256-byte aligned)."""
    n = int(_lib.load().purin_train_route_workspace_bytes(tokens, count, slots))
    if n < 0:
        _lib.check(_lib.ERR_ARG)
    return n


def route(weights, slots, *, workspace=None):
    """The experts of every token's ``slots`` largest positive weights, and the order of rows.

    ``weights`` (tokens, experts), any floating type, at most 1024 experts.  Zero and negative
    weights choose nothing, so that a token may have fewer experts than slots, or none; ties go
    to the lowest expert; NaN counts as larger than any number.  ``workspace``: a contiguous
    device tensor of ``route_workspace_bytes(tokens, experts, slots)`` bytes (new memory
    otherwise).
    """
    if slots.__class__ is not int:
        raise ValueError(f"slots must be a positive integer; got {slots!r}")
    try:
        return Routing(*_front.route(weights, slots, workspace))
    except TypeError:
        raise ValueError("weights and workspace must be tensors on the GPU; got "
                         f"{type(weights).__name__} and {type(workspace).__name__}") from None


def route_experts(experts, count, *, weights=None, workspace=None):
    """The order of rows for experts that are given: ``experts`` (tokens, slots), int32 or int64,
    of ``count`` experts.  A value outside [0, count) leaves its slot empty; a token may name an
    expert more than once.  ``weights`` (tokens, slots) are kept for ``combine``."""
    if count.__class__ is not int:
        raise ValueError(f"count must be a positive integer; got {count!r}")
    try:
        return Routing(*_front.route_experts(experts, count, weights, workspace))
    except TypeError:
        raise ValueError("experts, weights and workspace must be tensors on the GPU") from None


def _routing(routing):
    if not isinstance(routing, Routing):
        raise ValueError("routing must be what route() or route_experts() returns")
    return routing


def dispatch(x, routing):
    """The tokens' rows sorted by expert: ``x`` (tokens, width) to (tokens * slots, width), a
    row for each slot that has an expert, zeros behind them."""
    _routing(routing)
    try:
        return _front.dispatch(x, routing.place, routing.offsets)
    except TypeError:
        raise ValueError(f"x must be a tensor on the GPU; got {type(x).__name__}") from None


def combine(rows, routing, weights=None):
    """Each token's sum of its slots' rows times their weights: ``rows`` (tokens * slots, width)
    to (tokens, width); zeros for a token without experts.  ``weights`` (tokens, slots), of any
    floating type: ``routing.weights`` where they are not given.  Sums are held in 32 bits, in 64
    for float64 rows: beside narrower rows float64 weights are rounded to 32 bits, and their
    gradient holds sums of 32 bits."""
    _routing(routing)
    weights = routing.weights if weights is None else weights
    if weights is None:
        raise ValueError("the routing holds no weights: give them")
    try:
        return _front.combine(rows, weights, routing.place, routing.offsets)
    except TypeError:
        raise ValueError("rows and weights must be tensors on the GPU; got "
                         f"{type(rows).__name__} and {type(weights).__name__}") from None


def expert_product(rows, weight, offsets, *, saved=None):
    """Every expert's rows times its matrix: ``rows`` (rows, inner) sorted by expert, ``weight``
    (experts, inner, outer) in either order of its last two dimensions in memory, to
    (rows, outer), zeros behind the last expert's rows.

    ``offsets``: a ``Routing``, or (experts + 1) int32 on the GPU: each expert's first row and
    the rows' number last, ascending from 0 and at most ``rows``.

    ``weight`` may be packed (``pack(weight, "fp4", axis=1)``), ``rows`` then float32, bfloat16 or
    float16, or packed too (``pack(rows, "fp4")``), which gives results of the type that they were
    packed from.  Sums are held in 32 bits.  Packed operands have no gradient; the rows' beside
    packed weights, and products of float32 rows with them, unpack the weights to the rows' type
    for the length of the call.

    ``saved="int8"``: what a graph keeps of the rows for the weights' gradient is held in 8 bits
    (as ``pack(rows, "int8")``), and that gradient is at the rows which those stand for.  Not for
    float64.
    """
    if isinstance(offsets, Routing):
        offsets = offsets.offsets
    keep = kept(saved)
    try:
        if isinstance(weight, Microscaled):
            if keep:
                raise ValueError("packed weights have no gradient that rows are kept for")
            if isinstance(rows, Microscaled):
                return _front.expert_product_both(*fields(rows), rows.dtype, *fields(weight),
                                                  offsets)
            return _front.expert_product_packed(rows, *fields(weight), offsets)
        return _front.expert_product(rows, weight, offsets, keep)
    except TypeError:
        raise ValueError("rows, weight and offsets must be tensors on the GPU (packed rows go with "
                         f"packed weights); got {type(rows).__name__}, {type(weight).__name__} and "
                         f"{type(offsets).__name__}") from None
