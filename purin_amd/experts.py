"""What lies between the experts' products, and whole layers of experts.

    out = expert_layer(x, weights, slots, inner, outer)  # from routing weights to the layer's result

is ``route``, ``dispatch``, ``expert_product``, ``activate``, ``expert_product`` and ``combine`` in
turn, and for a few tokens of bfloat16 or float16 without a graph three or four kernels that read
every weight of the chosen experts once (a few times for experts with many tokens).  The HIP
library's conventions are those of ``routing``.  The reference has no counterpart.
"""

from __future__ import annotations

from purin_amd import _lib

_lib.load()
from purin_amd import _front  # noqa: E402  (linked to the library, which is built with it)
from purin_amd.microscaled import Microscaled, fields, kept  # noqa: E402
from purin_amd.routing import combine, dispatch, expert_product, route  # noqa: E402

ACTIVATIONS = {"relu": _lib.RELU, "silu": _lib.SILU, "gelu": _lib.GELU}


def _activation(kind):
    if not isinstance(kind, str) or kind not in ACTIVATIONS:
        raise ValueError(f'the activation must be "relu", "silu" or "gelu"; got {kind!r}')
    return ACTIVATIONS[kind]


def activate(rows, kind="silu", *, gated=True, saved=None):
    """``f(first half) * second half`` of the rows' columns, or ``f(rows)`` without a gate: ``rows``
    (rows, 2 * hidden) or (rows, hidden), any floating type, to (rows, hidden).

    ``kind``: "relu", "silu" (u / (1 + exp(-u))) or "gelu" (u times the share of a normal
    distribution below u).  ``saved="int8"``: what a graph keeps of the rows is held in 8 bits (each
    half as ``pack(half, "int8")``, made on the way), and the gradient is at the rows which those
    stand for: relu's slope is 0 where a positive number is nearer to zero than half a 64th of its
    block's power of two, about one in eighty of normal ones.  Not for float64.
    """
    code, keep = _activation(kind), kept(saved)
    try:
        return _front.activate(rows, code, bool(gated), keep)
    except TypeError:
        raise ValueError(f"rows must be a tensor on the GPU; got {type(rows).__name__}") from None


def expert_layer_workspace_bytes(dtype, tokens, experts, slots, width, hidden, outer):
    """Bytes of a caller's workspace (256-byte aligned) for an ``expert_layer`` of at most 64
    tokens; ``dtype``: ``_lib.BF16`` or ``_lib.F16``."""
    n = int(_lib.load().purin_train_expert_layer_workspace_bytes(dtype, tokens, experts, slots, width,
                                                                 hidden, outer))
    if n < 0:
        _lib.check(_lib.ERR_ARG)
    return n


def expert_layer(x, weights, slots, inner, outer, activation="silu", *, workspace=None):
    """A layer of experts: ``x`` (tokens, width) and the tokens' ``weights`` over the experts
    (tokens, experts) to (tokens, outer width), the sum over a token's ``slots`` largest positive
    weights (as ``route`` chooses) of weight * f(x inner[e]) outer[e].

    ``inner`` (experts, width, hidden), or (experts, width, 2 * hidden) with a gate (``activate``);
    ``outer`` (experts, hidden, outer width): tensors of x's type in either order of the last two
    dimensions, or packed (``pack(weight, "fp4", axis=1)``).  Up to 64 tokens (and 1024 slots of all
    of them) of bfloat16 or float16 without a graph run in three or four kernels, which keep the
    hidden values to twice the type's digits and need the ``workspace`` (new memory otherwise; left
    alone by other calls).  All others are the separate operators in turn, which round them to the
    type; float32 tokens, and a graph's backward pass, unpack a packed matrix of all experts for the
    length of its product.
    """
    code = _activation(activation)
    if slots.__class__ is not int:
        raise ValueError(f"slots must be a positive integer; got {slots!r}")
    a, b = (None, fields(inner)) if isinstance(inner, Microscaled) else (inner, None)
    c, d = (None, fields(outer)) if isinstance(outer, Microscaled) else (outer, None)
    if (inner is None) or (outer is None):
        raise ValueError("inner and outer must be tensors on the GPU, or packed")
    try:
        out = _front.expert_layer(x, weights, slots, a, b, c, d, code, workspace)
    except TypeError:
        raise ValueError("x, weights, inner, outer and workspace must be tensors on the GPU; got "
                         f"{type(x).__name__}, {type(weights).__name__}, {type(inner).__name__}, "
                         f"{type(outer).__name__} and {type(workspace).__name__}") from None
    if out is not None:
        return out
    routing = route(weights, slots)
    rows = expert_product(dispatch(x, routing), inner, routing)
    rows = activate(rows, activation, gated=rows.shape[1] != outer.shape[1])
    return combine(expert_product(rows, outer, routing), routing)
