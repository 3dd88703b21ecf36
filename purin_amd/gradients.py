"""The global norm of a step's gradients, and clipping by it.

Gradients that come through a projection layer's implicit VJP have no bound of their own: near
a degenerate active set the fixed point's linear system is close to singular.  A training step
limits their norm over all parameters together before the optimizer reads them.

Both calls run in the HIP library (``include/purin_train.h``) on the current stream of the
tensors' device and wait for nothing: the norm comes back as a tensor.  The reference has no
counterpart.
"""

from __future__ import annotations

import torch

from purin_amd import _lib

_lib.load()
from purin_amd import _front  # noqa: E402  (linked to the library, which is built with it)


def _list(tensors, name):
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    for i, t in enumerate(tensors):
        if t is not None and not isinstance(t, torch.Tensor):
            raise ValueError(f"{name}[{i}] must be a tensor on the GPU; got {type(t).__name__}")
    return tensors


def clip_workspace_bytes(tensors):
    """Bytes of a caller's workspace, a contiguous device tensor at 256 bytes, for a list of
    ``tensors`` gradients."""
    n = int(_lib.load().purin_train_clip_workspace_bytes(tensors))
    if n < 0:
        _lib.check(_lib.ERR_ARG)
    return n


def gradient_norm(gradients, *, workspace=None):
    """The 2-norm of all gradients together: a tensor without dimensions, float64 if any gradient
    is, float32 otherwise.  ``gradients``: a tensor, or a list whose ``None`` are left out; mixed
    types are fine.  Squares are summed in 64 bits, in an order that the sizes alone decide; those
    of float64 elements leave that range beyond about 1e154 (an infinite norm) and below 1e-162.
    Differentiable once (a gradient's is itself over the norm, zero where the norm is), so that a
    penalty on gradients reaches what they were made from."""
    return _front.gradient_norm(_list(gradients, "gradients"), workspace)


def clip_gradients(gradients, largest, out=None, *, workspace=None):
    """Scale the gradients, in place, to a global norm of at most ``largest``; returns the norm
    before (as ``gradient_norm``).

    Where the norm is not above ``largest`` nothing is written.  ``out``: tensors of the
    gradients' shapes and types to write instead, in full, the gradients staying as they are
    (``None`` beside ``None``).  An output that shares memory with another tensor of the call is
    refused, except a gradient's own ``out``.  A NaN norm makes all gradients NaN; an infinite one
    makes finite gradients zero and infinite ones NaN: the returned norm tells.  Autograd does
    not see the call: neither the norm nor what is written has a graph.
    """
    return _front.clip_gradients(_list(gradients, "gradients"), float(largest),
                                 None if out is None else _list(out, "out"), workspace)
