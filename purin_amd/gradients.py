"""The global norm of a step's gradients, and clipping by it.

Gradients that come through a projection layer's implicit VJP have no bound of their own: near
a degenerate active set the fixed point's linear system is close to singular.  A training step
limits their norm over all parameters together before the optimizer reads them.

Both calls run in the HIP library (``include/purin_train.h``) on the current stream of the
tensors' device and wait for nothing: the norm comes back as a tensor.  The reference has no
counterpart.
"""

from __future__ import annotations

import math

import torch

from purin_amd import _lib
from purin_amd.routing import _CODES, _call, _float_code, _workspace


def _dense(t):
    """Whether the tensor's elements fill one span of memory, each once, in whatever order."""
    if t.is_contiguous():
        return True
    need = 1
    for stride, size in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if stride != need:
            return False
        need *= size
    return True


def _overlaps_itself(t):
    """Whether some element of a strided tensor may share its place with another."""
    need = 1
    for stride, size in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if stride < need:
            return True
        need = stride * (size - 1) + need
    return False


def _run(pairs, largest, workspace):
    device = pairs[0][0].device if pairs else torch.device("cuda", torch.cuda.current_device())
    table = (_lib.TrainTensor * max(1, len(pairs)))()
    wide = False
    for row, (g, out) in zip(table, pairs):
        row.in_ = g.data_ptr()
        row.out = out.data_ptr()
        row.count = g.numel()
        row.dtype = _CODES[g.dtype]
        wide = wide or g.dtype == torch.float64
    norm = torch.empty((), dtype=torch.float64 if wide else torch.float32, device=device)
    need = _lib.load().purin_train_clip_workspace_bytes(len(pairs))
    _, ws, ws_bytes = _workspace(workspace, need, device)
    _call("purin_train_clip", device, len(pairs), table, largest, ws, ws_bytes,
          _lib.F64 if wide else _lib.F32, norm.data_ptr())
    return norm


def _list(gradients, name):
    if isinstance(gradients, torch.Tensor):
        gradients = [gradients]
    tensors = list(gradients)
    for i, t in enumerate(tensors):
        if t is None:
            continue
        _float_code(t, f"{name}[{i}]")
        if t.layout != torch.strided:
            raise ValueError(f"{name}[{i}] must be a dense tensor")
    return tensors


def _one_device(tensors, name):
    devices = {t.device for t in tensors}
    if len(devices) > 1:
        raise ValueError(f"{name} must be on one device; got {sorted(map(str, devices))}")


def clip_workspace_bytes(tensors):
    """Bytes of a caller's workspace for a list of ``tensors`` gradients (256-byte aligned)."""
    return int(_lib.load().purin_train_clip_workspace_bytes(tensors))


@torch.no_grad()
def gradient_norm(gradients, *, workspace=None):
    """The 2-norm of all gradients together: a tensor without dimensions, float64 if any gradient
    is, float32 otherwise.  ``gradients``: a tensor, or a list whose ``None`` are left out; mixed
    types are fine.  Squares are summed in 64 bits, in an order that the sizes alone decide."""
    tensors = [t for t in _list(gradients, "gradients") if t is not None]
    _one_device(tensors, "gradients")
    tensors = [t if _dense(t) else t.contiguous() for t in tensors]
    return _run([(t, t) for t in tensors], -1.0, workspace)


@torch.no_grad()
def clip_gradients(gradients, largest, out=None, *, workspace=None):
    """Scale the gradients, in place, to a global norm of at most ``largest``; returns the norm
    before (as ``gradient_norm``).

    Where the norm is not above ``largest`` nothing is written.  ``out``: tensors of the
    gradients' shapes and types to write instead, in full, the gradients staying as they are
    (``None`` beside ``None``).  No two tensors may share memory, but a gradient and its own
    ``out``.  A NaN norm makes all gradients NaN; an infinite one makes finite gradients zero
    and infinite ones NaN: the returned norm tells.
    """
    largest = float(largest)
    if math.isnan(largest) or largest < 0.0:
        raise ValueError(f"largest must not be negative; got {largest}")
    tensors = _list(gradients, "gradients")
    outs = tensors if out is None else _list(out, "out")
    if len(outs) != len(tensors):
        raise ValueError(f"out must hold {len(tensors)} tensors; got {len(outs)}")
    pairs, back = [], []
    for i, (g, o) in enumerate(zip(tensors, outs)):
        if (g is None) != (o is None):
            raise ValueError(f"out[{i}] must be None exactly where the gradient is")
        if g is None:
            continue
        if o is not g and (o.shape != g.shape or o.dtype != g.dtype):
            raise ValueError(f"out[{i}] must have shape {tuple(g.shape)} and type {g.dtype}; got "
                             f"{tuple(o.shape)} and {o.dtype}")
        if o.is_contiguous() and (o is g or g.is_contiguous()):
            pairs.append((g, o))
            continue
        if _overlaps_itself(o):
            raise ValueError(f"out[{i}] (or the gradient in place) has elements that share memory")
        if o is g and _dense(g):
            pairs.append((g, g))
            continue
        # any other order goes through a copy in order
        c = torch.empty(o.shape, dtype=o.dtype, device=o.device)
        pairs.append((g.contiguous(), c))
        back.append((o, c))
    _one_device([t for p in pairs for t in p], "gradients and out")
    norm = _run(pairs, largest, workspace)
    for o, c in back:
        o.copy_(c)
    # autograd's check for tensors that changed after they were saved
    torch.autograd.graph.increment_version([o for o in outs if o is not None])
    return norm
