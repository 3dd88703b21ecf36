"""Numbers of few bits that share a power of two: experts' weights in 4 bits, kept rows in 8.

    weight = pack(weight, "fp4", axis=1)         # (experts, inner, outer), blocks along inner
    out = expert_product(rows, weight, routing)  # or expert_layer, with weights in 4 bits

32 neighbours along an axis share 2^s, s from the largest magnitude m among them:

* ``"fp4"``: s = floor(log2 m) - 2, an element is the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 and
  their negatives to x / 2^s (ties to the even code, at most 6): 4.25 bits an element;
* ``"int8"``: s = floor(log2 m), an element is x / 2^s in 64ths, from -127 to 127: 8.25 bits.

s is at least -127.  A block with an infinity or NaN is NaN.  The values are exact in the type that
was packed.  Every call runs in the HIP library (``include/purin_train.h``) on the current stream of
its tensors' device and waits for nothing.  The reference has no counterpart.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from purin_amd import _lib

_lib.load()
from purin_amd import _front  # noqa: E402  (linked to the library, which is built with it)

KINDS = {"fp4": _lib.FP4, "int8": _lib.INT8}


@dataclass(eq=False)
class Microscaled:
    """A tensor of ``shape`` in few bits, its blocks of 32 along ``axis``.

    With that axis moved last and ``blocks`` = ceil(length / 32): ``codes`` uint8 (..., blocks * 16)
    for "fp4", two elements to a byte, the earlier one in the lower half, the sign above the
    magnitude's index; (..., blocks * 32) for "int8"; ``scales`` uint8 (..., blocks rounded up to a
    multiple of 4), s + 127, or 255 for NaN.  What is behind the length is zero in both, and has to
    be.  ``dtype``: the type that was packed, and that ``unpack`` gives.  The fields are a caller's
    to make from weights that come in this form: types and shapes are checked at each call.
    """

    codes: torch.Tensor
    scales: torch.Tensor
    kind: str
    shape: tuple
    axis: int
    dtype: torch.dtype


def kind_code(kind):
    if not isinstance(kind, str) or kind not in KINDS:
        raise ValueError(f'kind must be "fp4" or "int8"; got {kind!r}')
    return KINDS[kind]


def fields(packed):
    """What the front end takes of a Microscaled."""
    if not isinstance(packed.shape, (tuple, list)):
        raise ValueError(f"a Microscaled's shape must be a tuple; got {packed.shape!r}")
    return packed.codes, packed.scales, kind_code(packed.kind), list(packed.shape), packed.axis


def kept(saved):
    """Whether ``saved`` asks for rows in 8 bits."""
    if saved is not None and saved != "int8":
        raise ValueError(f'saved must be None or "int8"; got {saved!r}')
    return saved is not None


def pack(tensor, kind, axis=-1):
    """``tensor`` (float32, bfloat16 or float16, any strides) as a ``Microscaled`` of ``kind``,
    blocks along ``axis``.  It has no gradient, and refuses a tensor that wants one."""
    code = kind_code(kind)
    try:
        codes, scales = _front.pack(tensor, code, axis)
    except TypeError:
        raise ValueError("tensor must be a tensor on the GPU and axis an integer; got "
                         f"{type(tensor).__name__} and {axis!r}") from None
    return Microscaled(codes, scales, kind, tuple(tensor.shape), axis % tensor.dim(), tensor.dtype)


def unpack(packed, dtype=None):
    """The values that a ``Microscaled`` stands for, in its own type or ``dtype`` (float32, bfloat16
    or float16, rounded where that is narrower); its axis is contiguous in memory."""
    if not isinstance(packed, Microscaled):
        raise ValueError(f"packed must be a Microscaled; got {type(packed).__name__}")
    try:
        return _front.unpack(*fields(packed), packed.dtype if dtype is None else dtype)
    except TypeError:
        raise ValueError("a Microscaled's codes and scales must be tensors on the GPU, its shape a "
                         "tuple of integers, its axis an integer and dtype a torch.dtype") from None
