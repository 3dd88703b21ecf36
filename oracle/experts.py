"""Microscaled numbers, the activation and a whole layer of experts, from their definitions, in
float64 numpy.

Written apart from the HIP kernels and from torch; the GPU tests compare with it.  Inputs are
numpy arrays (the values as stored); sums and products are float64.
"""

from __future__ import annotations

import math

import numpy as np

from oracle import train

BLOCK = 32
FP4 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _scale_exponent(block, kind):
    """s of a block, None where it is NaN."""
    if not np.isfinite(block).all():
        return None
    most = float(np.max(np.abs(block), initial=0.0))
    if most == 0.0:
        return -127
    return max(math.frexp(most)[1] - 1 - (2 if kind == "fp4" else 0), -127)


def _nearest_fp4(a):
    """Index of the nearest magnitude, ties to the even index."""
    a = min(a, 6.0)
    distance = np.abs(FP4 - a)
    best = np.flatnonzero(distance == distance.min())
    return int(best[0] if best[0] % 2 == 0 or best.size == 1 else best[1])


def pack(rows, kind):
    """(codes, scales) uint8 of rows (rows, length)."""
    rows = np.asarray(rows, np.float64)
    n, length = rows.shape
    blocks = -(-length // BLOCK)
    filled = -(-blocks // 4) * 4
    element = np.zeros((n, blocks * BLOCK), np.uint8)
    scales = np.zeros((n, filled), np.uint8)
    for r in range(n):
        for b in range(blocks):
            x = rows[r, b * BLOCK:(b + 1) * BLOCK]
            s = _scale_exponent(x, kind)
            if s is None:
                scales[r, b] = 255
                continue
            scales[r, b] = s + 127
            for i, v in enumerate(x):
                y = math.ldexp(v, -s)
                if kind == "fp4":
                    c = _nearest_fp4(abs(y)) + (8 if math.copysign(1.0, v) < 0 else 0)
                else:
                    c = int(np.clip(np.rint(64 * y), -127, 127)) & 255
                element[r, b * BLOCK + i] = c
    if kind == "fp4":
        element = element[:, ::2] | (element[:, 1::2] << 4)
    return element, scales


def unpack(codes, scales, kind, length):
    """The values (rows, length)."""
    codes, scales = np.asarray(codes), np.asarray(scales)
    if kind == "fp4":
        both = np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1)
        value = FP4[both & 7] * np.where(both & 8, -1.0, 1.0)
    else:
        value = codes.astype(np.int8).astype(np.float64) / 64
    s = np.repeat(scales, BLOCK, 1)[:, : value.shape[1]]
    value = value * np.exp2(s.astype(np.float64) - 127)
    return np.where(s == 255, np.nan, value)[:, :length]


def values(rows, kind):
    """What packed rows stand for."""
    rows = np.asarray(rows, np.float64)
    return unpack(*pack(rows, kind), kind, rows.shape[1])


_erf = np.vectorize(math.erf, otypes=[float])


def activation(u, kind):
    """(f, slope)."""
    u = np.asarray(u, np.float64)
    with np.errstate(over="ignore"):
        if kind == "relu":
            return np.maximum(u, 0.0), (u > 0).astype(float)
        if kind == "silu":
            s = 1 / (1 + np.exp(-u))
            return u * s, s * (1 + u * (1 - s))
    share = 0.5 * (1 + _erf(u / math.sqrt(2)))
    return u * share, share + u * np.exp(-u * u / 2) / math.sqrt(2 * math.pi)


def activate(u, kind, gated):
    if not gated:
        return activation(u, kind)[0]
    h = u.shape[1] // 2
    return activation(u[:, :h], kind)[0] * u[:, h:]


def activate_vjp(u, g, kind, gated):
    if not gated:
        return activation(u, kind)[1] * g
    h = u.shape[1] // 2
    f, slope = activation(u[:, :h], kind)
    return np.concatenate((slope * u[:, h:] * g, f * g), 1)


def layer(x, weights, slots, inner, outer, kind):
    """(out, terms): the layer's result, and the sums of its second products' terms' magnitudes
    plus those that the first products' reach through the activation (slope at most 1.13)."""
    x, weights = np.asarray(x, np.float64), np.asarray(weights, np.float64)
    ids, chosen = train.choose(weights, slots)
    hidden = outer.shape[1]
    gated = inner.shape[2] != hidden
    out = np.zeros((x.shape[0], outer.shape[2]))
    terms = np.zeros_like(out)
    for t, j in zip(*np.nonzero(ids >= 0)):
        e, w = ids[t, j], chosen[t, j]
        u, size = x[t] @ inner[e], np.abs(x[t]) @ np.abs(inner[e])
        if gated:
            f = activation(u[:hidden], kind)[0]
            h = f * u[hidden:]
            reach = 1.13 * size[:hidden] * np.abs(u[hidden:]) + np.abs(f) * size[hidden:]
        else:
            h, reach = activation(u, kind)[0], 1.13 * size
        out[t] += w * (h @ outer[e])
        terms[t] += abs(w) * ((np.abs(h) + reach) @ np.abs(outer[e]))
    return out, terms
