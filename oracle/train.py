"""The operators around the projection layer, from their definitions, in float64 numpy.

Written apart from the HIP kernels and from torch; the GPU tests compare with it.  Inputs are
numpy arrays of any type (the values as stored); sums and products are float64.
"""

from __future__ import annotations

import numpy as np


def choose(weights, slots):
    """(ids, chosen): a token's largest positive weights, ties to the lowest expert, NaN first."""
    w = np.asarray(weights, np.float64)
    tokens = w.shape[0]
    ids = np.full((tokens, slots), -1, np.int64)
    chosen = np.zeros((tokens, slots))
    for t in range(tokens):
        row = w[t]
        order = sorted((e for e in range(w.shape[1]) if row[e] > 0 or np.isnan(row[e])),
                       key=lambda e: (0 if np.isnan(row[e]) else 1,
                                      0.0 if np.isnan(row[e]) else -row[e], e))
        for j, e in enumerate(order[:slots]):
            ids[t, j], chosen[t, j] = e, row[e]
    return ids, chosen


def sort(ids, count):
    """(ids, offsets, place, source) of pairs sorted stably by expert."""
    ids = np.asarray(ids)
    ids = np.where((ids >= 0) & (ids < count), ids, -1)
    flat = ids.reshape(-1)
    place = np.full(flat.size, -1, np.int64)
    source = np.full(flat.size, -1, np.int64)
    offsets = np.zeros(count + 1, np.int64)
    p = 0
    for e in range(count):
        for i in np.flatnonzero(flat == e):
            place[i], source[p] = p, i
            p += 1
        offsets[e + 1] = p
    return ids, offsets, place.reshape(ids.shape), source


def route_vjp(ids, g_chosen, count):
    out = np.zeros((ids.shape[0], count))
    for t, j in zip(*np.nonzero(ids >= 0)):
        out[t, ids[t, j]] += g_chosen[t, j]
    return out


def dispatch(x, place):
    rows = np.zeros((place.size, x.shape[1]))
    for t, j in zip(*np.nonzero(place >= 0)):
        rows[place[t, j]] = x[t]
    return rows


def combine(rows, place, weights):
    rows = np.asarray(rows, np.float64)
    out = np.zeros((place.shape[0], rows.shape[1]))
    for t, j in zip(*np.nonzero(place >= 0)):
        out[t] += weights[t, j] * rows[place[t, j]]
    return out


def combine_vjp(g_out, rows, place, weights):
    g_out, rows = np.asarray(g_out, np.float64), np.asarray(rows, np.float64)
    g_rows, g_weights = np.zeros(rows.shape), np.zeros(place.shape)
    for t, j in zip(*np.nonzero(place >= 0)):
        g_rows[place[t, j]] = weights[t, j] * g_out[t]
        g_weights[t, j] = g_out[t] @ rows[place[t, j]]
    return g_rows, g_weights


def product(rows, weight, offsets):
    rows, weight = np.asarray(rows, np.float64), np.asarray(weight, np.float64)
    out = np.zeros((rows.shape[0], weight.shape[2]))
    for e in range(weight.shape[0]):
        a, z = offsets[e], offsets[e + 1]
        out[a:z] = rows[a:z] @ weight[e]
    return out


def product_vjp(g, rows, weight, offsets):
    g, rows = np.asarray(g, np.float64), np.asarray(rows, np.float64)
    weight = np.asarray(weight, np.float64)
    g_rows, g_weight = np.zeros(rows.shape), np.zeros(weight.shape)
    for e in range(weight.shape[0]):
        a, z = offsets[e], offsets[e + 1]
        g_rows[a:z] = g[a:z] @ weight[e].T
        g_weight[e] = rows[a:z].T @ g[a:z]
    return g_rows, g_weight


def clip(gradients, largest):
    """(norm, scaled gradients)."""
    with np.errstate(over="ignore", invalid="ignore"):
        gradients = [np.asarray(g, np.float64) for g in gradients]
        norm = np.sqrt(sum((g * g).sum() for g in gradients))
        factor = 1.0 if norm <= largest else largest / norm
        return norm, [g * factor for g in gradients]
