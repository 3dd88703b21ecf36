"""The float64 oracle of the operators around the projection layer: known answers, and its
gradients against differences (CPU)."""

import numpy as np

from oracle import train as ot


def test_choose_known_answers():
    nan, inf = np.nan, np.inf
    w = np.array([[0.2, 0.5, 0.2, 0.0],       # ties go to the lowest expert
                  [0.0, 0.0, 0.0, 0.0],       # nothing
                  [-1.0, -inf, 0.1, -0.0],    # one positive
                  [1.0, nan, inf, 2.0]])      # NaN, infinity, then numbers
    ids, chosen = ot.choose(w, 3)
    np.testing.assert_array_equal(ids, [[1, 0, 2], [-1, -1, -1], [2, -1, -1], [1, 2, 3]])
    np.testing.assert_array_equal(chosen, [[0.5, 0.2, 0.2], [0, 0, 0], [0.1, 0, 0],
                                           [nan, inf, 2.0]])


def test_sort_is_stable_and_drops_what_names_no_expert():
    ids, offsets, place, source = ot.sort(np.array([[2, 0], [-1, 2], [0, 7]]), 3)
    np.testing.assert_array_equal(ids, [[2, 0], [-1, 2], [0, -1]])
    np.testing.assert_array_equal(offsets, [0, 2, 2, 4])
    np.testing.assert_array_equal(place, [[2, 0], [-1, 3], [1, -1]])
    np.testing.assert_array_equal(source, [1, 4, 0, 3, -1, -1])


def _differences(f, x, h=1e-6):
    g = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        a, b = x.copy(), x.copy()
        a[i] += h
        b[i] -= h
        g[i] = (f(a) - f(b)) / (2 * h)
    return g


def test_gradients_against_differences():
    rng = np.random.default_rng(3)
    tokens, count, slots, width, outer = 5, 4, 2, 3, 4
    w = rng.uniform(0.1, 1.0, (tokens, count)) * (rng.random((tokens, count)) < 0.6)
    w[2] = 0.0
    ids, _ = ot.choose(w, slots)
    _, offsets, place, _ = ot.sort(ids, count)
    x = rng.normal(size=(tokens, width))
    matrix = rng.normal(size=(count, width, outer))
    cot = rng.normal(size=(tokens, outer))

    def loss(x, w, matrix):
        chosen = np.where(ids >= 0, np.take_along_axis(w, np.maximum(ids, 0), 1), 0.0)
        rows = ot.product(ot.dispatch(x, place), matrix, offsets)
        return float((cot * ot.combine(rows, place, chosen)).sum())

    chosen = np.where(ids >= 0, np.take_along_axis(w, np.maximum(ids, 0), 1), 0.0)
    rows = ot.dispatch(x, place)
    y = ot.product(rows, matrix, offsets)
    g_y, g_chosen = ot.combine_vjp(cot, y, place, chosen)
    g_rows, g_matrix = ot.product_vjp(g_y, rows, matrix, offsets)
    g_x = ot.combine(g_rows, place, np.ones_like(chosen))
    g_w = ot.route_vjp(ids, g_chosen, count)
    # central differences of a polynomial of degree 3: h^2 plus rounding / h
    tol = dict(rtol=0, atol=1e-7)
    np.testing.assert_allclose(g_x, _differences(lambda v: loss(v, w, matrix), x), **tol)
    np.testing.assert_allclose(g_matrix, _differences(lambda v: loss(x, w, v), matrix), **tol)
    inside = w > 0  # an entry at zero has no two-sided difference
    got = _differences(lambda v: loss(x, v, matrix), w)
    np.testing.assert_allclose(g_w[inside], got[inside], **tol)


def test_clip_known_answers():
    norm, out = ot.clip([np.array([3.0]), np.array([[4.0]])], 1.0)
    assert norm == 5.0 and abs(out[0][0] - 0.6) < 1e-15 and abs(out[1][0, 0] - 0.8) < 1e-15
    norm, out = ot.clip([np.array([3.0]), np.array([4.0])], 5.0)
    assert norm == 5.0 and out[0][0] == 3.0
    assert ot.clip([], 1.0)[0] == 0.0
