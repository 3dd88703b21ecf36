"""The oracle of microscaled numbers, the activation and the layer against what is known of them."""

import math

import numpy as np
import pytest

from oracle import experts as oe


def test_fp4_rounds_to_the_nearest_and_ties_to_even():
    borders = [(0.25, 0.0), (0.75, 1.0), (1.25, 1.0), (1.75, 2.0), (2.5, 2.0), (3.5, 4.0), (5.0, 4.0),
               (0.26, 0.5), (5.01, 6.0), (7.9, 6.0), (6.0, 6.0)]
    for x, want in borders:
        block = np.zeros((1, 32))
        block[0, 0], block[0, 1], block[0, 2] = 4.0, x if x < 4 else 0.0, -x if x < 4 else 0.0
        if x >= 4:
            block[0, 0] = x
            assert oe.values(block, "fp4")[0, 0] == want
        else:
            assert oe.values(block, "fp4")[0, 1] == want and oe.values(block, "fp4")[0, 2] == -want


@pytest.mark.parametrize("kind", ["fp4", "int8"])
def test_values_are_within_half_a_step_and_stay_fixed(kind):
    rng = np.random.default_rng(0)
    x = rng.normal(size=(7, 75)) * np.exp(rng.normal(size=(7, 1)) * 5)
    y = oe.values(x, kind)
    for r in range(7):
        for b in range(0, 75, 32):
            most = np.abs(x[r, b:b + 32]).max()
            step = 2.0 ** math.floor(math.log2(most))
            # fp4: half of the widest step (2 / 4 of it), or what is cut off above 6; int8: half a
            # 64th, and a whole one at the end of the range
            bound = step / 2 if kind == "fp4" else step / 64
            assert np.abs(x[r, b:b + 32] - y[r, b:b + 32]).max() <= bound
    np.testing.assert_array_equal(oe.values(y, kind), y)


def test_int8_holds_what_fp4_holds():
    rng = np.random.default_rng(1)
    y = oe.values(rng.normal(size=(5, 64)), "fp4")
    np.testing.assert_array_equal(oe.values(y, "int8"), y)


@pytest.mark.parametrize("kind", ["fp4", "int8"])
def test_odd_blocks(kind):
    tiny, inf, nan = 2.0 ** -149, math.inf, math.nan
    x = np.zeros((5, 40))
    x[1, 3] = tiny
    x[2, 5], x[2, 6] = inf, 1.0
    x[3, 39] = nan
    x[4] = -0.0
    codes, scales = oe.pack(x, kind)
    assert scales.shape == (5, 4) and (scales[:, 2:] == 0).all() and scales[0, 0] == 0
    assert scales[2, 0] == 255 and scales[2, 1] == 0 and scales[3, 1] == 255
    y = oe.unpack(codes, scales, kind, 40)
    assert np.isnan(y[2, :32]).all() and (y[2, 32:] == 0).all() and np.isnan(y[3, 32:]).all()
    assert (y[[0, 1, 4]] == 0).all()
    assert codes.shape[1] == (32 if kind == "fp4" else 64)


@pytest.mark.parametrize("kind", ["relu", "silu", "gelu"])
@pytest.mark.parametrize("gated", [False, True])
def test_activation_gradients_by_differences(kind, gated):
    rng = np.random.default_rng(2)
    u, g = rng.normal(size=(3, 8)), rng.normal(size=(3, 4 if gated else 8))
    got = oe.activate_vjp(u, g, kind, gated)
    for i in np.ndindex(u.shape):
        d = np.zeros_like(u)
        d[i] = 1e-5
        slope = ((oe.activate(u + d, kind, gated) - oe.activate(u - d, kind, gated)) * g).sum() / 2e-5
        assert abs(slope - got[i]) < 1e-8


def test_layer_is_the_sum_over_the_chosen_experts():
    rng = np.random.default_rng(3)
    x, w = rng.normal(size=(3, 5)), np.array([[0.5, 0.0, 0.25], [0.0, 0.0, 0.0], [0.1, 0.2, 0.3]])
    a, b = rng.normal(size=(3, 5, 8)), rng.normal(size=(3, 4, 6))
    out, _ = oe.layer(x, w, 2, a, b, "silu")
    one = lambda t, e: oe.activate((x[t] @ a[e])[None], "silu", True)[0] @ b[e]  # noqa: E731
    np.testing.assert_allclose(out[0], 0.5 * one(0, 0) + 0.25 * one(0, 2))
    assert (out[1] == 0).all()
    np.testing.assert_allclose(out[2], 0.3 * one(2, 2) + 0.2 * one(2, 1))
