"""The experts' products at sizes where the widest kernels use every place of their rings again,
and where the 64-bit products take their taller tiles."""

import numpy as np
import pytest

import tests.test_gpu_train as base
from tests._gpu import require_gpu

pytestmark = pytest.mark.gpu

# rows, experts, inner, outer.  Products of 256 x 256 tiles (from 4096 tiles of 128 x 128 on): a
# contraction of five stages of 64 and a part in a ring of two, forward and the rows' gradient;
# on 16-byte rows and off them.  Weights' gradients of 256 x 256 tiles (from 4096 tiles of
# 128 x 128 over all experts): some hundred rows to an expert, five stages and more.
WIDE = [(16400, 4, 328, 4104), (16401, 4, 331, 4099), (33000, 3, 2056, 2056), (1900, 4, 4104, 4104),
        (1903, 4, 4099, 4101)]


def _tiles(n):
    return -(-n // 128)


def test_the_sizes_reach_the_widest_tiles():
    rows, experts, inner, outer = WIDE[0]
    assert _tiles(rows) * _tiles(outer) >= 4096 and inner > 5 * 64
    rows, experts, inner, outer = WIDE[2]
    assert _tiles(rows) * _tiles(outer) >= 4096 and _tiles(rows) * _tiles(inner) >= 4096
    rows, experts, inner, outer = WIDE[3]
    assert experts * _tiles(inner) * _tiles(outer) >= 4096 and 0.9 * rows / experts > 5 * 64


@pytest.mark.parametrize("rows,experts,inner,outer", WIDE)
@pytest.mark.parametrize("order", ["io", "oi"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_wide_products(rows, experts, inner, outer, order, dtype):
    base.test_large_products(rows, experts, inner, outer, order, dtype)


# 64-bit products of 64 x 64 tiles: more than 32 rows to an expert, and at least 512 tiles of
# 64 x 64 (rows / 64 times outer / 64); the rows' gradient has them where inner is as long
DOUBLE = [(2100, 3, 520, 1100), (2101, 2, 1031, 1033), (4200, 5, 70, 580)]


@pytest.mark.parametrize("rows,experts,inner,outer", DOUBLE)
@pytest.mark.parametrize("order", ["io", "oi"])
def test_tall_products_in_64_bits(rows, experts, inner, outer, order):
    """Against torch's product in 64 bits: of K terms ours is within 2 (K + 2) roundings of the
    sum of their magnitudes, and torch's within K + 1."""
    torch = require_gpu()
    from purin_amd import expert_product

    print(f"tall product {rows} {experts} {inner} {outer} {order}", flush=True)
    assert rows > 32 * experts and (rows // 64) * -(-outer // 64) >= 512
    counts = base._counts(rows, experts, rows)
    offsets = np.concatenate(([0], np.cumsum(counts)))
    g = torch.Generator(device="cuda").manual_seed(rows)
    make = lambda *s: torch.randn(s, generator=g, device="cuda", dtype=torch.float64)  # noqa: E731
    a = make(rows, inner).requires_grad_()
    w = make(experts, inner, outer) if order == "io" else make(experts, outer, inner).transpose(1, 2)
    w.requires_grad_()
    cot = make(rows, outer)
    out = expert_product(a, w, torch.as_tensor(offsets, dtype=torch.int32).cuda())
    g_a, g_w = torch.autograd.grad(out, (a, w), cot)

    def check(got, x, y):
        k = x.shape[1]
        bound = (2 * (k + 2) + k + 1) * 2.0 ** -53 * (x.abs() @ y.abs()) * 1.01
        assert ((got - x @ y).abs() <= bound).all()

    a, w = a.detach(), w.detach()
    for e in range(experts):
        i, j = int(offsets[e]), int(offsets[e + 1])
        if i == j:
            assert (g_w[e] == 0).all()
            continue
        check(out[i:j], a[i:j], w[e])
        check(g_a[i:j], cot[i:j], w[e].T)
        check(g_w[e], a[i:j].T, cot[i:j])
    last = int(offsets[-1])
    assert last < rows and (out[last:] == 0).all() and (g_a[last:] == 0).all()
