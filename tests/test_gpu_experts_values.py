"""Infinities in rows, hidden values and weights of layers and of products with packed weights.

No tolerance: an infinity times a number that is not zero is one of its product's sign, sums of
infinities of one sign stay, and what has none is finite.  float64 numpy says which of the three
each result is.  Contractions are as long as several wavefronts' parts, and every part has rows
whose infinity lies there.
"""

import numpy as np
import pytest

from tests._gpu import require_gpu
from tests.test_gpu_train import _np, _types

pytestmark = pytest.mark.gpu

HALF = ["bf16", "f16"]
# whole lines of 64 (dense) or 256 (codes) and others, odd and even numbers of them to a part
LENGTHS = [64, 192, 320, 576, 768, 1000, 1024, 1096, 1280, 1536, 2112, 2560]


def _kinds(a):
    """0 where finite, the sign where infinite, 2 where NaN."""
    a = np.asarray(a, np.float64)
    return np.where(np.isnan(a), 2, np.where(np.isinf(a), np.sign(a), 0))


def _same_kinds(got, want):
    got, want = _kinds(_np(got)), _kinds(want)
    bad = got != want
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


def _nonzero(torch, seed, shape, dtype, scale):
    """From scale to 2 scale, either sign: no zero in 4 bits either."""
    g = torch.Generator().manual_seed(seed)
    w = (1 + torch.rand(shape, generator=g)) * scale
    return (w * (1 - 2 * torch.randint(0, 2, shape, generator=g))).to(dtype).cuda()


def _given(torch, w, form):
    """A weight in one of its forms, and the numbers it stands for."""
    from purin_amd import pack, unpack

    if form == "packed":
        m = pack(w, "fp4", axis=1)
        return m, _np(unpack(m))
    if form == "io":
        return w.contiguous(), _np(w)
    if form == "odd":  # at any address
        wide = torch.zeros((w.shape[0], w.shape[1], w.shape[2] + 1), dtype=w.dtype, device=w.device)
        wide[:, :, 1:] = w
        return wide[:, :, 1:], _np(w)
    return w.transpose(1, 2).contiguous().transpose(1, 2), _np(w)


def _spread(length, rows):
    """A place in the contraction for each row, over all of it."""
    return np.linspace(0, length - 1, rows).astype(int)


@pytest.mark.parametrize("inner", LENGTHS)
@pytest.mark.parametrize("rows,experts,outer", [(16, 1, 40), (40, 1, 72), (41, 3, 136)])
@pytest.mark.parametrize("dtype", HALF)
def test_infinite_rows_of_products_with_packed_weights(inner, rows, experts, outer, dtype):
    torch = require_gpu()
    from purin_amd import expert_product

    print(f"infinite rows {inner} {rows} {experts} {outer} {dtype}", flush=True)
    t = _types(torch)[dtype]
    m, w = _given(torch, _nonzero(torch, 1, (experts, inner, outer), t, 0.125), "packed")
    a = _nonzero(torch, 2, (rows, inner), t, 0.125)
    a[torch.arange(rows), torch.as_tensor(_spread(inner, rows))] = float("inf")
    offsets = np.linspace(0, rows, experts + 1).astype(np.int32)
    out = expert_product(a, m, torch.as_tensor(offsets).cuda())
    want = np.concatenate([_np(a)[i:j] @ w[e]
                           for e, (i, j) in enumerate(zip(offsets[:-1], offsets[1:]))])
    assert np.isinf(want).all()
    _same_kinds(out, want)


@pytest.mark.parametrize("width", LENGTHS)
@pytest.mark.parametrize("form", ["io", "oi", "odd", "packed"])
@pytest.mark.parametrize("tokens", [3, 16, 40])
@pytest.mark.parametrize("dtype", HALF)
def test_infinite_tokens_of_layers(width, form, tokens, dtype):
    """Every hidden value of a token with an infinity is infinite or, through relu, zero."""
    torch = require_gpu()
    from purin_amd import expert_layer

    print(f"infinite tokens {width} {form} {tokens} {dtype}", flush=True)
    t = _types(torch)[dtype]
    a, an = _given(torch, _nonzero(torch, 1, (2, width, 40), t, 0.125), form)
    b, bn = _given(torch, _nonzero(torch, 2, (2, 40, 24), t, 0.125).abs(), form)
    x = _nonzero(torch, 3, (tokens, width), t, 0.125)
    x[torch.arange(tokens), torch.as_tensor(_spread(width, tokens))] = float("inf")
    w = torch.ones((tokens, 2), device="cuda")
    out = expert_layer(x, w, 2, a, b, "relu")
    assert bool((out == float("inf")).all())
    h = [np.maximum(_np(x) @ an[e], 0.0) for e in range(2)]
    with np.errstate(invalid="ignore"):
        _same_kinds(out, h[0] @ bn[0] + h[1] @ bn[1])


@pytest.mark.parametrize("hidden", LENGTHS)
@pytest.mark.parametrize("form", ["io", "oi", "odd", "packed"])
@pytest.mark.parametrize("tokens", [3, 16, 40])
def test_hidden_values_beyond_the_range_in_every_part(hidden, form, tokens):
    """float16: one hidden value of 90000 to a token, which is infinite in the type."""
    torch = require_gpu()
    from purin_amd import expert_layer

    print(f"hidden {hidden} {form} {tokens}", flush=True)
    a = torch.zeros((1, 64, hidden), device="cuda")
    a[0, torch.arange(tokens), torch.as_tensor(_spread(hidden, tokens))] = 256.0
    a, _ = _given(torch, a.half(), form)
    b, _ = _given(torch, _nonzero(torch, 2, (1, hidden, 24), torch.float16, 2.0 ** -10), form)
    x = torch.zeros((tokens, 64), dtype=torch.float16, device="cuda")
    x[torch.arange(tokens), torch.arange(tokens)] = 352.0
    out = expert_layer(x, torch.ones((tokens, 1), device="cuda"), 1, a, b, "relu")
    want = np.zeros((tokens, hidden))
    want[np.arange(tokens), _spread(hidden, tokens)] = np.inf
    from purin_amd import unpack

    full = _np(unpack(b) if form == "packed" else b)[0]
    with np.errstate(invalid="ignore"):
        want = np.where(np.isinf(want), want, 1.0) @ full  # a zero changes no infinity
    assert np.isinf(want).all()
    _same_kinds(out, want)


@pytest.mark.parametrize("form", ["io", "oi", "odd", "packed"])
@pytest.mark.parametrize("tokens,hidden", [(1, 64), (3, 40), (16, 768), (40, 200), (64, 264)])
@pytest.mark.parametrize("exact", [True, False])  # whether hidden values are numbers of the type
@pytest.mark.parametrize("dtype", HALF)
def test_infinite_weights_of_a_layers_second_product(form, tokens, hidden, exact, dtype):
    """Columns with an infinite weight: infinite where the hidden values are not zero.  In codes:
    weights above float16's range, which are infinite beside float16 (codes have no infinity of
    their own)."""
    torch = require_gpu()
    from purin_amd import Microscaled, expert_layer

    print(f"infinite weights {form} {tokens} {hidden} {exact} {dtype}", flush=True)
    t = _types(torch)[dtype]
    a = torch.full((1, 64, hidden), 0.25) if exact else 0.01 + _nonzero(
        torch, 1, (1, 64, hidden), torch.float32, 0.25).abs().cpu()
    a, _ = _given(torch, a.to(t).cuda(), form)
    b = _nonzero(torch, 2, (1, hidden, 40), t, 2.0 ** -8)
    if form == "packed":
        # a block of 32 is above the range as a whole
        wide = b.float()
        wide[0, :32, 3], wide[0, -(hidden % 32 or 32):, 17] = 2.0 ** 17, -(2.0 ** 17)
        b, full = _given(torch, wide, form)
        b = Microscaled(b.codes, b.scales, b.kind, b.shape, b.axis, t)
        if dtype == "f16":
            full = np.where(np.abs(full) > 65504, np.copysign(np.inf, full), full)
    else:
        b[0, 0, 3], b[0, hidden - 1, 17], b[0, hidden // 2, 18] = (float("inf"), -float("inf"),
                                                                    float("inf"))
        b, full = _given(torch, b, form)
    x = torch.ones((tokens, 64), device="cuda").to(t)
    out = expert_layer(x, torch.ones((tokens, 1), device="cuda"), 1, a, b, "relu")
    _same_kinds(out, np.broadcast_to(np.ones(hidden) @ full[0], (tokens, 40)))
