"""The operators around the projection layer against the float64 oracle (``oracle/train.py``).

Tolerances follow from the arithmetic: a sum of K products held in the sums' type (unit
roundoff ``a``; 2 a where the matrix units round each addition their own way) and rounded once to
the output's type (unit roundoff ``u``) is within  u |exact| + 2 (K + 2) a sum|terms|  of the
exact value, and within the type's smallest step where it is near zero.
"""

import numpy as np
import pytest

from oracle import train as ot
from tests._gpu import require_gpu, to_np

pytestmark = pytest.mark.gpu

TYPES = ["f32", "f64", "bf16", "f16"]
UNIT = {"f32": 2.0 ** -24, "f64": 2.0 ** -53, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
STEP = {"f32": 2.0 ** -126, "f64": 2.0 ** -1022, "bf16": 2.0 ** -126, "f16": 2.0 ** -24}
SUMS = {"f32": 2.0 ** -24, "f64": 2.0 ** -53, "bf16": 2.0 ** -24, "f16": 2.0 ** -24}


def _types(torch):
    return {"f32": torch.float32, "f64": torch.float64, "bf16": torch.bfloat16,
            "f16": torch.float16}


def _np(t):
    """Values as float64 numpy."""
    return to_np(t.double())


def _randn(torch, seed, shape, dtype, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * scale).to(dtype).cuda()


def _weights(torch, seed, tokens, count, dtype, share=0.4):
    """Sparse non-negative weights with empty rows, ties and whole rows."""
    rng = np.random.default_rng(seed)
    w = np.round(rng.random((tokens, count)) * 64) / 64 * (rng.random((tokens, count)) < share)
    if tokens > 3:
        w[1] = 0.0
        w[2] = 0.25
    return torch.as_tensor(w).to(_types(torch)[dtype]).cuda()


def _close(got, want, terms, count, dtype, sums=None):
    """|got - want| within the derived bound; ``terms``: the sums of the terms' magnitudes."""
    got, want = _np(got), np.asarray(want)
    assert got.shape == want.shape
    a = SUMS[sums or dtype]
    bound = (UNIT[dtype] * np.abs(want) + 2 * (count + 2) * a * np.asarray(terms)
             * (1 + UNIT[dtype]) + STEP[dtype])
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (np.argwhere(bad)[:3], got[bad][:3], want[bad][:3], bound[bad][:3])


def _same_index(routing, ids, offsets, place, source):
    np.testing.assert_array_equal(to_np(routing.experts), ids)
    np.testing.assert_array_equal(to_np(routing.offsets), offsets)
    np.testing.assert_array_equal(to_np(routing.place), place)
    np.testing.assert_array_equal(to_np(routing.source), source)


# ---------------------------------------------------------------------------
# routing
# ---------------------------------------------------------------------------

ROUTES = [(1, 1, 1), (1, 64, 8), (3, 5, 5), (37, 9, 3), (200, 33, 4), (257, 130, 6),
          (700, 16, 16), (1500, 300, 2), (130, 1024, 40), (4100, 65, 3), (50, 100, 37), (90, 300, 70)]


@pytest.mark.parametrize("tokens,count,slots", ROUTES)
@pytest.mark.parametrize("dtype", TYPES)
def test_route(tokens, count, slots, dtype):
    torch = require_gpu()
    from purin_amd import route

    print(f"route {tokens} {count} {slots} {dtype}", flush=True)
    w = _weights(torch, tokens + count, tokens, count, dtype)
    r = route(w, slots)
    ids, chosen = ot.choose(_np(w), slots)
    _same_index(r, *ot.sort(ids, count))
    np.testing.assert_array_equal(_np(r.weights), chosen)
    assert r.weights.dtype == w.dtype and r.rows == tokens * slots


@pytest.mark.parametrize("dtype", TYPES)
def test_route_odd_values_and_strides(dtype):
    torch = require_gpu()
    from purin_amd import route

    t = _types(torch)[dtype]
    big, nan, inf = torch.finfo(t).max, float("nan"), float("inf")
    tiny = torch.finfo(t).smallest_normal
    w = torch.tensor([[0.0, -0.0, -1.0, -inf, -big], [big, inf, nan, tiny, 0.0],
                      [nan, nan, 1.0, 1.0, 1.0], [tiny, tiny / 4, 0.0, tiny, -tiny],
                      [-nan, 0.5, 0.5, 0.25, 0.5]], dtype=t, device="cuda")
    ids, chosen = ot.choose(_np(w), 3)
    for x in (w, torch.cat((w, w), 1)[:, 3:8].roll(0), w.t().contiguous().t()):
        if x is not w and not torch.equal(torch.nan_to_num(x), torch.nan_to_num(w)):
            x = torch.cat((w * 0 + 1, w), 1)[:, 5:]  # a row pitch wider than the row
        r = route(x, 3)
        _same_index(r, *ot.sort(ids, 5))
        np.testing.assert_array_equal(_np(r.weights), chosen)
    r = route(w[:1].expand(4, 5), 2)  # one row for all tokens
    ids, _ = ot.choose(np.repeat(_np(w[:1]), 4, 0), 2)
    _same_index(r, *ot.sort(ids, 5))
    r = route(w[:0], 2)  # no token
    assert r.rows == 0 and to_np(r.offsets).tolist() == [0] * 6


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("tokens,count,slots", [(1, 1, 1), (5, 3, 7), (900, 1000, 3),
                                                (3000, 7, 5), (20011, 256, 2)])
def test_route_experts(tokens, count, slots, wide):
    torch = require_gpu()
    from purin_amd import route_experts

    rng = np.random.default_rng(tokens)
    given = rng.integers(-2, count + 2, (tokens, slots))
    if wide:
        given[0, 0] = (1 << 32) + 0  # names expert 0 in its low half alone
    r = route_experts(torch.as_tensor(given, dtype=torch.int64 if wide else torch.int32).cuda(),
                      count)
    _same_index(r, *ot.sort(given, count))
    one = route_experts(torch.zeros((tokens, slots), dtype=torch.int32, device="cuda"), count)
    assert to_np(one.source).tolist() == list(range(tokens * slots))  # all to one expert
    none = route_experts(torch.full((tokens, slots), -1, device="cuda"), count)
    assert (to_np(none.place) == -1).all() and to_np(none.offsets)[-1] == 0


WIDTHS = [(1, 4, 2, 1), (1, 64, 8, 2048), (7, 5, 3, 16), (64, 9, 4, 37), (33, 8, 8, 511),
          (129, 17, 6, 1030), (300, 6, 1, 8), (40, 12, 5, 4104)]


@pytest.mark.parametrize("tokens,count,slots,width", WIDTHS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("wdtype", ["f32", "same", "f64"])
def test_dispatch_combine_and_gradients(tokens, count, slots, width, dtype, wdtype):
    torch = require_gpu()
    from purin_amd import combine, dispatch, route

    print(f"rows {tokens} {count} {slots} {width} {dtype} {wdtype}", flush=True)
    wdtype = dtype if wdtype == "same" else wdtype
    t = _types(torch)[dtype]
    w = _weights(torch, 5, tokens, count, wdtype).requires_grad_()
    x = _randn(torch, 1, (tokens, width), t).requires_grad_()
    y = _randn(torch, 2, (tokens * slots, width), t).requires_grad_()
    c_rows = _randn(torch, 3, (tokens * slots, width), t)
    c_out = _randn(torch, 4, (tokens, width), t)
    r = route(w, slots)
    rows, out = dispatch(x, r), combine(y, r)
    g_x, g_w, g_y = torch.autograd.grad((rows, out), (x, w, y), (c_rows, c_out))
    assert (rows.dtype, out.dtype, g_x.dtype, g_y.dtype, g_w.dtype) == (t, t, t, t, w.dtype)
    place, chosen = to_np(r.place), _np(r.weights)
    # copies are exact, zeros behind the last row
    np.testing.assert_array_equal(_np(rows), ot.dispatch(_np(x), place))
    _close(out, ot.combine(_np(y), place, chosen), ot.combine(np.abs(_np(y)), place, chosen),
           slots, dtype)
    ones = np.ones_like(chosen)
    _close(g_x, ot.combine(_np(c_rows), place, ones), ot.combine(np.abs(_np(c_rows)), place, ones),
           slots, dtype)
    want_y, want_c = ot.combine_vjp(_np(c_out), _np(y), place, chosen)
    # a weight of 64 bits is rounded to the sums' type first
    _close(g_y, want_y, np.abs(want_y), 1, dtype)
    _, terms = ot.combine_vjp(np.abs(_np(c_out)), np.abs(_np(y)), place, chosen)
    ids = to_np(r.experts)
    _close(g_w, ot.route_vjp(ids, want_c, count), ot.route_vjp(ids, terms, count), width, wdtype,
           sums=dtype)


def test_rows_with_other_strides_and_alignment():
    torch = require_gpu()
    from purin_amd import combine, dispatch, route

    w = _weights(torch, 9, 50, 7, "f32")
    r = route(w, 3)
    place, chosen = to_np(r.place), _np(r.weights)
    for dtype, t in _types(torch).items():
        wide = _randn(torch, 1, (50, 201), t)
        wide_rows = _randn(torch, 2, (150, 201), t)
        for a, z in ((1, 98), (3, 200), (0, 96)):
            x, y = wide[:, a:z], wide_rows[:, a:z]
            np.testing.assert_array_equal(_np(dispatch(x, r)), ot.dispatch(_np(x), place))
            _close(combine(y, r), ot.combine(_np(y), place, chosen),
                   ot.combine(np.abs(_np(y)), place, chosen), 3, dtype)
        x = wide.t()[:50].t()[:, :50].t()  # columns for rows
        np.testing.assert_array_equal(_np(dispatch(x, r)), ot.dispatch(_np(x), place))
        x = wide[:1].expand(50, 201)
        np.testing.assert_array_equal(_np(dispatch(x, r)), ot.dispatch(_np(x), place))
        # a gradient that is broadcast over the rows
        x = wide.clone().requires_grad_()
        (g,) = torch.autograd.grad(dispatch(x, r).sum(), x)
        np.testing.assert_array_equal(_np(g), np.repeat((place >= 0).sum(1)[:, None], 201, 1))
    assert dispatch(_randn(torch, 1, (50, 0), torch.float32), r).shape == (150, 0)


def test_masked_rows_do_not_reach_the_result():
    """Rows that no pair has, and tokens without experts: NaN and infinities there change
    nothing."""
    torch = require_gpu()
    from purin_amd import combine, dispatch, expert_product, route

    w = _weights(torch, 9, 40, 6, "f32")
    w[10:20] = 0.0
    r = route(w, 4)
    total = int(r.offsets[-1])
    assert total < r.rows
    x = _randn(torch, 1, (40, 24), torch.float32)
    x[12] = float("nan")
    rows = dispatch(x, r)
    assert torch.isfinite(rows).all() and (rows[total:] == 0).all()
    y = _randn(torch, 2, (r.rows, 24), torch.float32)
    y[total:] = float("inf")
    y[total::2] = float("nan")
    y.requires_grad_()
    out = combine(y, r)
    assert torch.isfinite(out).all() and (out[10:20] == 0).all()
    cot = _randn(torch, 3, (40, 24), torch.float32)
    cot[15] = float("nan")
    (g,) = torch.autograd.grad(out, y, cot)
    assert torch.isfinite(g).all() and (g[total:] == 0).all()
    for t in _types(torch).values():
        m = _randn(torch, 4, (6, 24, 40), t).requires_grad_()
        z = y.detach().to(t).requires_grad_()
        p = expert_product(z, m, r)
        assert torch.isfinite(p).all() and (p[total:] == 0).all()
        cot = _randn(torch, 5, tuple(p.shape), t)
        cot[total:] = float("nan")
        g_z, g_m = torch.autograd.grad(p, (z, m), cot)
        assert torch.isfinite(g_m).all() and torch.isfinite(g_z).all() and (g_z[total:] == 0).all()


def test_a_nan_weight_shows():
    torch = require_gpu()
    from purin_amd import combine, route

    w = _weights(torch, 9, 20, 6, "f32")
    w[4, 3] = float("nan")
    r = route(w, 2)
    assert int(r.experts[4, 0]) == 3
    out = combine(_randn(torch, 1, (40, 8), torch.float32), r)
    assert torch.isnan(out[4]).all() and torch.isfinite(out[:4]).all()


def test_rows_beyond_32_bit_offsets():
    """More than 2^32 elements of rows: copies and sums at both ends."""
    torch = require_gpu()
    from purin_amd import combine, dispatch, route_experts

    tokens, slots, width = 140_000, 8, 4096
    ids = torch.arange(slots, dtype=torch.int32, device="cuda").expand(tokens, slots)
    r = route_experts(ids, slots, weights=torch.ones((tokens, slots), device="cuda"))
    x = torch.arange(tokens, dtype=torch.float32, device="cuda").remainder(251)
    x = x.to(torch.bfloat16)[:, None].expand(tokens, width).contiguous()
    x[:, -1] = 7.0
    rows = dispatch(x, r)
    assert rows.numel() > 1 << 32
    for e in range(slots):  # the rows of expert e are the tokens in order
        assert torch.equal(rows[e * tokens:(e + 1) * tokens], x)
    out = combine(rows, r)
    assert torch.equal(out, x * 8)


# ---------------------------------------------------------------------------
# the experts' products
# ---------------------------------------------------------------------------

# rows to each expert (the last number: rows behind them), inner, outer
PRODUCTS = [((1, 0), 1, 1), ((0, 0, 0, 5), 8, 8), ((8, 0), 64, 64), ((1, 0, 2, 1, 0), 128, 96),
            ((3, 130, 0, 17, 2), 37, 53), ((128, 256, 64, 0), 64, 128), ((129, 1, 0, 300, 9), 200, 136),
            ((16,) * 12 + (0,), 256, 192), ((5,) * 70 + (3,), 33, 40), ((600, 40, 0), 136, 264),
            ((1,) * 3 + (0,), 2048, 72), ((2, 1, 4, 0), 72, 1408)]


@pytest.mark.parametrize("counts,inner,outer", PRODUCTS)
@pytest.mark.parametrize("order", ["io", "oi"])
@pytest.mark.parametrize("dtype", TYPES)
def test_product_and_gradients(counts, inner, outer, order, dtype):
    torch = require_gpu()
    from purin_amd import expert_product

    print(f"product {counts[:6]} {inner} {outer} {order} {dtype}", flush=True)
    t = _types(torch)[dtype]
    offsets = np.concatenate(([0], np.cumsum(counts[:-1])))
    rows, experts = int(offsets[-1]) + counts[-1], len(counts) - 1
    a = _randn(torch, 1, (rows, inner), t).requires_grad_()
    w = _randn(torch, 2, (experts, inner, outer), t, inner ** -0.5)
    w = (w if order == "io" else w.transpose(1, 2).contiguous().transpose(1, 2)).requires_grad_()
    cot = _randn(torch, 3, (rows, outer), t)
    at = torch.as_tensor(offsets, dtype=torch.int32).cuda()
    out = expert_product(a, w, at)
    g_a, g_w = torch.autograd.grad(out, (a, w), cot)
    assert out.dtype == t and g_w.stride() == w.stride()
    an, wn, cn = _np(a), _np(w), _np(cot)
    _close(out, ot.product(an, wn, offsets), ot.product(abs(an), abs(wn), offsets), inner, dtype)
    want, terms = (ot.product_vjp(c, x, m, offsets) for c, x, m in
                   ((cn, an, wn), (abs(cn), abs(an), abs(wn))))
    _close(g_a, want[0], terms[0], outer, dtype)
    most = max(counts[:-1])
    _close(g_w, want[1], terms[1], most, dtype)
    with torch.no_grad():  # the same without a graph
        assert torch.equal(expert_product(a, w, at), out)


@pytest.mark.parametrize("dtype", TYPES)
def test_product_strides_and_alignment(dtype):
    torch = require_gpu()
    from purin_amd import expert_product

    t = _types(torch)[dtype]
    offsets = np.array([0, 9, 9, 60])
    at = torch.as_tensor(offsets, dtype=torch.int32).cuda()
    wide = _randn(torch, 1, (64, 150), t)
    big = _randn(torch, 2, (3, 150, 140), t, 0.1)
    for a, z in ((0, 128), (1, 129), (3, 100)):
        rows = wide[:, a:z]
        for w in (big[:, a:z, :], big[:, a:z, 1:130], big[:, :, a:z].transpose(1, 2)[:, :, :],
                  big[1:2, a:z, :].expand(3, z - a, 140), big[:, a:z, ::2],
                  big[:, a:a + 1, ::3], big[:, a:z, 5:6], big[:, a:z:2, 5:6],
                  big[:, a:a + 1, 7:8], big.transpose(1, 2)[:, a:a + 1, ::2]):
            if w.shape[1] != z - a:
                w = w[:, :z - a, :]
            rows = wide[:, a:a + w.shape[1]]
            out = expert_product(rows, w, at)
            rn, wn = _np(rows), _np(w)
            _close(out, ot.product(rn, wn, offsets), ot.product(abs(rn), abs(wn), offsets),
                   w.shape[1], dtype)
    # one matrix for all experts: its gradient is the sum over them
    one = big[0, :128, :].clone().requires_grad_()
    rows = wide[:, :128].contiguous()
    out = expert_product(rows, one.expand(3, 128, 140), at)
    (g,) = torch.autograd.grad(out, one, torch.ones_like(out))
    want = _np(rows)[:60].T @ np.ones((60, 140))
    terms = abs(_np(rows)[:60]).T @ np.ones((60, 140))
    # three experts' gradients, each rounded, then summed and rounded
    assert (abs(_np(g) - want) <= 4 * UNIT[dtype] * terms + 124 * SUMS[dtype] * terms).all()
    # a gradient that is broadcast
    rows.requires_grad_()
    (g,) = torch.autograd.grad(expert_product(rows, big[:, :128], at).sum(), rows)
    wn = _np(big[:, :128]).sum(2)
    want = np.concatenate((np.repeat(wn[0:1], 9, 0), np.repeat(wn[2:3], 51, 0), np.zeros((4, 128))))
    terms = np.abs(_np(big[:, :128])).sum(2).max()
    _close(g, want, np.full(want.shape, terms), 140, dtype)


def test_product_of_empty_sizes():
    torch = require_gpu()
    from purin_amd import expert_product

    for t in _types(torch).values():
        for rows, inner, outer in ((0, 8, 8), (4, 0, 8), (4, 8, 0)):
            a = torch.ones((rows, inner), dtype=t, device="cuda", requires_grad=True)
            w = torch.ones((2, inner, outer), dtype=t, device="cuda", requires_grad=True)
            at = torch.tensor([0, rows // 2, rows], dtype=torch.int32, device="cuda")
            out = expert_product(a, w, at)
            assert out.shape == (rows, outer) and (out == 0).all()
            g_a, g_w = torch.autograd.grad(out, (a, w), torch.ones_like(out))
            assert (g_a == 0).all() and (g_w == 0).all()


def test_offsets_out_of_range_stay_inside():
    """Offsets past the rows are read as the rows' end (nothing outside is read or written)."""
    torch = require_gpu()
    from purin_amd import expert_product

    a = _randn(torch, 1, (10, 16), torch.float32)
    w = _randn(torch, 2, (2, 16, 8), torch.float32)
    at = torch.tensor([0, 4, 1 << 30], dtype=torch.int32, device="cuda")
    got = expert_product(a, w, at)
    want = expert_product(a, w, torch.tensor([0, 4, 10], dtype=torch.int32, device="cuda"))
    assert torch.equal(got, want)


# ---------------------------------------------------------------------------
# the global norm
# ---------------------------------------------------------------------------

SIZES = [(1,), (7,), (3, 0, 5), (65, 1, 4096, 3), (16384, 16385, 1), (100_003,),
         tuple(range(1, 131)), (5, 300_000) + (11,) * 200]


def _norm_close(norm, want, sizes):
    # squares and their sum in 64 bits, rounded once
    u = 2.0 ** -24 if norm.element_size() == 4 else 2.0 ** -50
    assert abs(float(norm) - want) <= 1.01 * u * want


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("dtype", TYPES + ["mixed"])
def test_clip(sizes, dtype):
    torch = require_gpu()
    from purin_amd import clip_gradients, gradient_norm

    print(f"clip {sizes[:5]} {dtype}", flush=True)
    names = [TYPES[i % 4] if dtype == "mixed" else dtype for i in range(len(sizes))]
    g = [_randn(torch, i, (n,), _types(torch)[d], 0.1 + i % 3)
         for i, (n, d) in enumerate(zip(sizes, names))]
    plain = [_np(x) for x in g]
    want, _ = ot.clip(plain, 0.0)
    norm = gradient_norm(g)
    assert norm.dtype == (torch.float64 if "f64" in names else torch.float32) and norm.ndim == 0
    _norm_close(norm, want, sizes)
    for largest in (want / 3, want * 2, 0.0):
        out = [torch.full_like(x, 9.0) for x in g]
        here = [x.clone() for x in g]
        assert torch.equal(clip_gradients(g, largest, out=out), norm)
        assert torch.equal(clip_gradients(here, largest), norm)
        _, scaled = ot.clip(plain, largest)
        for o, h, x, s, d in zip(out, here, g, scaled, names):
            assert torch.equal(o, h)
            if largest > want:
                assert torch.equal(o, x)
            # the factor and the product rounded in the sums' type, then once more
            _close(o, s, np.abs(s), 0, d)
        assert all(np.array_equal(_np(x), p) for x, p in zip(g, plain))


def test_clip_extremes():
    torch = require_gpu()
    from purin_amd import clip_gradients, gradient_norm

    assert float(gradient_norm([])) == 0.0
    assert float(clip_gradients([], 1.0)) == 0.0
    z = [torch.zeros(5, device="cuda"), None, torch.zeros(0, device="cuda")]
    assert float(clip_gradients(z, 0.0)) == 0.0
    # squares beyond the 32-bit range on both sides
    g = [torch.full((1000,), 1e30, device="cuda"), torch.full((3,), 1e-30, device="cuda")]
    assert abs(float(clip_gradients(g, 1.0)) / (1e30 * 1000 ** 0.5) - 1) < 1e-6
    assert abs(float(g[0].double().norm()) - 1) < 1e-6
    g = [torch.full((4,), 1e-30, device="cuda")]
    assert abs(float(gradient_norm(g)) / 2e-30 - 1) < 1e-6
    # a factor below the 32-bit numbers' normal range
    g = [torch.full((4,), 2.0 ** 120, device="cuda")]
    clip_gradients(g, 2.0 ** -20)
    assert float(g[0][0]) == 2.0 ** -21
    g = [torch.full((1,), 2.0 ** 127, device="cuda"), torch.full((1,), 1.0, device="cuda")]
    clip_gradients(g, 2.0 ** -10)
    assert float(g[0][0]) == 2.0 ** -10 and float(g[1][0]) == 2.0 ** -137
    # what is not finite shows
    nan = float("nan")
    g = [torch.tensor([1.0, nan], device="cuda"), torch.ones(3, device="cuda")]
    assert torch.isnan(clip_gradients(g, 1.0)) and all(torch.isnan(x).all() for x in g)
    g = [torch.tensor([1.0, float("inf")], device="cuda"), torch.ones(3, device="cuda")]
    assert torch.isinf(clip_gradients(g, 1.0))
    assert (g[1] == 0).all() and g[0][0] == 0 and torch.isnan(g[0][1])


def test_clip_strides():
    torch = require_gpu()
    from purin_amd import clip_gradients, gradient_norm

    base = _randn(torch, 1, (40, 33), torch.float32)
    views = {"transposed": lambda b: b.t(), "column": lambda b: b[:, 3],
             "odd start": lambda b: b.view(-1)[1:1001], "steps": lambda b: b[::2, ::3]}
    for name, view in views.items():
        b = base.clone()
        g = view(b)
        want, scaled = ot.clip([_np(g)], 0.5)
        _norm_close(gradient_norm([g]), want, None)
        out = view(torch.zeros_like(b))
        clip_gradients([g], 0.5, out=[out])
        assert torch.equal(b, base), name
        _close(out, scaled[0], np.abs(scaled[0]), 0, "f32")
        other = torch.zeros(g.shape, device="cuda")
        clip_gradients([g], 0.5, out=[other])
        assert torch.equal(other, out) and torch.equal(b, base)
        clip_gradients([g], 0.5)
        assert torch.equal(g, out), name
        mask = view(torch.ones_like(b, dtype=torch.bool).zero_())
        touched = torch.zeros_like(b, dtype=torch.bool)
        view(touched).fill_(True)
        assert torch.equal(b[~touched], base[~touched]) and mask.shape == g.shape
    # a broadcast gradient has a norm, and cannot be scaled in place
    g = base[:1].expand(5, 33)
    _norm_close(gradient_norm([g]), ot.clip([_np(g)], 0.0)[0], None)
    with pytest.raises(ValueError):
        clip_gradients([g], 0.5)


def test_clip_counts_as_a_change_for_autograd():
    torch = require_gpu()
    from purin_amd import clip_gradients

    x = torch.ones(4, device="cuda", requires_grad=True)
    saved = torch.full((4,), 3.0, device="cuda")
    y = (x * saved).sum()
    clip_gradients([saved], 1.0)
    with pytest.raises(RuntimeError):
        y.backward()


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------


def test_results_repeat_bit_for_bit():
    torch = require_gpu()
    from purin_amd import clip_gradients, combine, dispatch, expert_product, route

    w = torch.softmax(_randn(torch, 1, (3000, 40), torch.float32), 1).requires_grad_()
    x = _randn(torch, 2, (3000, 136), torch.bfloat16).requires_grad_()
    m = _randn(torch, 3, (40, 136, 72), torch.bfloat16, 0.1).requires_grad_()
    cot = _randn(torch, 4, (3000, 72), torch.bfloat16)

    def once():
        r = route(w, 4)
        out = combine(expert_product(dispatch(x, r), m, r), r)
        g = list(torch.autograd.grad(out, (w, x, m), cot))
        norm = clip_gradients(g, 1.0)
        return [r.experts, r.place, r.source, r.offsets, out, norm, *g]

    first = once()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


def test_another_stream_and_a_workspace_of_the_callers():
    torch = require_gpu()
    from purin_amd import clip_gradients, combine, dispatch, expert_product, route, route_experts
    from purin_amd.gradients import clip_workspace_bytes
    from purin_amd.routing import route_workspace_bytes

    w = torch.softmax(_randn(torch, 1, (4000, 20), torch.float32), 1)
    x = _randn(torch, 2, (4000, 64), torch.float32)
    m = _randn(torch, 3, (20, 64, 48), torch.float32)

    def once(**kw):
        r = route(w, 3, **kw)
        out = combine(expert_product(dispatch(x, r), m, r), r)
        g = [out.clone(), x.clone()]
        norm = clip_gradients(g, 1.0)
        return [r.place, r.offsets, out, norm, *g]

    want = once()
    torch.cuda.synchronize()
    need = route_workspace_bytes(4000, 20, 3)
    assert need > 0
    got = once(workspace=torch.empty(need, dtype=torch.uint8, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = once()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    with pytest.raises(Exception, match="workspace"):
        route(w, 3, workspace=torch.empty(need - 4, dtype=torch.uint8, device="cuda"))
    ids = torch.zeros((4000, 3), dtype=torch.int32, device="cuda")
    route_experts(ids, 20, workspace=torch.empty(need, dtype=torch.uint8, device="cuda"))
    need = clip_workspace_bytes(1)
    norm = clip_gradients([x.clone()], 1.0, workspace=torch.empty(need, dtype=torch.uint8,
                                                                  device="cuda"))
    assert torch.equal(norm, clip_gradients([x.clone()], 1.0))


def test_a_captured_step_replays():
    """All calls in one graph; replays on new inputs, with eager work between, give the eager
    results."""
    torch = require_gpu()
    from purin_amd import clip_gradients, combine, dispatch, expert_product, route

    w = torch.softmax(_randn(torch, 1, (3000, 24), torch.float32), 1)
    x = _randn(torch, 2, (3000, 64), torch.bfloat16)
    m = _randn(torch, 3, (24, 64, 64), torch.bfloat16, 0.1)
    g = [_randn(torch, 4, (5000,), torch.float32), _randn(torch, 5, (77,), torch.float32)]
    out_g = [torch.empty_like(t) for t in g]

    def once():
        r = route(w, 3)
        out = combine(expert_product(dispatch(x, r), m, r), r)
        return out, r.place, clip_gradients(g, 1.0, out=out_g)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    for k in range(4):
        w.copy_(torch.softmax(_randn(torch, 10 + k, (3000, 24), torch.float32), 1))
        x.copy_(_randn(torch, 20 + k, (3000, 64), torch.bfloat16))
        g[0].copy_(_randn(torch, 30 + k, (5000,), torch.float32))
        want = [t.clone() for t in once()] + [t.clone() for t in out_g]
        torch.cuda.synchronize()
        for t in out_g:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [*held, *out_g]
        assert all(torch.equal(a, b) for a, b in zip(want, got)), k


def test_refusals():
    torch = require_gpu()
    from purin_amd import (Routing, clip_gradients, combine, dispatch, expert_product,
                           gradient_norm, route, route_experts)
    from purin_amd._lib import PurinError

    w = torch.rand((6, 4), device="cuda")
    x = torch.rand((6, 8), device="cuda")
    r = route(w, 2)
    assert isinstance(r, Routing)
    y = dispatch(x, r)
    m = torch.rand((4, 8, 8), device="cuda")
    at = r.offsets
    bad = [
        lambda: route(w, 0), lambda: route(w, 5), lambda: route(w, 2.0), lambda: route(w, True),
        lambda: route(w[0], 1), lambda: route(w.int(), 1), lambda: route(w.cpu(), 1),
        lambda: route([[1.0]], 1), lambda: route(w, 2, workspace=5),
        lambda: route_experts(w, 4), lambda: route_experts(r.experts, 0),
        lambda: route_experts(r.experts[0], 4), lambda: route_experts(r.experts.cpu(), 4),
        lambda: route_experts(r.experts, 4, weights=w),
        lambda: dispatch(x[:5], r), lambda: dispatch(x[0], r), lambda: dispatch(x.int(), r),
        lambda: dispatch(x.cpu(), r), lambda: dispatch(x, None),
        lambda: combine(x, r), lambda: combine(y, r, w), lambda: combine(y, r.place),
        lambda: combine(y, route_experts(r.experts, 4)),
        lambda: combine(y, r, r.weights.int()),
        lambda: expert_product(y, m.double(), at), lambda: expert_product(y, m[0], at),
        lambda: expert_product(y[:, :7], m, at), lambda: expert_product(y, m, at[:-1]),
        lambda: expert_product(y, m, at.long()), lambda: expert_product(y, m, [0, 1, 2, 3, 12]),
        lambda: expert_product(y, m, at.cpu()), lambda: expert_product(y.cpu(), m, at),
        lambda: clip_gradients([x], -1.0), lambda: clip_gradients([x], float("nan")),
        lambda: clip_gradients([x.int()], 1.0), lambda: clip_gradients([x.cpu()], 1.0),
        lambda: clip_gradients([x], 1.0, out=[]), lambda: clip_gradients([x], 1.0, out=[y]),
        lambda: clip_gradients([x], 1.0, out=[x.double()]),
        lambda: clip_gradients([x], 1.0, out=[None]), lambda: gradient_norm([x.to_sparse()]),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print("not refused:", i)
    for f in (lambda: route(torch.rand((2, 1025), device="cuda"), 2),
              lambda: clip_gradients([x, x], 1.0), lambda: clip_gradients([x, x[1:3]], 1.0),
              lambda: clip_gradients([x, w], 1.0, out=[y[:6], y[2:5].view(-1)[:24].view(6, 4)])):
        with pytest.raises(PurinError):
            f()
    # gradients of gradients are not there, and say so
    w.requires_grad_()
    (g,) = torch.autograd.grad(route(w, 2).weights.square().sum(), w, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), w)


# ---------------------------------------------------------------------------
# the products at sizes that take every cut of the kernels
# ---------------------------------------------------------------------------

# rows, experts, inner, outer: 16-bit products of 32 x 64 tiles with and without splits, 128 x 128
# with four and with two stages, 256 x 256; weights' gradients split, 128 x 128 of both kinds and
# 256 x 256; 32-bit ones of 32, 64 and 128 rows, split and whole; and the same off 16-byte rows
LARGE = [(700, 4, 2048, 256), (1203, 3, 3000, 101), (2048, 2, 512, 1024), (2049, 2, 515, 1027),
         (4096, 3, 256, 2048), (4100, 3, 259, 2051), (16400, 4, 72, 4104), (16401, 4, 77, 4099),
         (9000, 2, 128, 136), (20000, 3, 200, 137), (1500, 16, 2048, 2056), (1400, 17, 2051, 2050),
         (6000, 1, 64, 64), (30000, 100, 67, 70)]


def _counts(rows, experts, seed):
    """Unequal shares with an expert that has none (of three or more), and rows left over."""
    rng = np.random.default_rng(seed)
    share = rng.uniform(0.5, 1.5, experts)
    if experts > 2:
        share[1] = 0.0
    return np.floor(share / share.sum() * rows * 0.97).astype(int)


@pytest.mark.parametrize("rows,experts,inner,outer", LARGE)
@pytest.mark.parametrize("order", ["io", "oi"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_large_products(rows, experts, inner, outer, order, dtype):
    torch = require_gpu()
    from purin_amd import expert_product

    print(f"large product {rows} {experts} {inner} {outer} {order} {dtype}", flush=True)
    t = _types(torch)[dtype]
    counts = _counts(rows, experts, rows)
    offsets = np.concatenate(([0], np.cumsum(counts)))
    g = torch.Generator(device="cuda").manual_seed(rows)
    make = lambda *shape: torch.randn(shape, generator=g, device="cuda").to(t)
    a = make(rows, inner).requires_grad_()
    w = make(experts, inner, outer) if order == "io" else make(experts, outer, inner).transpose(1, 2)
    w.requires_grad_()
    cot = make(rows, outer)
    out = expert_product(a, w, torch.as_tensor(offsets, dtype=torch.int32).cuda())
    g_a, g_w = torch.autograd.grad(out, (a, w), cot)
    u, s = UNIT[dtype], SUMS[dtype]

    def check(got, x, y, what):  # got against x @ y in 64 bits
        x, y = x.double(), y.double()
        want, terms = x @ y, x.abs() @ y.abs()
        bound = u * want.abs() + 2 * (x.shape[1] + 2) * s * terms * (1 + u) + STEP[dtype]
        bad = ~((got.double() - want).abs() <= bound)
        assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[:3].tolist())

    a, w = a.detach(), w.detach()
    for e in range(experts):
        i, j = int(offsets[e]), int(offsets[e + 1])
        if i < j:
            check(out[i:j], a[i:j], w[e], ("out", e))
            check(g_a[i:j], cot[i:j], w[e].T, ("rows", e))
            check(g_w[e], a[i:j].T, cot[i:j], ("weight", e))
        else:
            assert (g_w[e] == 0).all()
    last = int(offsets[-1])
    assert last < rows and (out[last:] == 0).all() and (g_a[last:] == 0).all()


def test_long_sums_in_32_bits():
    """A contraction of 40,000 in f32: the error against 64 bits stays what sums in blocks leave
    (kBlock32 = 64 in one run, 625 such runs), far below that of one running sum."""
    torch = require_gpu()
    from purin_amd import expert_product

    g = torch.Generator(device="cuda").manual_seed(4)
    a = torch.rand((64, 40000), generator=g, device="cuda")
    w = torch.rand((1, 40000, 64), generator=g, device="cuda")
    at = torch.tensor([0, 64], dtype=torch.int32, device="cuda")
    want = a.double() @ w[0].double()
    got = expert_product(a, w, at).double()
    # every partial sum is positive: 64 + 625 additions, half a unit each at most
    assert float(((got - want).abs() / want).max()) <= (64 + 625 + 4) * 2.0 ** -24


def test_gradients_against_differences():
    """All calls in f64 through torch's own check by differences."""
    torch = require_gpu()
    from purin_amd import combine, dispatch, expert_product, route

    w = _weights(torch, 3, 7, 5, "f64")
    r0 = route(w, 2)
    x = _randn(torch, 1, (7, 6), torch.float64).requires_grad_()
    m = _randn(torch, 2, (5, 6, 4), torch.float64).requires_grad_()
    # weights that keep their order under the differences' steps
    w = (w * 1.0 + torch.arange(5, device="cuda") * 1e-3 * (w > 0)).requires_grad_()
    assert torch.equal(route(w, 2).experts >= 0, r0.experts >= 0)

    def f(x, m, w):
        r = route(w, 2)
        return combine(expert_product(dispatch(x, r), m, r), r)

    # entries at zero have no difference to both sides: only the chosen weights are checked
    chosen = route(w.detach(), 2)
    c = chosen.weights.clone().requires_grad_()

    def h(x, m, c):
        return combine(expert_product(dispatch(x, chosen), m, chosen), chosen, c)

    assert torch.autograd.gradcheck(h, (x, m, c), eps=1e-6, atol=1e-7, rtol=0)
    out = f(x, m, w)
    cot = _randn(torch, 5, (7, 4), torch.float64)
    (g,) = torch.autograd.grad(out, w, cot)
    for t, e in [(0, int(chosen.experts[0, 0])), (3, int(chosen.experts[3, 0]))]:
        if e < 0:
            continue
        d = torch.zeros_like(w)
        d[t, e] = 1e-6
        with torch.no_grad():
            slope = ((f(x, m, w + d) - f(x, m, w - d)) * cot).sum() / 2e-6
        assert abs(float(slope - g[t, e])) <= 1e-7
