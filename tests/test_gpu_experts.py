"""Microscaled numbers, products with them, the activation and whole layers against the float64
oracle (``oracle/experts.py``, ``oracle/train.py``).

Packing rounds once after exact scalings: codes, scales and values are compared bit for bit.
Products: as in ``test_gpu_train`` (u |exact| + 2 (K + 2) a sum|terms|), with the values that the
packed operands stand for.  Elementary functions: an exponential, a reciprocal or a normal share
in the sums' type is within (8 + 4 |u| + 2 u^2) a of itself, of which |u| and u^2 come from its
rounded argument.  The layer keeps its hidden values as two numbers of the type, u^2 of them off
(and half of float16's smallest step, 2^-25).
"""

import numpy as np
import pytest

from oracle import experts as oe
from oracle import train as ot
from tests._gpu import require_gpu, to_np
from tests.test_gpu_train import STEP, SUMS, UNIT, _close, _np, _randn, _types, _weights

pytestmark = pytest.mark.gpu

HALF = ["bf16", "f16"]
PACKED = ["f32", "bf16", "f16"]


def _rows(torch, seed, shape, dtype):
    """Rows of different size, zeros and far elements among them."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g, dtype=torch.float64)
    x *= torch.exp2(torch.randint(-6, 6, (*shape[:-1], 1), generator=g).double())
    x[torch.rand(shape, generator=g) < 0.05] = 0.0
    x[torch.rand(shape, generator=g) < 0.02] *= 16
    return x.to(dtype).cuda()


# ---------------------------------------------------------------------------
# packing
# ---------------------------------------------------------------------------

SHAPES = [(1, 1), (3, 31), (5, 32), (4, 33), (2, 200), (70, 129), (9, 64)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", ["fp4", "int8"])
@pytest.mark.parametrize("dtype", PACKED)
def test_pack_and_unpack(shape, kind, dtype):
    torch = require_gpu()
    from purin_amd import pack, unpack

    print(f"pack {shape} {kind} {dtype}", flush=True)
    t = _types(torch)[dtype]
    x = _rows(torch, 1, shape, t)
    codes, scales = oe.pack(_np(x), kind)
    for given, axis in ((x, -1), (x, 1), (x.t().contiguous().t(), 1), (x.t(), 0),
                        (torch.cat((x, x), 1)[:, :shape[1]], 1), (x.t().contiguous(), 0)):
        m = pack(given, kind, axis)
        assert m.dtype == t and m.shape == tuple(given.shape)
        np.testing.assert_array_equal(to_np(m.codes), codes)
        np.testing.assert_array_equal(to_np(m.scales), scales)
        y = unpack(m)
        assert y.dtype == t and y.shape == given.shape
        want = oe.unpack(codes, scales, kind, shape[1])
        np.testing.assert_array_equal(_np(y), want if axis % 2 == 1 else want.T)
        # again: what few bits hold, they hold exactly
        again = pack(y, kind, axis)
        np.testing.assert_array_equal(_np(unpack(again)), _np(y))


@pytest.mark.parametrize("kind", ["fp4", "int8"])
@pytest.mark.parametrize("dtype", PACKED)
def test_pack_of_three_and_more_dimensions(kind, dtype):
    torch = require_gpu()
    from purin_amd import pack, unpack

    x = _rows(torch, 2, (3, 70, 101), _types(torch)[dtype])
    for given, axis in ((x, 2), (x, 1), (x, 0), (x.transpose(1, 2), 1), (x[:, 1:, 3:], 1),
                        (x[:, ::2], 2), (x[:, :, ::3], 1), (x[1:2], 1), (x[:, :1], 2), (x[:1, :1], 1),
                        (x.view(3, 7, 10, 101), 2), (x.view(3, 7, 10, 101), 3), (x[0, 0], 0),
                        (x[:1].expand(4, 70, 101), 2), (x[0, :, :1].expand(70, 40), 1)):
        m = pack(given, kind, axis)
        moved = np.moveaxis(_np(given), axis, -1)
        codes, scales = oe.pack(moved.reshape(-1, moved.shape[-1]), kind)
        np.testing.assert_array_equal(to_np(m.codes).reshape(codes.shape), codes)
        np.testing.assert_array_equal(to_np(m.scales).reshape(scales.shape), scales)
        want = oe.unpack(codes, scales, kind, moved.shape[-1]).reshape(moved.shape)
        np.testing.assert_array_equal(_np(unpack(m)), np.moveaxis(want, -1, axis))
    for shape in ((0, 8), (8, 0), (3, 0, 5), (0,)):
        m = pack(torch.zeros(shape, dtype=x.dtype, device="cuda"), kind)
        assert unpack(m).shape == shape


@pytest.mark.parametrize("kind", ["fp4", "int8"])
@pytest.mark.parametrize("dtype", PACKED)
def test_pack_of_odd_values(kind, dtype):
    """Borders between codes, the ends of the type's range, zeros, infinities and NaN."""
    torch = require_gpu()
    from purin_amd import pack, unpack

    t = _types(torch)[dtype]
    big, small = torch.finfo(t).max, torch.finfo(t).smallest_normal
    step = float(torch.nextafter(torch.zeros((), dtype=t), torch.ones((), dtype=t)))
    one = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.75, 0.0, -0.0, -0.25, -5.0]
    lines = [[4.0] + [v for v in one if abs(v) < 4], one, [big, -big, big / 2, 1.0],
             [small, step, -step, 3 * step, 0.0], [step] * 3, [step * 7, step * 5, step], [0.0] * 4,
             [1.0, float("inf")], [float("-inf")], [float("nan"), 2.0], [127 / 64, 1.0, 0.5 / 64, 1.5 / 64]]
    x = torch.zeros((len(lines), 40), dtype=t)
    for i, line in enumerate(lines):
        x[i, :len(line)] = torch.tensor(line, dtype=torch.float64).to(t)
        x[i, 35] = 1.0
    x = x.cuda()
    codes, scales = oe.pack(_np(x), kind)
    m = pack(x, kind)
    np.testing.assert_array_equal(to_np(m.codes), codes)
    np.testing.assert_array_equal(to_np(m.scales), scales)
    np.testing.assert_array_equal(_np(unpack(m)), oe.unpack(codes, scales, kind, 40))
    m = pack(x.t().contiguous(), kind, axis=0)
    np.testing.assert_array_equal(to_np(m.codes), codes)


def test_every_scale_unpacks():
    torch = require_gpu()
    from purin_amd import Microscaled, unpack

    for kind, width in (("fp4", 16), ("int8", 32)):
        codes = torch.arange(256, dtype=torch.uint8).view(-1, width).repeat(256, 1)
        scales = torch.zeros((codes.shape[0], 4), dtype=torch.uint8)
        scales[:, 0] = torch.arange(256).repeat_interleave(256 // width)
        m = Microscaled(codes.cuda(), scales.cuda(), kind, (codes.shape[0], 32), 1, torch.float32)
        want = oe.unpack(to_np(codes), to_np(scales), kind, 32)
        for t in (torch.float32, torch.bfloat16, torch.float16):
            got = unpack(m, t)
            assert torch.equal(torch.nan_to_num(got.cpu(), nan=77.0),
                               torch.nan_to_num(torch.as_tensor(want).to(t), nan=77.0)), (kind, t)


# ---------------------------------------------------------------------------
# products with packed operands
# ---------------------------------------------------------------------------

# rows to each expert (the last number: rows behind them), inner, outer
PRODUCTS = [((1, 0), 1, 1), ((0, 0, 0, 5), 8, 8), ((8, 0), 64, 64), ((1, 0, 2, 1, 0), 128, 96),
            ((3, 130, 0, 17, 2), 37, 53), ((128, 256, 64, 0), 64, 128), ((129, 1, 0, 300, 9), 200, 136),
            ((16,) * 12 + (0,), 256, 192), ((5,) * 70 + (3,), 33, 40), ((600, 40, 0), 136, 264),
            ((1,) * 3 + (0,), 2048, 72), ((2, 1, 4, 0), 72, 1408), ((40, 33, 70, 1), 1032, 2048),
            ((300, 260), 260, 4100), ((2,) * 40 + (0,), 64, 2600), ((1,) * 100 + (0,), 40, 2700)]


def _packed_weight(torch, seed, shape, dtype):
    from purin_amd import pack, unpack

    m = pack(_randn(torch, seed, shape, dtype, shape[1] ** -0.5), "fp4", axis=1)
    return m, _np(unpack(m))


@pytest.mark.parametrize("counts,inner,outer", PRODUCTS)
@pytest.mark.parametrize("dtype", PACKED)
def test_product_with_packed_weights(counts, inner, outer, dtype):
    torch = require_gpu()
    from purin_amd import expert_product

    print(f"packed product {counts[:6]} {inner} {outer} {dtype}", flush=True)
    t = _types(torch)[dtype]
    offsets = np.concatenate(([0], np.cumsum(counts[:-1])))
    rows, experts = int(offsets[-1]) + counts[-1], len(counts) - 1
    m, wn = _packed_weight(torch, 2, (experts, inner, outer), t)
    wide = _randn(torch, 1, (rows, inner + 3), t)
    at = torch.as_tensor(offsets, dtype=torch.int32).cuda()
    cot = _randn(torch, 3, (rows, outer), t)
    for a in (wide[:, :inner].contiguous(), wide[:, 1:1 + inner]):
        a = a.detach().requires_grad_()
        out = expert_product(a, m, at)
        (g_a,) = torch.autograd.grad(out, a, cot)
        an, cn = _np(a), _np(cot)
        assert out.dtype == t and g_a.dtype == t
        _close(out, ot.product(an, wn, offsets), ot.product(abs(an), abs(wn), offsets), inner, dtype)
        back = wn.transpose(0, 2, 1)
        _close(g_a, ot.product(cn, back, offsets), ot.product(abs(cn), abs(back), offsets), outer, dtype)
        with torch.no_grad():
            assert torch.equal(expert_product(a, m, at), out)


@pytest.mark.parametrize("counts,inner,outer", PRODUCTS)
@pytest.mark.parametrize("dtype", PACKED)
def test_product_with_both_packed(counts, inner, outer, dtype):
    torch = require_gpu()
    from purin_amd import expert_product, pack, unpack

    print(f"both packed {counts[:6]} {inner} {outer} {dtype}", flush=True)
    t = _types(torch)[dtype]
    offsets = np.concatenate(([0], np.cumsum(counts[:-1])))
    rows, experts = int(offsets[-1]) + counts[-1], len(counts) - 1
    m, wn = _packed_weight(torch, 2, (experts, inner, outer), torch.float32)
    a = pack(_rows(torch, 1, (rows, inner), t), "fp4")
    out = expert_product(a, m, torch.as_tensor(offsets, dtype=torch.int32).cuda())
    assert out.dtype == t
    an = _np(unpack(a))
    _close(out, ot.product(an, wn, offsets), ot.product(abs(an), abs(wn), offsets), inner, dtype)


@pytest.mark.parametrize("both", [False, True])
def test_packed_products_of_many_tiles(both):
    """Enough tiles for the largest ones; checked on the card in 64 bits."""
    torch = require_gpu()
    from purin_amd import expert_product, pack, unpack

    rows, inner, outer = 8200, 328, 8200
    m = pack(_randn(torch, 2, (2, inner, outer), torch.bfloat16, inner ** -0.5), "fp4", axis=1)
    a = _randn(torch, 1, (rows, inner), torch.bfloat16)
    at = torch.tensor([0, 4000, 8190], dtype=torch.int32, device="cuda")
    given = pack(a, "fp4") if both else a
    out = expert_product(given, m, at).double()
    an, wn = (unpack(given) if both else a).double(), unpack(m).double()
    for e, (i, j) in enumerate(((0, 4000), (4000, 8190))):
        want, terms = an[i:j] @ wn[e], an[i:j].abs() @ wn[e].abs()
        bound = UNIT["bf16"] * want.abs() + 2 * (inner + 2) * SUMS["bf16"] * terms + STEP["bf16"]
        assert bool(((out[i:j] - want).abs() <= bound).all())
    assert bool((out[8190:] == 0).all())


def test_packed_products_of_empty_sizes_and_masked_rows():
    torch = require_gpu()
    from purin_amd import expert_product, pack

    for t in (torch.bfloat16, torch.float16, torch.float32):
        for rows, inner, outer in ((0, 8, 8), (4, 0, 8), (4, 8, 0)):
            m = pack(torch.ones((2, inner, outer), dtype=t, device="cuda"), "fp4", axis=1)
            at = torch.tensor([0, rows // 2, rows], dtype=torch.int32, device="cuda")
            a = torch.ones((rows, inner), dtype=t, device="cuda", requires_grad=True)
            out = expert_product(a, m, at)
            assert out.shape == (rows, outer) and bool((out == 0).all())
            (g,) = torch.autograd.grad(out, a, torch.ones_like(out))
            assert g.shape == a.shape and bool((g == 0).all())
            out = expert_product(pack(a.detach(), "fp4"), m, at)
            assert out.shape == (rows, outer) and bool((out == 0).all())
        # rows that no expert has: NaN there changes nothing
        m = pack(_randn(torch, 1, (3, 70, 40), t), "fp4", axis=1)
        at = torch.tensor([0, 9, 9, 50], dtype=torch.int32, device="cuda")
        a = _randn(torch, 2, (60, 70), t)
        want = expert_product(a, m, at)
        a[50:] = float("nan")
        a.requires_grad_()
        out = expert_product(a, m, at)
        assert torch.equal(out, want) and bool((out[50:] == 0).all())
        cot = _randn(torch, 3, (60, 40), t)
        cot[50:] = float("nan")
        (g,) = torch.autograd.grad(out, a, cot)
        assert bool(torch.isfinite(g).all()) and bool((g[50:] == 0).all())
        both = expert_product(pack(a.detach(), "fp4"), m, at)
        assert bool(torch.isfinite(both).all()) and bool((both[50:] == 0).all())
        # a NaN in an expert's row shows there alone
        a = a.detach()
        a[3, 5] = float("nan")
        out = expert_product(a, m, at)
        assert bool(torch.isnan(out[3]).all()) and bool(torch.isfinite(out[:3]).all())
        assert bool(torch.isfinite(out[4:50]).all())
        out = expert_product(pack(a, "fp4"), m, at)
        assert bool(torch.isnan(out[3]).all()) and bool(torch.isfinite(out[4:50]).all())


def test_weights_beyond_the_rows_type():
    """float16 rows beside weights of a wider type: infinite above its range."""
    torch = require_gpu()
    from purin_amd import expert_product, pack

    w = torch.zeros((1, 64, 8), device="cuda")
    w[0, 0, 0], w[0, 0, 1], w[0, 32, 2] = 2.0 ** 17, 2.0 ** 15, 2.0 ** -30
    m = pack(w, "fp4", axis=1)
    at = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    out = expert_product(torch.ones((2, 64), dtype=torch.float16, device="cuda"), m, at)
    assert bool(torch.isinf(out[:, 0]).all()) and bool((out[:, 1] == 2.0 ** 15).all())
    assert bool((out[:, 2] == 0).all())
    out = expert_product(torch.ones((2, 64), dtype=torch.bfloat16, device="cuda"), m, at)
    assert out[0, 0] == 2.0 ** 17 and out[0, 2] == 2.0 ** -30


# ---------------------------------------------------------------------------
# rows kept in 8 bits
# ---------------------------------------------------------------------------

KEPT = [((3, 130, 0, 17, 2), 37, 53), ((129, 1, 0, 300, 9), 200, 136), ((1, 0), 1, 1),
        ((16,) * 12 + (0,), 256, 192), ((1, 0, 2, 1, 0), 128, 96)]


@pytest.mark.parametrize("counts,inner,outer", KEPT)
@pytest.mark.parametrize("order", ["io", "oi"])
@pytest.mark.parametrize("dtype", PACKED)
def test_product_with_kept_rows(counts, inner, outer, order, dtype):
    torch = require_gpu()
    from purin_amd import expert_product

    print(f"kept {counts[:6]} {inner} {outer} {order} {dtype}", flush=True)
    t = _types(torch)[dtype]
    offsets = np.concatenate(([0], np.cumsum(counts[:-1])))
    rows, experts = int(offsets[-1]) + counts[-1], len(counts) - 1
    a = _rows(torch, 1, (rows, inner), t).requires_grad_()
    w = _randn(torch, 2, (experts, inner, outer), t, inner ** -0.5)
    w = (w if order == "io" else w.transpose(1, 2).contiguous().transpose(1, 2)).requires_grad_()
    cot = _randn(torch, 3, (rows, outer), t)
    at = torch.as_tensor(offsets, dtype=torch.int32).cuda()
    plain = expert_product(a, w, at)
    g_plain, _ = torch.autograd.grad(plain, (a, w), cot)
    out = expert_product(a, w, at, saved="int8")
    g_a, g_w = torch.autograd.grad(out, (a, w), cot)
    assert torch.equal(out, plain) and torch.equal(g_a, g_plain) and g_w.stride() == w.stride()
    kept, cn = oe.values(_np(a), "int8"), _np(cot)
    want, terms = (ot.product_vjp(c, x, _np(w), offsets)[1] for c, x in
                   ((cn, kept), (abs(cn), abs(kept))))
    _close(g_w, want, terms, max(counts[:-1]), dtype)
    # only one of the two wants a gradient
    (g_only,) = torch.autograd.grad(expert_product(a.detach(), w, at, saved="int8"), w, cot)
    assert torch.equal(g_only, g_w)
    (g_only,) = torch.autograd.grad(expert_product(a, w.detach(), at, saved="int8"), a, cot)
    assert torch.equal(g_only, g_a)


def test_kept_rows_take_half_the_memory():
    torch = require_gpu()
    from purin_amd import activate, expert_product

    at = torch.tensor([0, 4096], dtype=torch.int32, device="cuda")
    w = _randn(torch, 1, (1, 1024, 64), torch.bfloat16).requires_grad_()

    def held(call, make):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = call(make())
        return torch.cuda.memory_allocated() - before - out.numel() * out.element_size()

    rows = lambda: _randn(torch, 2, (4096, 1024), torch.bfloat16)  # noqa: E731
    full = 4096 * 1024 * 2
    assert held(lambda r: expert_product(r, w, at), rows) >= full
    assert held(lambda r: expert_product(r, w, at, saved="int8"), rows) < 0.53 * full
    grad = lambda: rows().requires_grad_()  # noqa: E731
    assert held(lambda r: activate(r * 1, "silu"), grad) >= full
    # the input of r * 1 is not held by its graph, and activate keeps 8 bits of the result
    assert held(lambda r: activate(r * 1, "silu", saved="int8"), rows) == 0


def test_a_graph_holds_packed_weights_packed():
    torch = require_gpu()
    from purin_amd import expert_product, pack

    at = torch.tensor([0, 16], dtype=torch.int32, device="cuda")
    m = pack(_randn(torch, 1, (1, 1024, 2048), torch.bfloat16), "fp4", axis=1)
    for t in (torch.float32, torch.bfloat16):
        rows = _randn(torch, 2, (16, 1024), t).requires_grad_()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = expert_product(rows, m, at)
        # the result, and what else an allocation rounds up
        assert torch.cuda.memory_allocated() - before <= out.numel() * out.element_size() + 4096


# ---------------------------------------------------------------------------
# the activation
# ---------------------------------------------------------------------------


def _terms(u, kind):
    """Magnitudes of the terms of f and of its slope, and the elementary functions' error in a."""
    u = np.asarray(u)
    if kind == "relu":
        return np.abs(u), np.ones_like(u), 1.0
    with np.errstate(over="ignore"):
        s = 1 / (1 + np.exp(-u)) if kind == "silu" else oe.activation(np.where(u == 0, 1, u), "gelu")[0] / np.where(u == 0, 1, u)
        s = np.where((u == 0) & (kind == "gelu"), 0.5, s)
        rest = s * (1 - s) if kind == "silu" else 0.4 * np.exp(-u * u / 2)
    return np.abs(u) * s, s + np.abs(u) * rest, 8 + 4 * np.abs(u) + 2 * u * u


@pytest.mark.parametrize("rows,hidden", [(1, 1), (3, 8), (5, 33), (64, 96), (70, 131), (2, 1408)])
@pytest.mark.parametrize("kind", ["relu", "silu", "gelu"])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("dtype", ["f32", "f64", "bf16", "f16"])
def test_activate_and_gradient(rows, hidden, kind, gated, dtype):
    torch = require_gpu()
    from purin_amd import activate

    print(f"activate {rows} {hidden} {kind} {gated} {dtype}", flush=True)
    t = _types(torch)[dtype]
    columns = 2 * hidden if gated else hidden
    wide = _randn(torch, 1, (rows, columns + 5), t, 2.0)
    cot = _randn(torch, 2, (rows, hidden), t)
    for u in (wide[:, :columns].contiguous(), wide[:, 3:3 + columns]):
        for saved in (None, "int8"):
            if saved and dtype == "f64":
                continue
            u = u.detach().requires_grad_()
            out = activate(u, kind, gated=gated, saved=saved)
            (g,) = torch.autograd.grad(out, u, cot)
            assert out.dtype == t and g.dtype == t and g.shape == u.shape
            with torch.no_grad():
                assert torch.equal(activate(u, kind, gated=gated, saved=saved), out)
            a, un, cn = SUMS[dtype], _np(u), _np(cot)
            gate, value = un[:, :hidden], un[:, hidden:] if gated else np.ones_like(un)
            f, _, off = _terms(gate, kind)
            want = oe.activate(un, kind, gated)
            # the oracle's own share, 1 + erf, is off by 2^-52
            bound = (UNIT[dtype] * np.abs(want) + (a * off + 2 * a) * f * np.abs(value)
                     + 2.0 ** -50 * np.abs(gate * value) + STEP[dtype])
            assert (np.abs(_np(out) - want) <= bound).all()
            if saved:
                if gated:
                    gate, value = oe.values(gate, "int8"), oe.values(value, "int8")
                    un = np.concatenate((gate, value), 1)
                else:
                    gate = un = oe.values(un, "int8")
            f, slope, off = _terms(gate, kind)
            want = oe.activate_vjp(un, cn, kind, gated)
            size = np.concatenate((slope * np.abs(value), f), 1) if gated else slope
            off = np.concatenate((off, off), 1) if gated and kind != "relu" else off
            size = size * (np.concatenate((np.abs(cn), np.abs(cn)), 1) if gated else np.abs(cn))
            bound = (UNIT[dtype] * np.abs(want) + (a * off + 4 * a) * size + 2.0 ** -50 * size
                     + 2.0 ** -50 * np.abs(np.tile(cn * gate, (1, 2)) if gated else cn) + STEP[dtype])
            assert (np.abs(_np(g) - want) <= bound).all()


@pytest.mark.parametrize("hidden", [1, 32, 33, 70, 128, 161])
@pytest.mark.parametrize("gated", [True, False])
def test_kept_codes_are_packs(hidden, gated):
    """The codes and scales that activate makes on its way, the zeros behind them included."""
    torch = require_gpu()
    from purin_amd import _lib, pack

    halves = 2 if gated else 1
    u = _randn(torch, 1, (5, halves * hidden), torch.bfloat16)
    want = pack(u.view(5, halves, hidden), "int8")
    codes, scales = torch.full_like(want.codes, 77), torch.full_like(want.scales, 77)
    out = torch.empty((5, hidden), dtype=torch.bfloat16, device="cuda")
    _lib.check(_lib.load().purin_train_activate(
        torch.cuda.current_stream().cuda_stream, _lib.BF16, _lib.SILU, int(gated), 5, hidden,
        u.data_ptr(), halves * hidden, out.data_ptr(), codes.data_ptr(), scales.data_ptr()))
    assert torch.equal(codes, want.codes) and torch.equal(scales, want.scales)


@pytest.mark.parametrize("kind", ["relu", "silu", "gelu"])
@pytest.mark.parametrize("gated", [True, False])
def test_activation_gradient_by_differences(kind, gated):
    torch = require_gpu()
    from purin_amd import activate

    u = _randn(torch, 1, (3, 10), torch.float64).requires_grad_()
    cot = _randn(torch, 2, (3, 5 if gated else 10), torch.float64)
    (g,) = torch.autograd.grad(activate(u, kind, gated=gated), u, cot)
    for i in np.ndindex(3, 10):
        d = torch.zeros_like(u)
        d[i] = 1e-5
        with torch.no_grad():
            up, down = activate(u + d, kind, gated=gated), activate(u - d, kind, gated=gated)
        # the third derivative is below 2, and so is what the squares of 1e-5 leave
        assert abs(float(((up - down) * cot).sum()) / 2e-5 - float(g[i])) < 1e-8


def test_activation_of_far_values():
    """Ends of the range: no NaN where the formula has a limit."""
    torch = require_gpu()
    from purin_amd import activate

    for t in _types(torch).values():
        big = torch.finfo(t).max
        for kind in ("relu", "silu", "gelu"):
            u = torch.tensor([[big, -big, 200.0, -200.0, 0.0, -0.0, 1e-4]], dtype=t, device="cuda",
                             requires_grad=True)
            out = activate(u, kind, gated=False)
            (g,) = torch.autograd.grad(out, u, torch.ones_like(out))
            # 200 exp(-200) = 2.8e-85, which float64 has and the other types round to zero
            none = 3e-85 if t == torch.float64 else 0.0
            assert out[0, 0] == big and out[0, 1] == 0 and out[0, 2] == 200
            assert g[0, 0] == 1 and g[0, 1] == 0
            assert abs(float(out.detach()[0, 3])) <= none and abs(float(g[0, 3])) <= none
            assert float(g[0, 4]) == (0.0 if kind == "relu" else 0.5)
            nan = torch.full((1, 3), float("nan"), dtype=t, device="cuda")
            assert bool(torch.isnan(activate(nan, kind, gated=False)).all())
    for shape in ((0, 8), (4, 0)):
        u = torch.zeros(shape, device="cuda", requires_grad=True)
        out = activate(u)
        (g,) = torch.autograd.grad(out, u, torch.ones_like(out))
        assert out.shape == (shape[0], shape[1] // 2) and g.shape == shape


# ---------------------------------------------------------------------------
# the layer
# ---------------------------------------------------------------------------

# tokens, experts, slots, width, hidden, outer width
LAYERS = [(1, 1, 1, 1, 1, 1), (1, 8, 3, 64, 32, 64), (3, 5, 5, 37, 19, 53), (1, 70, 6, 264, 72, 136),
          (17, 9, 2, 128, 40, 72), (33, 6, 3, 96, 64, 200), (64, 4, 2, 72, 136, 64),
          (64, 300, 8, 40, 24, 33), (40, 40, 3, 520, 200, 65), (2, 1024, 9, 33, 8, 16),
          # on both sides of where a launch of its own chooses
          (16, 256, 8, 64, 32, 64), (16, 257, 8, 64, 32, 64), (17, 20, 3, 64, 32, 64),
          (13, 40, 10, 64, 40, 72),
          # the most pairs; more rows to an expert than a tile has; wide ones, which share less
          (64, 16, 16, 64, 32, 40), (64, 2, 2, 256, 96, 128), (24, 64, 4, 72, 48, 4104),
          (24, 64, 4, 40, 1560, 24)]


def _layer_weights(torch, packed, order, gated, shape, t):
    """(given, values) of both matrices."""
    from purin_amd import pack, unpack

    _, experts, _, width, hidden, outer = shape
    given, values = [], []
    for seed, size in ((2, (experts, width, 2 * hidden if gated else hidden)),
                       (3, (experts, hidden, outer))):
        w = _randn(torch, seed, size, t, size[1] ** -0.5)
        if packed:
            m = pack(w, "fp4", axis=1)
            given.append(m)
            values.append(_np(unpack(m)))
        else:
            given.append(w if order == "io" else w.transpose(1, 2).contiguous().transpose(1, 2))
            values.append(_np(w))
    return given, values


def _layer_close(torch, out, x, w, slots, values, kind, dtype):
    xn, wn = _np(x), _np(w)
    want, terms = oe.layer(xn, wn, slots, *values, kind)
    u, a = UNIT[dtype], SUMS[dtype]
    off = 2 * (xn.shape[1] + values[1].shape[1] + 4) * a + 2 * u * u + 128 * a
    floor = STEP[dtype]
    if dtype == "f16":
        ids, _ = ot.choose(wn, slots)
        size = np.abs(values[1]).sum(1)
        floor = floor + 2.0 ** -25 * np.array([size[i[i >= 0]].sum(0) for i in ids])
    got = _np(out)
    assert got.shape == want.shape
    bad = ~(np.abs(got - want) <= u * np.abs(want) + off * terms + floor)
    assert not bad.any(), (np.argwhere(bad)[:3], got[bad][:3], want[bad][:3])


@pytest.mark.parametrize("shape", LAYERS)
@pytest.mark.parametrize("weights", ["io", "oi", "packed"])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("dtype", HALF)
def test_layer(shape, weights, gated, dtype):
    torch = require_gpu()
    from purin_amd import expert_layer

    print(f"layer {shape} {weights} {gated} {dtype}", flush=True)
    tokens, experts, slots, width, hidden, outer = shape
    t = _types(torch)[dtype]
    kind = {1: "relu", 2: "silu", 0: "gelu"}[(tokens + width) % 3]
    given, values = _layer_weights(torch, weights == "packed", weights, gated, shape, t)
    w = _weights(torch, 5, tokens, experts, "f32", share=max(0.4, 3 / experts))
    wide = _randn(torch, 1, (tokens, width + 3), t)
    for x in (wide[:, :width].contiguous(), wide[:, 3:]):
        out = expert_layer(x, w, slots, *given, kind)
        assert out.dtype == t and out.shape == (tokens, outer)
        _layer_close(torch, out, x, w, slots, values, kind, dtype)
        assert torch.equal(expert_layer(x, w, slots, *given, kind), out)


@pytest.mark.parametrize("wdtype", ["f32", "f64", "bf16", "f16"])
@pytest.mark.parametrize("packed", [False, True])
def test_layer_weights_of_any_type_ties_and_empty_tokens(wdtype, packed):
    torch = require_gpu()
    from purin_amd import expert_layer

    shape = (12, 20, 4, 64, 32, 40)
    given, values = _layer_weights(torch, packed, "oi", True, shape, torch.bfloat16)
    w = _weights(torch, 7, 12, 20, wdtype)
    w[5] = 0.0
    w[6] = -1.0
    w[7, :] = 0.125
    x = _randn(torch, 1, (12, 64), torch.bfloat16)
    x[5] = float("nan")  # a token without experts
    for given_w in (w, torch.cat((w, w), 1)[:, :20], w.t().contiguous().t()):
        out = expert_layer(x, given_w, 4, *given, "silu")
        assert bool((out[5:7] == 0).all())
        safe = torch.nan_to_num(x)
        _layer_close(torch, out, safe, w, 4, values, "silu", "bf16")
    # what is not finite shows in its own token alone
    x[3, 2] = float("inf")
    w[4, 0] = float("nan")
    out = expert_layer(x, w, 4, *given, "silu")
    assert not bool(torch.isfinite(out[3]).any()) and bool(torch.isnan(out[4]).all())
    rest = [0, 1, 2, 5, 6, 7, 8, 9, 10, 11]
    assert bool(torch.isfinite(out[rest]).all())
    none = expert_layer(x, w * 0 - 1, 4, *given, "silu")
    assert bool((none[[0, 1, 2]] == 0).all())


def test_layer_strides_of_the_weights():
    torch = require_gpu()
    from purin_amd import expert_layer

    x = _randn(torch, 1, (9, 40), torch.float16)
    w = _weights(torch, 2, 9, 3, "f32")
    big = _randn(torch, 3, (3, 90, 100), torch.float16, 0.1)
    small = _randn(torch, 4, (3, 70, 90), torch.float16, 0.1)
    for inner in (big[:, :40, :64], big[:, 1:41, 3:67], big.transpose(1, 2)[:, 8:48, 9:73],
                  big[:, :40, :64].contiguous(), big[:1, :40, :64].expand(3, 40, 64),
                  big[:, ::2][:, :40, :64], big[:, :40, ::1][:, :, 31:95]):
        for outer in (small[:, :32, :50], small[:, 1:33, 1:52], small.transpose(1, 2)[:, :32, :50],
                      small[:, :32, ::2], small[:, :32, :1]):
            out = expert_layer(x, w, 2, inner, outer, "gelu")
            _layer_close(torch, out, x, w, 2, [_np(inner), _np(outer)], "gelu", "f16")


def test_layer_of_empty_sizes():
    torch = require_gpu()
    from purin_amd import expert_layer

    for tokens, width, hidden, outer in ((0, 8, 8, 8), (3, 0, 8, 8), (3, 8, 0, 8), (3, 8, 8, 0)):
        x = torch.ones((tokens, width), dtype=torch.bfloat16, device="cuda")
        a = torch.ones((4, width, 2 * hidden), dtype=torch.bfloat16, device="cuda")
        b = torch.ones((4, hidden, outer), dtype=torch.bfloat16, device="cuda")
        out = expert_layer(x, torch.ones((tokens, 4), device="cuda"), 2, a, b)
        assert out.shape == (tokens, outer) and bool((out == 0).all())


def test_hidden_values_beyond_the_type():
    """float16: a hidden value beyond its range is infinite, not NaN."""
    torch = require_gpu()
    from purin_amd import expert_layer

    x = torch.full((1, 64), 100.0, dtype=torch.float16, device="cuda")
    a = torch.full((1, 64, 32), 100.0, dtype=torch.float16, device="cuda")
    b = torch.full((1, 32, 8), 1.0, dtype=torch.float16, device="cuda")
    out = expert_layer(x, torch.ones((1, 1), device="cuda"), 1, a, b, "relu")
    assert bool((out == float("inf")).all())


@pytest.mark.parametrize("experts", [1, 300])  # the choice inside the first product, and before it
def test_weights_far_from_one(experts):
    """float16: a token's weight neither takes hidden values out of the range nor results' digits."""
    torch = require_gpu()
    from purin_amd import expert_layer

    def run(weight, a, b):
        ones = lambda *size: torch.ones(size, dtype=torch.float16, device="cuda")  # noqa: E731
        w = torch.zeros((1, experts), device="cuda")
        w[0, -1] = weight
        return expert_layer(ones(1, 64), w, 1, a * ones(experts, 64, 32), b * ones(experts, 32, 8), "relu")

    # all sums are of equal powers of two times 125: exact, and rounded once
    out = run(1000.0, 15.625, 2.0 ** -10)  # hidden 1000, 31.25 without the weight
    assert bool((out == torch.tensor(31250.0).half().cuda()).all())
    out = run(2.0 ** -20, 2.0 ** -16, 2.0 ** 15)  # hidden 2^-10, 2^10 without the weight
    assert bool((out == 2.0 ** -10).all())


def test_layer_wider_than_the_kernels():
    torch = require_gpu()
    from purin_amd import expert_layer

    for width, hidden, outer in (((1 << 20) + 8, 2, 2), (2, (1 << 19) + 8, 2), (2, 2, (1 << 20) + 8)):
        # powers of two: sums within 24 bits, exact, from 1 to 1 + 2^-16, 1 when rounded
        x = torch.full((2, width), 2.0 ** -(width.bit_length() - 1), dtype=torch.bfloat16, device="cuda")
        a = torch.ones((1, width, hidden), dtype=torch.bfloat16, device="cuda")
        b = torch.full((1, hidden, outer), 2.0 ** -(hidden.bit_length() - 1), dtype=torch.bfloat16,
                       device="cuda")
        out = expert_layer(x, torch.ones((2, 1), device="cuda"), 1, a, b, "relu")
        assert out.shape == (2, outer) and bool((out == 1).all())


@pytest.mark.parametrize("dtype", ["f32", "f64", "bf16"])
def test_layer_as_separate_operators(dtype):
    """Other types, more tokens, and gradients: the same layer from its operators."""
    torch = require_gpu()
    from purin_amd import activate, combine, dispatch, expert_layer, expert_product, route

    t = _types(torch)[dtype]
    tokens = 100 if dtype == "bf16" else 20
    x = _randn(torch, 1, (tokens, 24), t).requires_grad_()
    w = _weights(torch, 2, tokens, 6, "f32").requires_grad_()
    a = _randn(torch, 3, (6, 24, 32), t, 0.2).requires_grad_()
    b = _randn(torch, 4, (6, 16, 24), t, 0.2).requires_grad_()
    cot = _randn(torch, 5, (tokens, 24), t)
    out = expert_layer(x, w, 3, a, b, "gelu")
    r = route(w, 3)
    rows = activate(expert_product(dispatch(x, r), a, r), "gelu")
    want = combine(expert_product(rows, b, r), r)
    assert torch.equal(out, want)
    for got, other in zip(torch.autograd.grad(out, (x, w, a, b), cot),
                          torch.autograd.grad(want, (x, w, a, b), cot)):
        assert torch.equal(got, other)
    with torch.no_grad():
        assert torch.equal(expert_layer(x, w, 3, a, b, "gelu"), want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_layer_of_packed_weights_with_a_gradient(dtype):
    """Packed weights beside float32 tokens, or tokens that want a gradient: separate operators."""
    torch = require_gpu()
    from purin_amd import activate, combine, dispatch, expert_layer, expert_product, pack, route

    t = _types(torch)[dtype]
    x = _randn(torch, 1, (20, 40), t).requires_grad_()
    w = _weights(torch, 2, 20, 6, "f32").requires_grad_()
    a = pack(_randn(torch, 3, (6, 40, 64), t, 0.2), "fp4", axis=1)
    b = pack(_randn(torch, 4, (6, 32, 40), t, 0.2), "fp4", axis=1)
    cot = _randn(torch, 5, (20, 40), t)
    out = expert_layer(x, w, 3, a, b)
    r = route(w, 3)
    want = combine(expert_product(activate(expert_product(dispatch(x, r), a, r)), b, r), r)
    assert torch.equal(out, want)
    for got, other in zip(torch.autograd.grad(out, (x, w), cot), torch.autograd.grad(want, (x, w), cot)):
        assert torch.equal(got, other)


# ---------------------------------------------------------------------------
# beyond 32 bits
# ---------------------------------------------------------------------------


def test_packed_weights_beyond_32_bit_offsets():
    """More than 2^32 bytes of codes, more than 2^33 elements: both ends."""
    torch = require_gpu()
    from purin_amd import Microscaled, expert_layer, expert_product, unpack

    experts, inner, outer = 550, 4096, 4096
    codes = torch.zeros((experts, outer, inner // 2), dtype=torch.uint8, device="cuda")
    scales = torch.full((experts, outer, inner // 32), 120, dtype=torch.uint8, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    for e in (0, experts - 1):
        codes[e].random_(0, 256, generator=g)
    assert codes.numel() > 1 << 32
    m = Microscaled(codes, scales, "fp4", (experts, inner, outer), 1, torch.bfloat16)
    x = _randn(torch, 2, (8, inner), torch.bfloat16)
    at = torch.full((experts + 1,), 3, dtype=torch.int32, device="cuda")
    at[0], at[-1] = 0, 8
    out = expert_product(x, m, at).double()
    weights = torch.zeros((2, experts), device="cuda")
    weights[0, 0] = weights[1, -1] = 1.0
    back = Microscaled(codes, scales, "fp4", (experts, outer, inner), 1, torch.bfloat16)
    layer = expert_layer(x[:2], weights, 1, m, back, "relu").double()
    for e, (i, j), row in ((0, (0, 3), 0), (experts - 1, (3, 8), 1)):
        one = unpack(Microscaled(codes[e:e + 1], scales[e:e + 1], "fp4", (1, inner, outer), 1,
                                 torch.bfloat16))[0].double()
        want, terms = x[i:j].double() @ one, x[i:j].double().abs() @ one.abs()
        bound = UNIT["bf16"] * want.abs() + 2 * (inner + 2) * SUMS["bf16"] * terms + STEP["bf16"]
        assert bool(((out[i:j] - want).abs() <= bound).all())
        h = torch.relu(x[row].double() @ one)
        reach = 1.13 * (x[row].double().abs() @ one.abs())
        want, terms = h @ one, (h + reach) @ one.abs()
        off = 2 * (inner + outer + 4) * SUMS["bf16"] + 2 * UNIT["bf16"] ** 2
        bound = UNIT["bf16"] * want.abs() + off * terms + STEP["bf16"]
        assert bool(((layer[row] - want).abs() <= bound).all())


def test_rows_beyond_32_bit_offsets():
    """Packing, unpacking and the activation of more than 2^33 elements."""
    torch = require_gpu()
    from purin_amd import activate, pack, unpack

    rows, length = (1 << 21) + 3, 4128
    one = _randn(torch, 1, (1, length), torch.bfloat16)
    x = one.expand(rows, length).contiguous()
    x[-1] *= 3
    m, small = pack(x, "int8"), pack(one, "int8")
    last = pack(x[-1:], "int8")
    for got, first, end in ((m.codes, small.codes, last.codes), (m.scales, small.scales, last.scales)):
        assert bool((got[:-1] == first).all()) and torch.equal(got[-1:], end)
    y = unpack(m)
    assert bool((y[:-1] == unpack(small)).all()) and torch.equal(y[-1:], unpack(last))
    del y, m
    out = activate(x, "relu")
    assert bool((out[:-1] == activate(one, "relu")).all())
    assert torch.equal(out[-1:], activate(x[-1:].contiguous(), "relu"))


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------


def test_a_training_step_with_kept_rows_against_one_without():
    """route to combine with ``saved`` everywhere: outputs equal; gradients as far apart as half a
    64th of each block's power of two lets them."""
    torch = require_gpu()
    from purin_amd import activate, combine, dispatch, expert_product, route

    w = torch.softmax(_randn(torch, 1, (300, 12), torch.float32), 1).requires_grad_()
    x = _randn(torch, 2, (300, 64), torch.float32).requires_grad_()
    a = _randn(torch, 3, (12, 64, 96), torch.float32, 0.125).requires_grad_()
    b = _randn(torch, 4, (12, 48, 64), torch.float32, 0.14).requires_grad_()
    cot = _randn(torch, 5, (300, 64), torch.float32)

    def step(saved):
        r = route(w, 3)
        rows = expert_product(dispatch(x, r), a, r, saved=saved)
        rows = activate(rows, "silu", saved=saved)
        out = combine(expert_product(rows, b, r, saved=saved), r)
        return out, torch.autograd.grad(out, (w, x, a, b), cot)

    (out, grads), (want, exact) = step("int8"), step(None)
    assert torch.equal(out, want) and torch.equal(grads[0], exact[0])
    for g, e in zip(grads[1:], exact[1:]):
        # an element is off by at most 2^-7 of its block's largest, which is below 4 times the
        # root mean square of normal rows; errors of both signs add up as squares do
        assert float((g - e).norm() / e.norm()) < 2.0 ** -7 * 4


def test_results_repeat_bit_for_bit():
    torch = require_gpu()
    from purin_amd import activate, expert_layer, expert_product, pack

    x = _randn(torch, 1, (50, 264), torch.bfloat16)
    w = torch.softmax(_randn(torch, 2, (50, 24), torch.float32), 1)
    a = pack(_randn(torch, 3, (24, 264, 144), torch.bfloat16, 0.06), "fp4", axis=1)
    b = pack(_randn(torch, 4, (24, 72, 264), torch.bfloat16, 0.1), "fp4", axis=1)
    at = torch.arange(25, dtype=torch.int32, device="cuda") * 2

    def once():
        u = expert_product(x, a, at)
        return [expert_layer(x, w, 4, a, b), u, activate(u), expert_product(pack(x, "fp4"), a, at)]

    first = once()
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, once()))


def test_another_stream_and_a_workspace_of_the_callers():
    torch = require_gpu()
    from purin_amd import activate, expert_layer, expert_product, pack, unpack
    from purin_amd._lib import BF16
    from purin_amd.experts import expert_layer_workspace_bytes

    x = _randn(torch, 1, (50, 200), torch.bfloat16)
    w = torch.softmax(_randn(torch, 2, (50, 24), torch.float32), 1)
    a = _randn(torch, 3, (24, 200, 144), torch.bfloat16, 0.06)
    b = _randn(torch, 4, (24, 72, 200), torch.bfloat16, 0.1)
    at = torch.arange(25, dtype=torch.int32, device="cuda") * 2

    def once(**kw):
        m = pack(a, "fp4", axis=1)
        u = expert_product(x, m, at)
        return [expert_layer(x, w, 4, a, b, **kw), u, activate(u), unpack(m)]

    want = once()
    torch.cuda.synchronize()
    need = expert_layer_workspace_bytes(BF16, 50, 24, 4, 200, 72, 200)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    for fill in (0, 255):  # whatever it holds
        ws.fill_(fill)
        assert all(torch.equal(p, q) for p, q in zip(want, once(workspace=ws)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = once()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    with pytest.raises(Exception, match="workspace"):
        expert_layer(x, w, 4, a, b, workspace=ws[: need - 256])


def test_a_captured_layer_and_step_replay():
    """Served layers and products in one graph, replayed on new inputs with eager work between."""
    torch = require_gpu()
    from purin_amd import activate, expert_layer, expert_product, pack

    x = _randn(torch, 1, (24, 128), torch.bfloat16)
    w = torch.softmax(_randn(torch, 2, (24, 12), torch.float32), 1)
    a = _randn(torch, 3, (12, 128, 96), torch.bfloat16, 0.09)
    b = _randn(torch, 4, (12, 48, 128), torch.bfloat16, 0.14)
    pa, pb = pack(a, "fp4", axis=1), pack(b, "fp4", axis=1)
    at = torch.arange(13, dtype=torch.int32, device="cuda") * 2

    def once():
        u = expert_product(x, pa, at)
        return [expert_layer(x, w, 3, a, b), expert_layer(x, w, 3, pa, pb), activate(u),
                expert_product(pack(x, "fp4"), pa, at)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    with torch.cuda.graph(other):
        held_too = once()
    for k in range(4):
        x.copy_(_randn(torch, 10 + k, (24, 128), torch.bfloat16))
        w.copy_(torch.softmax(_randn(torch, 20 + k, (24, 12), torch.float32), 1))
        want = [t.clone() for t in once()]
        torch.cuda.synchronize()
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, held)), k
        assert all(torch.equal(p, q) for p, q in zip(want, held_too)), k


def test_refusals():
    torch = require_gpu()
    from purin_amd import (Microscaled, activate, expert_layer, expert_product, pack, unpack)
    from purin_amd._lib import PurinError

    x = torch.rand((6, 64), device="cuda").bfloat16()
    w = torch.rand((6, 4), device="cuda")
    a = torch.rand((4, 64, 32), device="cuda").bfloat16()
    b = torch.rand((4, 16, 8), device="cuda").bfloat16()
    m, r = pack(a, "fp4", axis=1), pack(x, "fp4")
    at = torch.tensor([0, 1, 2, 3, 6], dtype=torch.int32, device="cuda")
    part = lambda **kw: Microscaled(**{**m.__dict__, **kw})  # noqa: E731
    bad = [
        lambda: pack(x.double(), "fp4"), lambda: pack(x.int(), "int8"), lambda: pack(x, "fp4", axis=2),
        lambda: pack(x[0, 0], "fp4", axis=0), lambda: pack(x.cpu(), "fp4"), lambda: pack(x, 4),
        lambda: pack(x.to_sparse(), "fp4"),
        lambda: unpack(m, torch.float64), lambda: unpack(m, "f32"), lambda: unpack(part(kind="int8")),
        lambda: unpack(part(axis=3)), lambda: unpack(part(shape=(4, 65, 32))),
        lambda: unpack(part(codes=m.codes.int())), lambda: unpack(part(scales=m.scales[:, :, :2])),
        lambda: unpack(part(scales=m.scales.cpu())), lambda: unpack(part(codes=None)),
        lambda: activate(x.int()), lambda: activate(x[0]), lambda: activate(x[:, :63]),
        lambda: activate(x.double(), saved="int8"),
        lambda: expert_product(x.double(), m, at), lambda: expert_product(x[:, :63], m, at),
        lambda: expert_product(x, m, at[:-1]), lambda: expert_product(x, m, at.long()),
        lambda: expert_product(x, m, at, saved="int8"), lambda: expert_product(r, a, at),
        lambda: expert_product(x, pack(a, "int8", axis=1), at),
        lambda: expert_product(x, pack(a, "fp4", axis=2), at),
        lambda: expert_product(pack(x, "int8"), m, at), lambda: expert_product(x.cpu(), m, at),
        lambda: expert_product(pack(x, "fp4", axis=0), m, at), lambda: expert_product(x, m, at.cpu()),
        lambda: expert_product(pack(x[:, :32], "fp4"), m, at),
        lambda: expert_product(x.double(), a.double(), at, saved="int8"),
        lambda: expert_layer(x, w, 0, a, b), lambda: expert_layer(x, w, 5, a, b),
        lambda: expert_layer(x, w, True, a, b), lambda: expert_layer(x, w[:5], 2, a, b),
        lambda: expert_layer(x, w[:, :3], 2, a, b), lambda: expert_layer(x[:, :32], w, 2, a, b),
        lambda: expert_layer(x, w, 2, a, b[:, :15]), lambda: expert_layer(x, w, 2, a.float(), b),
        lambda: expert_layer(x, w, 2, a, b.half()), lambda: expert_layer(x, w, 2, a[0], b),
        lambda: expert_layer(x.double(), w, 2, m, pack(b, "fp4", axis=1)),
        lambda: expert_layer(x, w, 2, pack(a, "int8", axis=1), b), lambda: expert_layer(x, w.int(), 2, a, b),
        lambda: expert_layer(x, w, 2, a, b, workspace=5), lambda: expert_layer(x.cpu(), w, 2, a, b),
        lambda: expert_layer(x, w.cpu(), 2, a, b), lambda: expert_layer(x, w, 2, a.cpu(), b),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            print("not refused:", i)
    for f in (lambda: pack(a.clone().requires_grad_(), "fp4"),
              lambda: expert_layer(x, w, 2, a, b, workspace=torch.empty(8, device="cuda"))):
        with pytest.raises(PurinError):
            f()
    # once differentiable, in reverse; no tangents and no traces
    u = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(activate(u).sum(), u, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        g.sum().backward()
    (g,) = torch.autograd.grad(expert_product(u, m, at).sum(), u, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        g.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, x)
        for f in (lambda: activate(dual), lambda: pack(dual, "fp4"), lambda: expert_product(dual, m, at),
                  lambda: expert_layer(dual, w, 2, a, b)):
            with pytest.raises(PurinError, match="forward-mode"):
                f()
    with pytest.raises(PurinError, match="traced"):
        torch.jit.trace(lambda v: activate(v), (x,), check_trace=False)
