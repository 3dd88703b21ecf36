"""The operators around the projection layer on inputs that need care: what is refused, and what
has to come out right in spite of an unusual form."""

import dataclasses

import numpy as np
import pytest

from oracle import train as ot
from tests._gpu import require_gpu, to_np

pytestmark = pytest.mark.gpu


def test_a_routing_with_other_index_tensors():
    """``place`` and ``offsets`` of a routing are read as int32 in order: another type, shape or
    device is refused, another order in memory is read as what it says."""
    torch = require_gpu()
    from purin_amd import combine, dispatch, route

    rng = np.random.default_rng(2)
    w = torch.as_tensor(rng.random((7, 5)) * (rng.random((7, 5)) < 0.6)).cuda()
    x = torch.as_tensor(rng.standard_normal((7, 6))).cuda()
    r = route(w, 3)
    y = torch.as_tensor(rng.standard_normal((21, 6))).cuda()
    bad = [dict(place=r.place.long()), dict(place=r.place.float()), dict(place=r.place.cpu()),
           dict(place=r.place.view(-1)), dict(place=r.place[:, :0]), dict(place=None),
           dict(offsets=r.offsets.long()), dict(offsets=r.offsets.cpu()), dict(offsets=None),
           dict(offsets=r.offsets[:1]), dict(offsets=r.offsets.view(2, 3))]
    for change in bad:
        other = dataclasses.replace(r, **change)
        for f in (lambda: dispatch(x, other), lambda: combine(y, other),
                  lambda: combine(y.clone().requires_grad_(), other)):
            with pytest.raises(ValueError):
                f()
                print("not refused:", change, flush=True)
    # the same values in another order, and one row of places for all tokens
    turned = dataclasses.replace(r, place=r.place.t().contiguous().t(),
                                 offsets=torch.stack((r.offsets, r.offsets), 1)[:, 0])
    assert not turned.place.is_contiguous() and not turned.offsets.is_contiguous()
    assert torch.equal(dispatch(x, turned), dispatch(x, r))
    assert torch.equal(combine(y, turned), combine(y, r))
    one = dataclasses.replace(r, place=r.place[:1].expand(7, 3))
    place, chosen = np.repeat(to_np(r.place[:1]), 7, 0), to_np(r.weights)
    want = ot.combine(to_np(y), place, chosen)
    terms = ot.combine(np.abs(to_np(y)), place, chosen)
    # three products and sums in 64 bits
    assert (np.abs(to_np(combine(y, one)) - want) <= 2 * 5 * 2.0 ** -53 * terms).all()


def test_a_workspace_is_one_piece_of_memory():
    """A broadcast or strided workspace has fewer bytes in one piece than its size says."""
    torch = require_gpu()
    from purin_amd import clip_gradients, gradient_norm, route, route_experts
    from purin_amd.gradients import clip_workspace_bytes
    from purin_amd.routing import route_workspace_bytes

    w = torch.rand((4000, 20), device="cuda")
    ids = torch.zeros((4000, 3), dtype=torch.int32, device="cuda")
    g = [torch.rand(50, device="cuda")]
    need = max(route_workspace_bytes(4000, 20, 3), clip_workspace_bytes(1))
    whole = torch.empty((need, 2), dtype=torch.uint8, device="cuda")
    for ws in (whole[:1, :1].expand(need, 1), whole[:, 0], whole.t(), whole.cpu()):
        for f in (lambda: route(w, 3, workspace=ws), lambda: route_experts(ids, 20, workspace=ws),
                  lambda: gradient_norm(g, workspace=ws),
                  lambda: clip_gradients(g, 1.0, workspace=ws)):
            with pytest.raises(ValueError, match="workspace"):
                f()
    route(w, 3, workspace=whole)


def _layer(torch):
    """Tensors and the calls that have a derivative, each of one of them."""
    from purin_amd import clip_gradients, combine, dispatch, expert_product, gradient_norm, route

    rng = np.random.default_rng(4)
    make = lambda *shape: torch.as_tensor(rng.random(shape), dtype=torch.float32).cuda()  # noqa: E731
    w, x, y, m = make(6, 4), make(6, 8), make(12, 8), make(4, 8, 5)
    r = route(w, 2)
    return [(w, lambda t: route(t, 2).weights), (x, lambda t: dispatch(t, r)),
            (y, lambda t: combine(t, r)), (r.weights, lambda t: combine(y, r, t)),
            (y, lambda t: expert_product(t, m, r)), (m, lambda t: expert_product(y, t, r)),
            (x, lambda t: gradient_norm([t])),
            (x, lambda t: clip_gradients([t], 1.0, out=[torch.empty_like(x)])),
            (x, lambda t: clip_gradients([x], 1.0, out=[t]))]


def test_a_tangent_is_refused_and_not_lost():
    torch = require_gpu()
    import torch.autograd.forward_ad as fw
    from purin_amd._lib import PurinError

    for i, (t, f) in enumerate(_layer(torch)):
        for grad in (False, True):
            with fw.dual_level():
                dual = fw.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t))
                with pytest.raises(PurinError, match="forward-mode"):
                    f(dual)
                    print("not refused:", i, grad, flush=True)
        out = f(t.clone())  # outside a level as before
        assert torch.isfinite(out).all()
    # forward over reverse: a tangent that comes in with the gradient
    for i, (t, f) in enumerate(_layer(torch)[:6]):
        x = t.clone().requires_grad_()
        out = f(x)
        with fw.dual_level():
            cot = fw.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(out, x, cot)
                print("not refused in reverse:", i, flush=True)


def test_a_trace_is_refused():
    """A trace would hold the outputs' allocation and not the kernels that fill them."""
    torch = require_gpu()
    from torch.fx.experimental.proxy_tensor import make_fx

    for i, (t, f) in enumerate(_layer(torch)[:7]):
        for trace in (lambda: torch.jit.trace(f, (t,)), lambda: make_fx(f)(t)):
            with pytest.raises(RuntimeError, match="cannot be traced"):
                trace()
                print("not refused:", i, flush=True)
        assert torch.isfinite(f(t)).all()


def test_function_transforms_raise():
    """Tensors of torch.func have no memory of their own: an error, and no wrong result."""
    torch = require_gpu()
    for t, f in _layer(torch)[:7]:
        for call in (lambda: torch.func.jvp(f, (t,), (t,)), lambda: torch.func.grad(
                lambda v: f(v).sum())(t), lambda: torch.func.vmap(f)(t[None])):
            with pytest.raises(Exception):
                call()


@pytest.mark.parametrize("width", [1, 8])
@pytest.mark.parametrize("view", ["imag", "whole"])
def test_lazily_negated_tensors(view, width):
    """The imaginary part of a conjugate holds its numbers' negatives and a mark; what a call
    reads and writes are the numbers."""
    torch = require_gpu()
    from purin_amd import (clip_gradients, combine, dispatch, expert_product, gradient_norm, route,
                           route_experts)

    def negated(t):  # t's numbers behind the mark, in memory of their own
        if view == "whole":
            return torch._neg_view(-t)
        return torch.complex(torch.zeros_like(t), -t).conj().imag

    rng = np.random.default_rng(6)
    make = lambda *s: torch.as_tensor(rng.standard_normal(s), dtype=torch.float32).cuda()  # noqa: E731
    w, x, y, m = make(9, 4), make(9, width), make(18, width), make(4, width, 5)
    assert negated(w).is_neg() and torch.equal(negated(w), w)
    r = route(w, 2)
    n = route(negated(w), 2)
    assert torch.equal(n.weights, r.weights) and torch.equal(n.experts, r.experts)
    assert torch.equal(dispatch(negated(x), r), dispatch(x, r))
    assert torch.equal(combine(negated(y), r), combine(y, r))
    assert torch.equal(combine(y, r, negated(r.weights)), combine(y, r))
    given = route_experts(r.experts, 4, weights=negated(r.weights))
    assert torch.equal(combine(y, given), combine(y, r))
    out = expert_product(y, m, r)
    assert torch.equal(expert_product(negated(y), m, r), out)
    assert torch.equal(expert_product(y, negated(m), r), out)

    def gradients(f, inputs, cot):
        inputs = [t.clone().requires_grad_() for t in inputs]
        return torch.autograd.grad(f(*inputs), inputs, cot)

    for f, inputs, shape in ((lambda a: route(a, 2).weights, (w,), (9, 2)),
                             (lambda a: dispatch(a, r), (x,), (18, width)),
                             (lambda a, b: combine(a, r, b), (y, r.weights), (9, width)),
                             (lambda a, b: expert_product(a, b, r), (y, m), (18, 5))):
        cot = make(*shape)
        want, got = gradients(f, inputs, cot), gradients(f, inputs, negated(cot))
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    # saved for the backward pass behind the mark
    a = torch.complex(torch.zeros_like(y), -y).requires_grad_()
    (g,) = torch.autograd.grad(expert_product(a.conj().imag, m, r).sum(), a)
    (want,) = gradients(lambda v: expert_product(v, m, r), (y,), torch.ones_like(out))
    assert torch.equal(g.imag, -want)

    assert torch.equal(gradient_norm([negated(x)]), gradient_norm([x]))
    want = [torch.empty_like(x)]
    clip_gradients([x], 1.0, out=want)
    for given, into in ((negated(x), torch.empty_like(x)), (x, negated(x)),
                        (negated(x), negated(x))):
        clip_gradients([given], 1.0, out=[into])
        assert torch.equal(into, want[0])
        assert torch.equal(given, x)
    here = negated(x)
    clip_gradients([here], 1.0)
    assert torch.equal(here, want[0])


def test_clip_refuses_strided_views_that_share_memory():
    torch = require_gpu()
    from purin_amd import clip_gradients
    from purin_amd._lib import PurinError

    base = torch.rand((6, 10), device="cuda") + 0.5
    other = torch.rand((6, 5), device="cuda")

    def refused(make):  # make(b): gradients and outputs on b
        b, o = base.clone(), other.clone()
        gradients, out = make(b, o)
        with pytest.raises((PurinError, ValueError)):
            clip_gradients(gradients, 0.1, out=out)
            print("not refused", flush=True)
        assert torch.equal(b, base) and torch.equal(o, other)  # and nothing was written

    refused(lambda b, o: ([b[:, :5], b[:, 3:8]], None))
    refused(lambda b, o: ([b[::2, ::3], b[2:, 6:]], None))
    refused(lambda b, o: ([b.t()[1:9], b[3]], None))
    refused(lambda b, o: ([b[:, 2], b[2]], None))
    refused(lambda b, o: ([b[:, 2], b.view(-1)[12:13]], None))
    # an output over another gradient, and over another output
    refused(lambda b, o: ([o, b[:, :5]], [b[:, 4:9], o.clone()]))
    refused(lambda b, o: ([o, b], [b[:, 4:9], b.clone()]))
    refused(lambda b, o: ([o, o.clone()], [b[:, :5], b[:, 4:9]]))
    refused(lambda b, o: ([o, o.clone()], [b[:, :5], b.view(-1)[7:37].view(6, 5)]))
    refused(lambda b, o: ([b[:, :5], o], [o.clone(), b[:, 4:9]]))

    def taken(make):  # disjoint views: as if each had memory of its own
        b = base.clone()
        gradients, out = make(b)
        alone = [g.clone() for g in gradients]
        norm = clip_gradients(alone, 0.1)
        assert torch.equal(clip_gradients(gradients, 0.1, out=out), norm)
        for o, a in zip(gradients if out is None else out, alone):
            assert torch.equal(o, a)

    taken(lambda b: ([b[:, :5], b[:, 5:]], None))
    taken(lambda b: ([b[:, i] for i in range(10)], None))
    taken(lambda b: ([b[::2, ::2], b[1::2, 1::2], b[::2, 1::2], b[1::2, ::2]], None))
    taken(lambda b: ([b[:2].t(), b[2:4].t(), b[4:, 1::2], b[4:, ::2]], None))
    taken(lambda b: ([b.t()[:5], b[:, 5], b.view(-1)[6:10], b[1:, 6:]], None))
    taken(lambda b: ([b[:, :5].clone(), b[:, 5:].clone()], [b[:, 5:], b[:, :5]]))
    # a gradient and its own output in another order
    square = torch.rand((8, 8), device="cuda")
    want = square.clone()
    norm = clip_gradients([want], 0.1)
    assert torch.equal(clip_gradients([square], 0.1, out=[square.t()]), norm)
    assert torch.equal(square.t(), want)
    # a broadcast gradient is read, and two may read the same memory where nothing is written
    row = base[:1].expand(4, 10)
    out = [torch.empty(4, 10, device="cuda"), torch.empty(4, 10, device="cuda")]
    clip_gradients([row, row.clone()], 0.1, out=out)
    assert torch.equal(out[0], out[1])
    clip_gradients([base[:, :5], base[:, 3:8]], 0.1, out=[torch.empty_like(other) for _ in "ab"])


@pytest.mark.parametrize("dtype", ["f32", "f64", "bf16", "f16", "mixed"])
def test_the_norm_has_a_gradient(dtype):
    """g / norm times the incoming gradient.  The norm is rounded to its type (u), the factor to
    the sums' type and the product once more, then to the gradient's type (h)."""
    torch = require_gpu()
    from purin_amd import gradient_norm

    types = {"f32": torch.float32, "f64": torch.float64, "bf16": torch.bfloat16,
             "f16": torch.float16}
    names = list(types) if dtype == "mixed" else [dtype] * 4
    rng = np.random.default_rng(8)
    shapes = [(700, 41), (1,), (33, 5, 7), (0, 3)]
    g = [torch.as_tensor(rng.standard_normal(s)).to(types[n]).cuda()
         for s, n in zip(shapes, names)]
    g[2] = g[2].permute(2, 0, 1)  # dense in another order
    with torch.no_grad():
        plain = gradient_norm(g)
    g = [t.requires_grad_() for t in g] + [None]
    norm = gradient_norm(g)
    assert torch.equal(norm.detach(), plain) and norm.requires_grad
    wide = norm.dtype == torch.float64
    got = torch.autograd.grad(norm * 3.0, [t for t in g if t is not None])
    exact = np.sqrt(sum((to_np(t.detach().double()) ** 2).sum() for t in g if t is not None))
    for t, d in zip(g, got):
        assert d.shape == t.shape and d.dtype == t.dtype
        want = 3.0 * to_np(t.detach().double()) / exact
        u = 2.0 ** -53 if wide else 2.0 ** -24  # norm, and its incoming gradient times 3
        a = 2.0 ** -53 if t.dtype == torch.float64 else 2.0 ** -24  # factor and product
        h = {8: 2.0 ** -53, 4: 2.0 ** -24}.get(t.element_size(),
                                                2.0 ** -8 if t.dtype == torch.bfloat16 else 2.0 ** -11)
        step = {torch.float16: 2.0 ** -24, torch.float64: 2.0 ** -1022}.get(t.dtype, 2.0 ** -126)
        bound = np.abs(want) * (2 * u + 4 * 2.0 ** -53 + 2 * a + h) * 1.01 + step
        assert (np.abs(to_np(d.double()) - want) <= bound).all()


def test_the_norms_gradient_at_the_edges():
    torch = require_gpu()
    from purin_amd import gradient_norm

    # at zero: zero, not NaN
    z = torch.zeros(5, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(gradient_norm([z]), z)
    assert (g == 0).all()
    # one of a list, a strided one, a broadcast one
    x = torch.rand((6, 8), device="cuda", dtype=torch.float64, requires_grad=True)
    y = torch.rand(3, device="cuda", dtype=torch.float64)
    (g,) = torch.autograd.grad(gradient_norm([y, x[:, ::2], x[:1].expand(4, 8)]), x)
    want = x.detach() * 0
    want[:, ::2] += x.detach()[:, ::2]
    want[0] += 4 * x.detach()[0]
    total = (y.square().sum() + x.detach()[:, ::2].square().sum()
             + 4 * x.detach()[0].square().sum()).sqrt()
    assert float((g - want / total).abs().max()) < 1e-14
    # by differences
    a, b = (torch.rand(s, device="cuda", dtype=torch.float64).requires_grad_() for s in (7, 4))
    assert torch.autograd.gradcheck(lambda a, b: gradient_norm([a, b]), (a, b), eps=1e-6,
                                    atol=1e-8, rtol=0)
    # a factor that 32 bits do not hold
    tiny = torch.full((4,), 2.0 ** -120, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(gradient_norm([tiny]), tiny)
    assert (g == 0.5).all()
    # NaN shows
    n = torch.tensor([1.0, float("nan")], device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(gradient_norm([n]), n)
    assert torch.isnan(g).all()
    # a penalty on gradients reaches what they came from
    p = torch.rand(9, device="cuda", dtype=torch.float64, requires_grad=True)
    (d,) = torch.autograd.grad(p.pow(3).sum(), p, create_graph=True)
    (g,) = torch.autograd.grad(gradient_norm([d]), p)
    d = d.detach()
    assert float((g - d / d.norm() * 6 * p.detach()).abs().max()) < 1e-13
    # no gradients of gradients
    (g,) = torch.autograd.grad(gradient_norm([p]), p, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), p)
    # no graph where none is wanted
    with torch.no_grad():
        assert not gradient_norm([p]).requires_grad
    assert not gradient_norm([p.detach()]).requires_grad


def test_the_norms_gradient_of_a_long_list():
    """More tensors than one launch takes, and a tensor of many pieces among them."""
    torch = require_gpu()
    from purin_amd import gradient_norm

    rng = np.random.default_rng(9)
    sizes = [int(n) for n in rng.integers(0, 40, 210)]
    sizes[100] = 200_003
    g = [torch.as_tensor(rng.standard_normal(n)).cuda().requires_grad_() for n in sizes]
    norm = gradient_norm(g)
    got = torch.autograd.grad(norm, g)
    exact = np.sqrt(sum((to_np(t) ** 2).sum() for t in g))
    for t, d in zip(g, got):
        want = to_np(t) / exact
        assert (np.abs(to_np(d) - want) <= 8 * 2.0 ** -53 * np.abs(want)).all()
