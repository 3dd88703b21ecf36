"""Layers, packed products, kept rows and the activation where other tests do not reach: what a
graph holds, the largest tiles, both sides of the launches' rules, mixed weights, offsets beyond 32
bits, two threads, a captured training step.

Tolerances as in ``test_gpu_experts``: u |exact| + 2 (K + 2) a sum|terms| of a sum of K products.
"""

import threading

import numpy as np
import pytest

from tests._gpu import require_gpu
from tests.test_gpu_experts import _layer_close
from tests.test_gpu_train import STEP, SUMS, UNIT, _np, _randn, _types, _weights

pytestmark = pytest.mark.gpu

HALF = ["bf16", "f16"]


# ---------------------------------------------------------------------------
# what a graph holds
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("gated", [True, False])
def test_a_graph_of_the_activation_holds_eight_bits(gated):
    """The input belongs to nothing but the graph: 2 bytes an element of it, or 33 / 32."""
    torch = require_gpu()
    from purin_amd import activate

    leaf = _randn(torch, 1, (4096, 1024), torch.bfloat16).requires_grad_()
    full = leaf.numel() * leaf.element_size()

    def held(saved):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = activate(leaf * 1, "silu", gated=gated, saved=saved)
        assert out.requires_grad
        return torch.cuda.memory_allocated() - before - out.numel() * out.element_size()

    assert held(None) >= full
    assert 0.5 * full < held("int8") < 0.53 * full


# ---------------------------------------------------------------------------
# tiles
# ---------------------------------------------------------------------------


def _uneven(torch, seed, shape, axis, dtype, spread=4):
    """Normal numbers whose blocks of 32 along ``axis`` differ by powers of two, each from the next."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g, dtype=torch.float32).movedim(axis, -1)
    blocks = -(-x.shape[-1] // 32)
    power = torch.randint(-spread, spread + 1, (*x.shape[:-1], blocks), generator=g)
    x = x * torch.exp2(power.float()).repeat_interleave(32, -1)[..., :x.shape[-1]]
    return x.movedim(-1, axis).contiguous().to(dtype).cuda()


def _product_close(torch, out, an, m, counts, dtype):
    """On the card in 64 bits, expert by expert; zeros behind the last one."""
    from purin_amd import Microscaled, unpack

    at = 0
    inner = an.shape[1]
    for e, n in enumerate(counts):
        wn = unpack(Microscaled(m.codes[e:e + 1], m.scales[e:e + 1], "fp4", (1, *m.shape[1:]), 1,
                                torch.float32))[0].double()
        want, terms = an[at:at + n].double() @ wn, an[at:at + n].double().abs() @ wn.abs()
        bound = UNIT[dtype] * want.abs() + 2 * (inner + 2) * SUMS[dtype] * terms + STEP[dtype]
        assert bool(((out[at:at + n].double() - want).abs() <= bound).all()), e
        at += n
    assert bool((out[at:] == 0).all())


# rows to each expert, inner, outer: with scales by whole pieces (a row's blocks, filled up to fours,
# are a multiple of 16) over several chunks of 32, the last one whole or in part; and with others
BOTH = [((4000, 4190), 4096, 8200), ((4000, 4190), 2500, 8200), ((4090, 4100), 3500, 8200),
        ((256, 128, 300, 0, 5), 4096, 384), ((256, 128, 300, 0, 5), 2500, 384),
        ((130, 0, 257), 3500, 200), ((1, 127), 2208, 136), ((260, 3), 4100, 264)]


@pytest.mark.parametrize("counts,inner,outer", BOTH)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_both_packed_over_several_chunks_of_scales(counts, inner, outer, dtype):
    torch = require_gpu()
    from purin_amd import expert_product, pack, unpack

    print(f"both packed {counts} {inner} {outer} {dtype}", flush=True)
    t = _types(torch)[dtype]
    rows = sum(counts) + 7
    m = pack(_uneven(torch, 1, (len(counts), inner, outer), 1, torch.float32), "fp4", axis=1)
    a = pack(_uneven(torch, 2, (rows, inner), 1, t) * inner ** -0.5, "fp4")
    at = torch.as_tensor(np.concatenate(([0], np.cumsum(counts))), dtype=torch.int32).cuda()
    out = expert_product(a, m, at)
    assert out.dtype == t
    _product_close(torch, out, unpack(a), m, counts, dtype)


@pytest.mark.parametrize("counts,inner,outer", [((4000, 4190), 328, 8200), ((4000, 4190), 333, 8200),
                                                ((300, 260, 0, 140), 333, 1100)])
@pytest.mark.parametrize("dtype", HALF)
def test_large_tiles_of_rows_at_odd_addresses(counts, inner, outer, dtype):
    torch = require_gpu()
    from purin_amd import expert_product, pack

    print(f"odd addresses {counts} {inner} {outer} {dtype}", flush=True)
    t = _types(torch)[dtype]
    m = pack(_uneven(torch, 1, (len(counts), inner, outer), 1, torch.float32), "fp4", axis=1)
    wide = _uneven(torch, 2, (sum(counts) + 7, inner + 5), 1, t) * inner ** -0.5
    at = torch.as_tensor(np.concatenate(([0], np.cumsum(counts))), dtype=torch.int32).cuda()
    a = wide[:, 3:3 + inner]
    _product_close(torch, expert_product(a, m, at), a, m, counts, dtype)


@pytest.mark.parametrize("counts,inner,outer", [((4000, 4190), 2048, 2048), ((2100, 0, 1999), 1032, 1528)])
@pytest.mark.parametrize("order", ["io", "oi"])
@pytest.mark.parametrize("dtype", HALF)
def test_kept_rows_at_sizes_of_large_tiles(counts, inner, outer, order, dtype):
    torch = require_gpu()
    from purin_amd import expert_product, pack, unpack

    print(f"kept rows {counts} {inner} {outer} {order} {dtype}", flush=True)
    t = _types(torch)[dtype]
    rows = sum(counts) + 7
    a = _uneven(torch, 1, (rows, inner), 1, t).requires_grad_()
    w = _randn(torch, 2, (len(counts), inner, outer), t, inner ** -0.5)
    w = (w if order == "io" else w.transpose(1, 2).contiguous().transpose(1, 2)).requires_grad_()
    cot = _randn(torch, 3, (rows, outer), t, 2.0 ** -6)
    at = torch.as_tensor(np.concatenate(([0], np.cumsum(counts))), dtype=torch.int32).cuda()
    out = expert_product(a, w, at, saved="int8")
    g_a, g_w = torch.autograd.grad(out, (a, w), cot)
    plain = expert_product(a, w, at)
    assert torch.equal(out, plain) and torch.equal(g_a, torch.autograd.grad(plain, a, cot)[0])
    kept = unpack(pack(a.detach(), "int8")).double()
    first = 0
    for e, n in enumerate(counts):
        k, c = kept[first:first + n], cot[first:first + n].double()
        want, terms = k.t() @ c, k.t().abs() @ c.abs()
        bound = UNIT[dtype] * want.abs() + 2 * (n + 2) * SUMS[dtype] * terms + STEP[dtype]
        assert bool(((g_w[e].double() - want).abs() <= bound).all()), e
        first += n


# ---------------------------------------------------------------------------
# layers
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("shape", [
    # up to 16 tokens and 128 pairs in codes: pairs times the first product's workgroups are too many
    # for each to choose by itself (81920 and 65536, of 49152), and few enough (40960)
    (16, 64, 8, 128, 320, 64), (16, 64, 8, 72, 256, 40), (16, 64, 8, 72, 160, 40),
    (13, 40, 5, 1032, 200, 264), (40, 12, 3, 200, 72, 520)])
@pytest.mark.parametrize("first,second", [("packed", "packed"), ("packed", "io"), ("packed", "oi"),
                                          ("io", "packed"), ("oi", "packed"), ("io", "oi"), ("oi", "io")])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("dtype", HALF)
def test_layer_of_weights_in_different_forms(shape, first, second, gated, dtype):
    torch = require_gpu()
    from purin_amd import expert_layer, pack, unpack

    print(f"layer {shape} {first} {second} {gated} {dtype}", flush=True)
    tokens, experts, slots, width, hidden, outer = shape
    t = _types(torch)[dtype]
    given, values = [], []
    for seed, form, size in ((2, first, (experts, width, 2 * hidden if gated else hidden)),
                             (3, second, (experts, hidden, outer))):
        w = _randn(torch, seed, size, t, size[1] ** -0.5)
        if form == "packed":
            w = pack(w, "fp4", axis=1)
        elif form == "oi":
            w = w.transpose(1, 2).contiguous().transpose(1, 2)
        given.append(w)
        values.append(_np(unpack(w) if form == "packed" else w))
    weights = _weights(torch, 5, tokens, experts, "f32")
    x = _randn(torch, 1, (tokens, width), t)
    out = expert_layer(x, weights, slots, *given, "silu")
    _layer_close(torch, out, x, weights, slots, values, "silu", dtype)


# ---------------------------------------------------------------------------
# beyond 32 bits
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["fp4", "int8"])
def test_packing_across_memory_beyond_32_bit_offsets(kind):
    torch = require_gpu()
    from purin_amd import pack

    rows, length = (1 << 20) + 70, 4128
    column = _randn(torch, 1, (1, length, 1), torch.bfloat16)
    x = column.expand(1, length, rows).contiguous()
    assert x.numel() > 1 << 32
    x[:, :, -3:] *= 3
    m = pack(x, kind, axis=1)
    want = [pack(column, kind, axis=1), pack(x[:, :, -1:].contiguous(), kind, axis=1)]
    for got, first, last in ((m.codes, want[0].codes, want[1].codes),
                             (m.scales, want[0].scales, want[1].scales)):
        assert bool((got[:, :-3] == first).all()) and bool((got[:, -3:] == last).all())


def test_the_activation_with_kept_rows_beyond_32_bit_offsets():
    torch = require_gpu()
    from purin_amd import activate

    rows, columns = (1 << 20) + 70, 4128
    one = _randn(torch, 1, (1, columns), torch.bfloat16)
    cot = _randn(torch, 2, (1, columns // 2), torch.bfloat16)
    u = one.expand(rows, columns).contiguous()
    assert u.numel() > 1 << 32
    u[-3:] *= 3
    want = []
    for small in (one, one * 3):
        leaf = small.requires_grad_()
        out = activate(leaf, "relu", saved="int8")
        want.append((out.detach(), torch.autograd.grad(out, leaf, cot)[0]))
    u.requires_grad_()
    for saved in ("int8", None):
        out = activate(u, "relu", saved=saved)
        (g,) = torch.autograd.grad(out, u, cot.expand(rows, columns // 2).contiguous())
        if saved is None:
            for i, small in enumerate((one, one * 3)):
                leaf = small.detach().requires_grad_()
                want[i] = (want[i][0], torch.autograd.grad(activate(leaf, "relu"), leaf, cot)[0])
        for got, k in ((out.detach(), 0), (g, 1)):
            assert bool((got[:-3] == want[0][k]).all()) and bool((got[-3:] == want[1][k]).all())
        del out, g


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------


def test_two_threads_on_streams_of_their_own():
    torch = require_gpu()
    from purin_amd import activate, expert_layer, expert_product, pack, unpack

    def work(seed):
        x = _randn(torch, seed, (24, 264), torch.bfloat16)
        w = torch.softmax(_randn(torch, seed + 1, (24, 30), torch.float32), 1)
        a = pack(_randn(torch, seed + 2, (30, 264, 144), torch.bfloat16, 0.06), "fp4", axis=1)
        b = _randn(torch, seed + 3, (30, 72, 264), torch.bfloat16, 0.1)
        at = torch.arange(31, dtype=torch.int32, device="cuda").clamp_max(24)

        def once():
            leaf = x.detach().requires_grad_()
            u = expert_product(leaf, a, at)
            h = activate(u, saved="int8")
            (g,) = torch.autograd.grad(h, leaf, torch.ones_like(h))
            return [expert_layer(x, w, 3, a, b), u.detach(), g, unpack(pack(b, "int8"))]

        return once

    calls = [work(10), work(20)]
    want = [f() for f in calls]
    torch.cuda.synchronize()
    bad = []

    def loop(k):
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            for _ in range(20):
                got = calls[k]()
                side.synchronize()
                if not all(torch.equal(p, q) for p, q in zip(want[k], got)):
                    bad.append(k)

    threads = [threading.Thread(target=loop, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_a_captured_training_step_with_kept_rows():
    """Forward and backward in one graph; the captured leaves are in no other graph."""
    torch = require_gpu()
    from purin_amd import activate, combine, dispatch, expert_product, pack, route

    def fresh(k):
        return (torch.softmax(_randn(torch, 10 + k, (300, 12), torch.float32), 1),
                _randn(torch, 20 + k, (300, 64), torch.bfloat16),
                _randn(torch, 30 + k, (12, 64, 96), torch.bfloat16, 0.125),
                _randn(torch, 40 + k, (12, 48, 64), torch.bfloat16, 0.14))

    cot = _randn(torch, 5, (300, 64), torch.bfloat16)
    head = pack(_randn(torch, 6, (12, 64, 64), torch.bfloat16, 0.125), "fp4", axis=1)

    def step(w, x, a, b):
        r = route(w, 3)
        rows = expert_product(dispatch(x, r), a, r, saved="int8")
        rows = activate(rows, "gelu", saved="int8")
        rows = expert_product(expert_product(rows, b, r, saved="int8"), head, r)
        out = combine(rows, r)
        return (out.detach(), *torch.autograd.grad(out, (w, x, a, b), cot))

    leaves = [t.clone().requires_grad_() for t in fresh(0)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*[t.clone().requires_grad_() for t in fresh(0)])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(*leaves)
    for k in range(4):
        given = fresh(k)
        with torch.no_grad():
            for leaf, t in zip(leaves, given):
                leaf.copy_(t)
        want = [t.clone() for t in step(*[t.requires_grad_() for t in given])]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, held)), k
