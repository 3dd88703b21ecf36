"""A network's experts held, trained and served in less memory, as a user's program calls them.

Five kinds of call:

* ``layer``: a whole layer of experts for a few tokens: from the tokens' weights over the experts
  to the weighted sum of their experts' results, the experts' matrices dense or microscaled;
* ``pack``: a tensor to microscaled numbers of 4 or 8 bits, and back to the values these stand for;
* ``product``: the experts' products with microscaled weights, on rows of 16 bits (forward, or with
  the rows' gradient) or on rows that are packed in the call;
* ``saved``: the experts' products of a training step that keeps its rows in 8 bits for the
  weights' gradient;
* ``activate``: the activation between two products, forward and backward, its input kept in 8 bits.

With ``own`` false ``run`` computes them from elementary torch operations in 32 bits (scaling by
powers of two and rounding to few bits in 64, where they are exact).
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 32  # elements that share a scale

# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # one token of a served request: every weight of its experts is read for one row
        dict(name="layer-one", kind="layer", tokens=1, experts=64, slots=8, width=2048, hidden=1408,
             dtype="bf16", order="oi", act="silu", gated=True, packed=False, sparse=0.0),
        # odd sizes in half precision, ungated, projected weights: some tokens have no expert
        dict(name="layer-odd", kind="layer", tokens=13, experts=23, slots=3, width=1111, hidden=515,
             dtype="f16", order="io", act="relu", gated=False, packed=False, sparse=1.2),
        # a served batch, one token for each request
        dict(name="layer-serve", kind="layer", tokens=24, experts=32, slots=4, width=4096,
             hidden=1280, dtype="bf16", order="io", act="silu", gated=True, packed=False, sparse=0.0),
        # the most tokens, on microscaled weights, a large layer
        dict(name="layer-packed", kind="layer", tokens=64, experts=64, slots=6, width=4096,
             hidden=1408, dtype="bf16", order="oi", act="silu", gated=True, packed=True, sparse=0.0),
        # rows of odd length in single precision, to 8 bits and back
        dict(name="pack-odd", kind="pack", shape0=1, rows=4099, length=1111, dtype="f32",
             to="int8", order="rows"),
        # a network's weights to 4 bits and back, blocks across the rows that lie in memory
        dict(name="pack-weights", kind="pack", shape0=16, rows=4096, length=2048, dtype="bf16",
             to="fp4", order="columns"),
        # the products of a served batch, a few rows to an expert
        dict(name="product-serve", kind="product", rows=768, used=1.0, experts=32, inner=4096,
             outer=1536, dtype="bf16", both=False, train=False),
        # many rows, packed in the call: both operands in 4 bits
        dict(name="product-large", kind="product", rows=32768, used=1.0, experts=16, inner=2048,
             outer=4096, dtype="bf16", both=True, train=False),
        # odd sizes in single precision, with slots left empty at the end
        dict(name="saved-odd", kind="saved", rows=3001, used=0.9, experts=7, inner=515, outer=777,
             dtype="f32", order="io"),
        # an ordinary training step's product with both gradients
        dict(name="saved-train", kind="saved", rows=32768, used=1.0, experts=16, inner=2048,
             outer=4096, dtype="bf16", order="io"),
        # odd sizes in half precision, an activation without a gate
        dict(name="activate-odd", kind="activate", rows=4099, hidden=777, dtype="f16", act="gelu",
             gated=False),
        # the hidden rows of an ordinary training step
        dict(name="activate-train", kind="activate", rows=49152, hidden=1408, dtype="bf16",
             act="silu", gated=True),
    ]


def _log(rng, low, high):
    """A whole number between low and high, evenly spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _length(rng, low, high, whole):
    """A length, often a multiple of ``whole``."""
    n = _log(rng, low, high)
    return max(whole, n // whole * whole) if rng.random() < 0.6 else n


def draw(rng):
    kind = rng.choice(["layer", "layer", "pack", "product", "product", "saved", "activate"])
    half = rng.choice(["bf16", "bf16", "f16"])
    dtype = rng.choice([half, half, half, "f32"])
    act = rng.choice(["silu", "silu", "gelu", "relu"])
    if kind == "layer":
        experts = _log(rng, 2, 256)
        slots = rng.randint(1, min(8, experts))
        width, hidden = _length(rng, 64, 4096, 64), _length(rng, 64, 4096, 64)
        gated, packed = rng.random() < 0.7, rng.random() < 0.4
        experts = max(2, min(experts, 2 ** 30 // (width * hidden * (3 if gated else 2))))
        slots = min(slots, experts)
        return dict(kind=kind, tokens=_log(rng, 1, 64), experts=experts, slots=slots, width=width,
                    hidden=hidden, dtype=half if packed else dtype, order=rng.choice(["io", "oi"]),
                    act=act, gated=gated, packed=packed, sparse=rng.choice([0.0, 0.0, 1.2]))
    if kind == "pack":
        length, rows = _length(rng, 1, 8192, 32), _length(rng, 1, 65536, 8)
        rows = max(1, min(rows, 2 ** 26 // length))
        return dict(kind=kind, shape0=max(1, min(_log(rng, 1, 64), 2 ** 26 // (rows * length))),
                    rows=rows, length=length, dtype=dtype, to=rng.choice(["fp4", "int8"]),
                    order=rng.choice(["rows", "columns"]))
    if kind == "activate":
        hidden, rows = _length(rng, 1, 8192, 32), _log(rng, 1, 65536)
        return dict(kind=kind, rows=max(1, min(rows, 2 ** 26 // hidden)), hidden=hidden,
                    dtype=dtype, act=act, gated=rng.random() < 0.7)
    inner, outer = _length(rng, 64, 4096, 64), _length(rng, 64, 4096, 64)
    experts = max(2, min(_log(rng, 2, 128), 2 ** 27 // (inner * outer)))
    rows = _log(rng, 1, 32768)
    # no more than a sixth of the largest case's operations in single precision
    most = 2 ** (35 if kind == "saved" and dtype == "f32" else 37)
    rows = max(1, min(rows, most // (inner * outer)))
    used = rng.choice([1.0, 1.0, 0.8])
    if kind == "saved":
        return dict(kind=kind, rows=rows, used=used, experts=experts, inner=inner, outer=outer,
                    dtype=dtype, order=rng.choice(["io", "oi"]))
    both = rng.random() < 0.4
    return dict(kind=kind, rows=rows, used=used, experts=experts, inner=inner, outer=outer,
                dtype=half, both=both, train=not both and rng.random() < 0.4)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _normal(generator, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=generator, device=DEVICE, dtype=dtype).mul_(scale)


def _microscaled(values):
    """A plan's weights: ``values`` (rows, length) to codes (rows, 16 bytes to a block, the earlier
    element in the lower half) and scales (rows, blocks filled up to a multiple of 4)."""
    rows, length = values.shape
    blocks = -(-length // BLOCK)
    x = torch.zeros((rows, blocks * BLOCK), dtype=torch.float32, device=DEVICE)
    x[:, :length] = values
    x = x.view(rows, blocks, BLOCK)
    _, exponent = torch.frexp(x.abs().amax(2))
    s = (exponent - 3).clamp_min(-127)
    a = (x.abs() * torch.exp2(-s.float())[:, :, None]).clamp_max(6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = torch.round(a / step) * step
    # the 8 magnitudes' numbers: 0 .5 1 1.5 2 3 4 6
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code += 8 * torch.signbit(x).to(torch.uint8)
    code = code.view(rows, blocks * BLOCK // 2, 2)
    scales = torch.zeros((rows, -(-blocks // 4) * 4), dtype=torch.uint8, device=DEVICE)
    scales[:, :blocks] = (s + 127).to(torch.uint8)
    return code[:, :, 0] | (code[:, :, 1] << 4), scales


def _packed_weight(generator, experts, inner, outer):
    """(codes, scales) of a weight (experts, inner, outer), blocks along inner."""
    parts = [_microscaled(_normal(generator, (outer, inner), torch.float32, 1.0 / math.sqrt(inner)))
             for _ in range(experts)]
    return tuple(torch.stack([p[i] for p in parts]) for i in range(2))


def _dense_weight(generator, experts, inner, outer, dtype, order):
    shape = (experts, inner, outer) if order == "io" else (experts, outer, inner)
    w = _normal(generator, shape, dtype, 1.0 / math.sqrt(inner))
    return w if order == "io" else w.transpose(1, 2)


def _offsets(rng, case):
    e = case["experts"]
    share = rng.lognormal(0.0, 0.4, e)
    counts = rng.multinomial(max(1, int(case["rows"] * case["used"])), share / share.sum())
    return torch.as_tensor(np.concatenate(([0], np.cumsum(counts))).astype(np.int32), device=DEVICE)


def prepare(case, seed):
    rng = np.random.default_rng([seed, 17])
    generator = torch.Generator(device=DEVICE).manual_seed(int(rng.integers(1 << 60)))
    dtype, kind = DTYPES[case["dtype"]], case["kind"]
    state = dict(case=case, kind=kind)
    if kind == "layer":
        n, e, h = case["tokens"], case["experts"], case["hidden"]
        score = _normal(generator, (n, e), torch.float32)
        score += torch.as_tensor(rng.normal(0.0, 0.3, e), dtype=torch.float32, device=DEVICE)
        weights = torch.softmax(score, 1)
        if case["sparse"]:  # positive for any number of experts; none at all for some tokens
            chance = torch.rand((n, e), generator=generator, device=DEVICE)
            weights = weights * (chance < case["sparse"] * case["slots"] / e)
            weights = weights / weights.sum(1, keepdim=True).clamp_min(1e-30)
        state.update(weights=weights, x=_normal(generator, (n, case["width"]), dtype))
        first = 2 * h if case["gated"] else h
        if case["packed"]:
            state["inner"] = _packed_weight(generator, e, case["width"], first)
            state["outer"] = _packed_weight(generator, e, h, case["width"])
        else:
            state["inner"] = _dense_weight(generator, e, case["width"], first, dtype, case["order"])
            state["outer"] = _dense_weight(generator, e, h, case["width"], dtype, case["order"])
        return state
    if kind == "pack":
        g, r, k = case["shape0"], case["rows"], case["length"]
        x = _normal(generator, (g, r, k) if case["order"] == "rows" else (g, k, r), dtype)
        # rows differ in size, and an element in a thousand is far from the others
        x *= torch.exp(_normal(generator, (x.shape[0], x.shape[1], 1), torch.float32)).to(dtype)
        x *= torch.where(torch.rand(x.shape, generator=generator, device=DEVICE) < 1e-3, 16, 1).to(dtype)
        state["x"] = x
        return state
    if kind == "activate":
        p, h = case["rows"], case["hidden"]
        state["rows"] = _normal(generator, (p, 2 * h if case["gated"] else h), dtype, 1.5).requires_grad_()
        state["cot"] = _normal(generator, (p, h), dtype)
        return state
    p, e, k, n = case["rows"], case["experts"], case["inner"], case["outer"]
    state.update(offsets=_offsets(rng, case), rows=_normal(generator, (p, k), dtype))
    if kind == "product":
        state["weight"] = _packed_weight(generator, e, k, n)
        state["rows"].requires_grad_(case["train"])
    else:
        state["weight"] = _dense_weight(generator, e, k, n, dtype, case["order"]).requires_grad_()
        state["rows"].requires_grad_()
    if kind == "saved" or case["train"]:
        state["cot"] = _normal(generator, (p, n), dtype)
    return state


# ---------------------------------------------------------------------------
# the plain forms: elementary operations in 32 bits
# ---------------------------------------------------------------------------


def _values(x, to):
    """What the microscaled numbers of x stand for, blocks along the last dimension; 32 bits."""
    length = x.shape[-1]
    blocks = -(-length // BLOCK)
    full = torch.zeros((*x.shape[:-1], blocks * BLOCK), dtype=torch.float32, device=x.device)
    full[..., :length] = x
    full = full.view(*x.shape[:-1], blocks, BLOCK)
    _, exponent = torch.frexp(full.abs().amax(-1, keepdim=True))
    s = (exponent - (3 if to == "fp4" else 1)).clamp_min(-127).double()
    y = full.double() * torch.exp2(-s)
    if to == "fp4":
        a = y.abs().clamp_max(6.0)
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
        y = torch.copysign(torch.round(a / step) * step, y)
    else:
        y = torch.round(y * 64).clamp(-127, 127) / 64
    return (y * torch.exp2(s)).float().flatten(-2)[..., :length]


def _unpacked(weight, length):
    """(experts, outer, inner) in 32 bits from codes and scales."""
    codes, scales = weight
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6],
                         device=codes.device)
    value = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1).flatten(-2)
    blocks = codes.shape[-1] // 16
    scale = torch.exp2(scales[..., :blocks].float() - 127.0)
    return (value.view(*codes.shape[:-1], blocks, BLOCK) * scale[..., None]).flatten(-2)[..., :length]


def _act(u, act):
    if act == "relu":
        return u * (u > 0)
    if act == "silu":
        return u / (1 + torch.exp(-u))
    return u * 0.5 * (1 + torch.erf(u * math.sqrt(0.5)))


def _act_slope(u, act):
    if act == "relu":
        return (u > 0).to(u.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-u))
        return s * (1 + u * (1 - s))
    return 0.5 * (1 + torch.erf(u * math.sqrt(0.5))) + u * torch.exp(-0.5 * u * u) / math.sqrt(2 * math.pi)


def _plain_layer(state):
    case, weights, x = state["case"], state["weights"], state["x"].float()
    best, index = torch.sort(weights, dim=1, descending=True, stable=True)
    best, index = best[:, :case["slots"]], index[:, :case["slots"]]
    chosen = torch.zeros_like(weights).scatter_(1, index, torch.where(best > 0, best, 0.0))
    if case["packed"]:
        w_in = _unpacked(state["inner"], case["width"]).transpose(1, 2)
        w_out = _unpacked(state["outer"], case["hidden"]).transpose(1, 2)
    else:
        w_in, w_out = state["inner"].float(), state["outer"].float()
    u = torch.bmm(x.expand(case["experts"], *x.shape).contiguous(), w_in.contiguous())
    if case["gated"]:
        h = _act(u[:, :, :case["hidden"]], case["act"]) * u[:, :, case["hidden"]:]
    else:
        h = _act(u, case["act"])
    y = torch.bmm(h, w_out.contiguous())
    taken = chosen.T[:, :, None]
    return torch.where(taken > 0, y * taken, 0.0).sum(0).to(state["x"].dtype)


def _blocks(offsets, rows):
    """Every expert's rows, filled up to the most that one has: indexes and which are filled."""
    offsets = offsets.long()
    counts = offsets[1:] - offsets[:-1]
    along = torch.arange(int(counts.max()), device=rows.device)
    valid = along < counts[:, None]
    return torch.where(valid, offsets[:-1, None] + along, 0), valid


def _plain_product(state):
    case, dtype, saved = state["case"], state["rows"].dtype, state["kind"] == "saved"
    rows = state["rows"].detach().float()
    if saved:
        weight = state["weight"].detach().float()
    else:
        weight = _unpacked(state["weight"], case["inner"]).transpose(1, 2)
        rows = _values(rows, "fp4") if case["both"] else rows
    at, valid = _blocks(state["offsets"], rows)
    out = torch.zeros((rows.shape[0], weight.shape[2]), device=rows.device)
    blocks = torch.where(valid[:, :, None], rows[at], 0.0)
    out[at[valid]] = torch.bmm(blocks, weight.contiguous())[valid]
    got = dict(out=out.to(dtype))
    if saved or case["train"]:
        cot = torch.where(valid[:, :, None], state["cot"].float()[at], 0.0)
        g_rows = torch.zeros_like(rows)
        g_rows[at[valid]] = torch.bmm(cot, weight.transpose(1, 2).contiguous())[valid]
        got["g_rows"] = g_rows.to(dtype)
    if saved:
        kept = torch.where(valid[:, :, None], _values(rows, "int8")[at], 0.0)
        got["g_weight"] = torch.bmm(kept.transpose(1, 2).contiguous(), cot).to(dtype)
    return got


def _plain_activate(state):
    case, dtype, h = state["case"], state["rows"].dtype, state["case"]["hidden"]
    u, cot = state["rows"].detach().float(), state["cot"].float()
    if not case["gated"]:
        kept = _values(u, "int8")
        return dict(out=_act(u, case["act"]).to(dtype),
                    g_rows=(_act_slope(kept, case["act"]) * cot).to(dtype))
    gate, value = _values(u[:, :h], "int8"), _values(u[:, h:], "int8")
    g_rows = torch.cat((_act_slope(gate, case["act"]) * value * cot, _act(gate, case["act"]) * cot), 1)
    return dict(out=(_act(u[:, :h], case["act"]) * u[:, h:]).to(dtype), g_rows=g_rows.to(dtype))


def _plain_pack(state):
    x = state["x"] if state["case"]["order"] == "rows" else state["x"].transpose(1, 2)
    y = _values(x.float(), state["case"]["to"]).to(x.dtype)
    return y if state["case"]["order"] == "rows" else y.transpose(1, 2)


# ---------------------------------------------------------------------------
# the call
# ---------------------------------------------------------------------------


def run(state):
    kind, case = state["kind"], state["case"]
    if not own:
        return dict(layer=_plain_layer, pack=_plain_pack, product=_plain_product,
                    saved=_plain_product, activate=_plain_activate)[kind](state)
    import purin_amd as pa

    def packed(weight, inner):
        codes, scales = weight
        return pa.Microscaled(codes=codes, scales=scales, kind="fp4",
                              shape=(codes.shape[0], inner, codes.shape[1]), axis=1,
                              dtype=DTYPES[case["dtype"]])

    if kind == "layer":
        inner, outer = state["inner"], state["outer"]
        if case["packed"]:
            inner, outer = packed(inner, case["width"]), packed(outer, case["hidden"])
        return pa.expert_layer(state["x"], state["weights"], case["slots"], inner, outer, case["act"])
    if kind == "pack":
        return pa.unpack(pa.pack(state["x"], case["to"], axis=2 if case["order"] == "rows" else 1))
    if kind == "activate":
        out = pa.activate(state["rows"], case["act"], gated=case["gated"], saved="int8")
        (g_rows,) = torch.autograd.grad(out, state["rows"], state["cot"])
        return dict(out=out, g_rows=g_rows)
    if kind == "product":
        rows = pa.pack(state["rows"], "fp4") if case["both"] else state["rows"]
        out = pa.expert_product(rows, packed(state["weight"], case["inner"]), state["offsets"])
        if not case["train"]:
            return dict(out=out)
        (g_rows,) = torch.autograd.grad(out, state["rows"], state["cot"])
        return dict(out=out, g_rows=g_rows)
    out = pa.expert_product(state["rows"], state["weight"], state["offsets"], saved="int8")
    g_rows, g_weight = torch.autograd.grad(out, (state["rows"], state["weight"]), state["cot"])
    return dict(out=out, g_rows=g_rows, g_weight=g_weight)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    b, kind = SIZES[case["dtype"]], case["kind"]
    if kind == "layer":
        n, e, h, w = case["tokens"], case["experts"], case["hidden"], case["width"]
        share = case["slots"] / e * (0.9 if case["sparse"] else 1.0)
        columns = 3 * h if case["gated"] else 2 * h
        # the experts that some token has, where tokens choose apart from each other
        busy = e * (1.0 - (1.0 - share) ** n)
        each = 17 / 32 if case["packed"] else b
        return {"bytes": busy * w * columns * each + 2 * n * w * b + n * e * 4,
                "flops": 2.0 * n * share * e * w * columns}
    if kind == "pack":
        count = case["shape0"] * case["rows"] * case["length"]
        held = count * (17 / 32 if case["to"] == "fp4" else 33 / 32)
        return {"bytes": 2.0 * (count * b + held), "flops": 4.0 * count}
    if kind == "activate":
        count, u = case["rows"] * case["hidden"], 2 if case["gated"] else 1
        return {"bytes": count * (2.0 * b * (u + 1) + 2 * u * 33 / 32), "flops": 20.0 * count}
    p, e, k, n = case["rows"], case["experts"], case["inner"], case["outer"]
    used = max(1, int(p * case["used"]))
    busy = e * (1.0 - (1.0 - 1.0 / e) ** used)
    if kind == "product":
        w = busy * k * n * 17 / 32
        whole, flops = used * k * b + p * n * b + w, 2.0 * used * k * n
        if case["both"]:
            whole += 2.0 * used * k * 17 / 32  # the packed rows, out and in
        if case["train"]:
            whole, flops = whole + used * n * b + p * k * b + w, 2.0 * flops
        return {"bytes": whole, "flops": flops}
    whole = (used * k + p * n + busy * k * n) * b  # forward
    whole += (used * n + p * k + busy * k * n) * b  # the rows' gradient
    whole += used * n * b + 2.0 * used * k * 33 / 32 + e * k * n * b  # the weights', from 8 bits
    return {"bytes": whole, "flops": 6.0 * used * k * n}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

FP4 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _exact_values(x, to):
    """x (rows, length) in 64 bits to what its blocks of 32 stand for."""
    rows, length = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -length % BLOCK)).reshape(-1, BLOCK)
    most = x.abs().max(1).values
    power = torch.floor(torch.log2(most.clamp_min(2.0 ** -140)))
    # next to a power of two the logarithm may be off by one
    power = torch.where(torch.exp2(power) > most, power - 1, power)
    power = torch.where(torch.exp2(power + 1) <= most, power + 1, power)
    power = torch.clamp_min(power - (2 if to == "fp4" else 0), -127.0)
    y = x * torch.exp2(-power)[:, None]
    if to == "fp4":
        grid = torch.tensor(FP4, dtype=torch.float64, device=x.device)
        border = (grid[1:] + grid[:-1]) / 2
        low = torch.bucketize(y.abs(), border, right=False)  # a border itself falls to the lower one
        high = torch.bucketize(y.abs(), border, right=True)
        pick = torch.where(low % 2 == 0, low, high)  # of two, the even one
        y = torch.where(y < 0, -1.0, 1.0) * grid[pick]
    else:
        whole = torch.floor(y * 64)
        rest = y * 64 - whole
        up = (rest > 0.5) | ((rest == 0.5) & (whole % 2 == 1))
        y = torch.clamp(whole + up, -127, 127) / 64
    return (y * torch.exp2(power)[:, None]).view(rows, -1)[:, :length]


def _exact_weight(weight, e, inner):
    """Expert e's matrix (inner, outer) of codes and scales."""
    codes, scales = weight[0][e], weight[1][e]
    outer, blocks = codes.shape[0], codes.shape[1] // 16
    grid = torch.tensor(FP4, dtype=torch.float64, device=codes.device)
    w = torch.zeros((outer, blocks * BLOCK), dtype=torch.float64, device=codes.device)
    for part in range(2):
        c = (codes >> (4 * part)).long() % 16
        w[:, part::2] = grid[c % 8] * (1.0 - 2.0 * (c // 8))
    w *= torch.repeat_interleave(2.0 ** (scales[:, :blocks].double() - 127.0), BLOCK, 1)
    return w[:, :inner].T


def _exact_act(u, act):
    if act == "relu":
        return torch.clamp_min(u, 0.0), torch.where(u > 0, 1.0, 0.0).double()
    if act == "silu":
        s = torch.sigmoid(u)
        return u * s, s + u * s * (1 - s)
    normal = 0.5 * torch.erfc(-u / math.sqrt(2.0))
    return u * normal, normal + u * torch.exp(-u * u / 2) / math.sqrt(2 * math.pi)


def exact(case, seed):
    state, kind = prepare(case, seed), case["kind"]
    if kind == "pack":
        x = state["x"] if case["order"] == "rows" else state["x"].transpose(1, 2)
        y = torch.stack([_exact_values(part, case["to"]) for part in x])
        return y if case["order"] == "rows" else y.transpose(1, 2)
    if kind == "layer":
        return _exact_layer(state)
    if kind == "activate":
        u, cot, h = state["rows"].detach().double(), state["cot"].double(), case["hidden"]
        if not case["gated"]:
            return dict(out=_exact_act(u, case["act"])[0],
                        g_rows=cot * _exact_act(_exact_values(u, "int8"), case["act"])[1])
        gate, value = u[:, :h], u[:, h:]
        f, slope = _exact_act(_exact_values(gate, "int8"), case["act"])
        return dict(out=_exact_act(gate, case["act"])[0] * value,
                    g_rows=torch.cat((slope * cot * _exact_values(value, "int8"), f * cot), 1))
    rows, offsets = state["rows"].detach().double(), state["offsets"].tolist()
    if kind == "product" and case["both"]:
        rows = _exact_values(rows, "fp4")
    zeros = lambda *shape: torch.zeros(shape, dtype=torch.float64, device=DEVICE)  # noqa: E731
    got = dict(out=zeros(rows.shape[0], case["outer"]))
    if "cot" in state:
        got["g_rows"] = zeros(*rows.shape)
    if kind == "saved":
        kept = _exact_values(rows, "int8")
        got["g_weight"] = zeros(case["experts"], case["inner"], case["outer"])
    for e, (a, z) in enumerate(zip(offsets, offsets[1:])):
        if a == z:
            continue
        w = (state["weight"][e].detach().double() if kind == "saved"
             else _exact_weight(state["weight"], e, case["inner"]))
        got["out"][a:z] = rows[a:z] @ w
        if "cot" in state:
            g = state["cot"][a:z].double()
            got["g_rows"][a:z] = g @ w.T
            if kind == "saved":
                got["g_weight"][e] = kept[a:z].T @ g
    return got


def _exact_layer(state):
    case, x = state["case"], state["x"].double()
    w = state["weights"].cpu().numpy()
    index = np.argsort(-w, axis=1, kind="stable")[:, :case["slots"]]
    taken = np.zeros(w.shape, bool)
    np.put_along_axis(taken, index, True, 1)
    taken &= w > 0
    out = torch.zeros((case["tokens"], case["width"]), dtype=torch.float64, device=DEVICE)
    for e in np.flatnonzero(taken.any(0)):
        t = torch.as_tensor(np.flatnonzero(taken[:, e]), device=DEVICE)
        if case["packed"]:
            w_in = _exact_weight(state["inner"], e, case["width"])
            w_out = _exact_weight(state["outer"], e, case["hidden"])
        else:
            w_in, w_out = state["inner"][e].double(), state["outer"][e].double()
        u = x[t] @ w_in
        h = _exact_act(u[:, :case["hidden"]], case["act"])[0]
        if case["gated"]:
            h = h * u[:, case["hidden"]:]
        out[t] += state["weights"][t, int(e)].double()[:, None] * (h @ w_out)
    return out
