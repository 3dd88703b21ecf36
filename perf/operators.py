"""The operators around a projection layer in a network of experts, as a user's program calls them.

Three kinds of call:

* ``tokens``: from a token's weights over the experts (a projection onto a routing polytope
  leaves most of them exactly zero; a softmax leaves none) to its experts, the tokens' rows
  sorted by expert, and the experts' rows back with the weights applied; forward, or forward and
  backward (``train``) with gradients for the tokens, the weights and the experts' rows;
* ``experts``: the experts' products on rows sorted by expert, forward, or forward and backward;
* ``clip``: the global norm of a list of gradients, and the gradients scaled to a largest norm,
  into the buffers that an optimizer reads.

With ``own`` false ``run`` computes them from elementary torch operations in 32 bits.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}

# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # one token of a served request: latency is all that counts
        dict(name="tokens-one", kind="tokens", tokens=1, experts=64, slots=8, width=2048,
             dtype="bf16", sparse=0.0, train=False),
        # a served batch, one token for each request, softmax weights
        dict(name="tokens-serve", kind="tokens", tokens=192, experts=32, slots=4, width=4096,
             dtype="bf16", sparse=0.0, train=False),
        # odd sizes in single precision: projected weights, so that a token has any number of
        # experts up to the slots, some tokens (padding) none
        dict(name="tokens-odd", kind="tokens", tokens=4099, experts=23, slots=3, width=1111,
             dtype="f32", sparse=1.2, train=True),
        # an ordinary training step on projected weights
        dict(name="tokens-train", kind="tokens", tokens=8192, experts=64, slots=6, width=2048,
             dtype="bf16", sparse=1.5, train=True),
        # the largest training step: long rows, many tokens, softmax weights
        dict(name="tokens-large", kind="tokens", tokens=32768, experts=128, slots=4, width=4096,
             dtype="bf16", sparse=0.0, train=True),
        # one token's experts: every weight is read for one row
        dict(name="experts-one", kind="experts", rows=8, used=1.0, experts=64, inner=2048,
             outer=1408, dtype="bf16", order="oi", train=False),
        # the products of a served batch: a few rows to an expert
        dict(name="experts-serve", kind="experts", rows=768, used=1.0, experts=32, inner=4096,
             outer=1536, dtype="bf16", order="io", train=False),
        # odd sizes in single precision, with slots left empty at the end
        dict(name="experts-odd", kind="experts", rows=3001, used=0.9, experts=7, inner=515,
             outer=777, dtype="f32", order="io", train=True),
        # an ordinary training step's products, forward and both gradients
        dict(name="experts-train", kind="experts", rows=32768, used=1.0, experts=16, inner=2048,
             outer=4096, dtype="bf16", order="io", train=True),
        # a small network's gradients: a handful of small tensors, launches are all that counts
        dict(name="clip-small", kind="clip", tensors=14, elements=50_000, dtype="f32", bias=0.5,
             largest=1.0),
        # unequal and odd tensors of a half-precision network, from one element up
        dict(name="clip-odd", kind="clip", tensors=77, elements=20_000_001, dtype="f16", bias=0.5,
             largest=1.0),
        # the gradients of a large network
        dict(name="clip-large", kind="clip", tensors=290, elements=1_000_000_000, dtype="bf16",
             bias=0.6, largest=1.0),
    ]


def _log(rng, low, high):
    """A whole number between low and high, evenly spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["tokens", "tokens", "experts", "experts", "clip"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "clip":
        return dict(kind="clip", tensors=_log(rng, 1, 300), elements=_log(rng, 1000, 500_000_000),
                    dtype=dtype, bias=rng.uniform(0.1, 0.9), largest=rng.choice([0.1, 1.0, 5.0]))
    train = rng.random() < 0.6
    experts = _log(rng, 2, 256)
    slots = rng.randint(1, min(8, experts))
    if kind == "tokens":
        width = _log(rng, 16, 4096)
        if rng.random() < 0.6:
            width = max(8, width // 8 * 8)
        tokens = _log(rng, 1, 32768)
        tokens = max(1, min(tokens, 2 ** 28 // (width * slots)))
        sparse = rng.choice([0.0, 0.8, 1.2, 2.0]) if tokens >= 16 else 0.0
        return dict(kind="tokens", tokens=tokens, experts=experts, slots=slots, width=width,
                    dtype=dtype, sparse=sparse, train=train)
    inner, outer = _log(rng, 64, 4096), _log(rng, 64, 4096)
    if rng.random() < 0.7:
        inner, outer = max(64, inner // 64 * 64), max(64, outer // 64 * 64)
    experts = max(2, min(experts, 2 ** 28 // (inner * outer)))
    rows = _log(rng, 1, 32768)
    # no more than a sixth of the largest case's operations in single precision
    most = 2 ** (35 if dtype == "f32" else 37)
    rows = max(1, min(rows, most // (inner * outer)))
    return dict(kind="experts", rows=rows, used=rng.choice([1.0, 1.0, 0.8]), experts=experts,
                inner=inner, outer=outer, dtype=dtype, order=rng.choice(["io", "oi"]), train=train)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _normal(generator, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=generator, device=DEVICE, dtype=dtype).mul_(scale)


def _share(case):
    """The chance that an entry of the projected weights is positive."""
    return min(1.0, case["sparse"] * case["slots"] / case["experts"])


def _sizes(case):
    """The element counts of the gradients, one network's at every seed: a few large ones, many
    small (their logarithms spread as ``bias`` says), one element at least, ``elements`` in all."""
    rng = np.random.default_rng([case["tensors"], case["elements"]])
    share = rng.lognormal(0.0, 3.0 * case["bias"], case["tensors"])
    sizes = np.maximum(1, (share / share.sum() * case["elements"]).astype(np.int64))
    sizes[np.argmax(sizes)] += max(0, case["elements"] - sizes.sum())
    return sizes


def prepare(case, seed):
    rng = np.random.default_rng([seed, 91])
    generator = torch.Generator(device=DEVICE).manual_seed(int(rng.integers(1 << 60)))
    dtype = DTYPES[case["dtype"]]
    kind = case["kind"]
    if kind == "tokens":
        n, e, k, h = case["tokens"], case["experts"], case["slots"], case["width"]
        score = _normal(generator, (n, e), torch.float32)
        score += torch.as_tensor(rng.normal(0.0, 0.3, e), dtype=torch.float32, device=DEVICE)
        weights = torch.softmax(score, 1)
        if case["sparse"]:
            # positive for any number of experts; none at all for the padding tokens
            chance = torch.rand((n, e), generator=generator, device=DEVICE)
            weights = weights * (chance < _share(case))
            weights = weights / weights.sum(1, keepdim=True).clamp_min(1e-30)
            weights[torch.rand((n,), generator=generator, device=DEVICE) < 0.02] = 0.0
        train = case["train"]
        state = dict(kind=kind, train=train, slots=k, weights=weights.requires_grad_(train),
                     x=_normal(generator, (n, h), dtype).requires_grad_(train),
                     y=_normal(generator, (n * k, h), dtype).requires_grad_(train))
        if train:
            state["cot_rows"] = _normal(generator, (n * k, h), dtype)
            state["cot_out"] = _normal(generator, (n, h), dtype)
        return state
    if kind == "experts":
        p, e = case["rows"], case["experts"]
        share = rng.lognormal(0.0, 0.4, e)
        used = max(1, int(p * case["used"]))
        counts = rng.multinomial(used, share / share.sum())
        offsets = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
        k, n = case["inner"], case["outer"]
        shape = (e, k, n) if case["order"] == "io" else (e, n, k)
        weight = _normal(generator, shape, dtype, 1.0 / math.sqrt(k))
        weight = weight if case["order"] == "io" else weight.transpose(1, 2)
        train = case["train"]
        state = dict(kind=kind, train=train, offsets=torch.as_tensor(offsets, device=DEVICE),
                     rows=_normal(generator, (p, k), dtype).requires_grad_(train),
                     weight=weight.requires_grad_(train))
        if train:
            state["cot"] = _normal(generator, (p, n), dtype)
        return state
    sizes = _sizes(case)
    scale = rng.lognormal(-2.0, 1.0, sizes.size)
    gradients = [_normal(generator, (int(s),), dtype, float(c)) for s, c in zip(sizes, scale)]
    # the optimizer's gradient buffer: one allocation, each tensor's part at 16 bytes
    step = 16 // SIZES[case["dtype"]]
    ends = np.cumsum(-(-sizes // step) * step)
    flat = torch.zeros(int(ends[-1]), dtype=dtype, device=DEVICE)
    starts = np.concatenate(([0], ends[:-1]))
    out = [flat[a:a + s] for a, s in zip(starts.tolist(), sizes.tolist())]
    return dict(kind=kind, gradients=gradients, out=out, flat=flat, largest=case["largest"])


# ---------------------------------------------------------------------------
# the plain forms: elementary operations in 32 bits
# ---------------------------------------------------------------------------


def _plain_tokens(state):
    weights, x, y, k = state["weights"].detach(), state["x"].detach(), state["y"].detach(), state["slots"]
    n, e = weights.shape
    dtype, p = x.dtype, n * k
    # a token's largest positive weights, ties to the lowest expert
    best, index = torch.sort(weights, dim=1, descending=True, stable=True)
    best, index = best[:, :k], index[:, :k]
    taken = best > 0
    chosen = torch.where(taken, best, 0.0)
    experts = torch.where(taken, index, -1)
    # pairs sorted by expert, in the tokens' order within each
    key = torch.where(taken, index, e).reshape(p)
    order = torch.sort(key, stable=True).indices
    counts = torch.zeros(e + 1, dtype=torch.int64, device=x.device).index_add_(
        0, key, torch.ones_like(key))
    offsets = torch.zeros(e + 1, dtype=torch.int64, device=x.device)
    offsets[1:] = torch.cumsum(counts[:e], 0)
    every = torch.arange(p, device=x.device)
    place = torch.zeros_like(every)
    place[order] = every
    place = torch.where(taken, place.reshape(n, k), -1)
    filled = every < offsets[e]
    source = torch.where(filled, order, -1)
    token = torch.where(filled, order // k, 0)
    rows = torch.where(filled[:, None], x[token], 0.0)
    at = place.clamp_min(0)
    picked = y.float()[at]
    out = (torch.where(taken[:, :, None], picked, 0.0) * chosen[:, :, None]).sum(1)
    got = dict(experts=experts.int(), weights=chosen, offsets=offsets.int(), place=place.int(),
               source=source.int(), rows=rows.to(dtype), out=out.to(dtype))
    if state["train"]:
        cot_rows, cot_out = state["cot_rows"].float(), state["cot_out"].float()
        got["g_x"] = torch.where(taken[:, :, None], cot_rows[at], 0.0).sum(1).to(dtype)
        factor = torch.where(filled, chosen.reshape(p)[order], 0.0)
        got["g_y"] = (cot_out[token] * factor[:, None]).to(dtype)
        along = torch.where(taken, (cot_out[:, None, :] * picked).sum(2), 0.0)
        got["g_weights"] = torch.zeros_like(weights).scatter_add_(1, index, along)
    return got


def _plain_experts(state):
    rows, weight, offsets = state["rows"].detach().float(), state["weight"].detach().float(), state["offsets"].long()
    dtype, p, n = state["rows"].dtype, rows.shape[0], weight.shape[2]
    counts = offsets[1:] - offsets[:-1]
    # every expert's rows, filled up with zeros to the most that one has
    along = torch.arange(int(counts.max()), device=rows.device)
    valid = along < counts[:, None]
    at = torch.where(valid, offsets[:-1, None] + along, 0)
    blocks = torch.where(valid[:, :, None], rows[at], 0.0)
    out = torch.zeros((p, n), device=rows.device)
    out[at[valid]] = torch.bmm(blocks, weight.contiguous())[valid]
    got = dict(out=out.to(dtype))
    if state["train"]:
        cot = torch.where(valid[:, :, None], state["cot"].float()[at], 0.0)
        g_rows = torch.zeros_like(rows)
        g_rows[at[valid]] = torch.bmm(cot, weight.transpose(1, 2).contiguous())[valid]
        got["g_rows"] = g_rows.to(dtype)
        got["g_weight"] = torch.bmm(blocks.transpose(1, 2).contiguous(), cot).to(dtype)
    return got


def _plain_clip(state):
    norm = torch.stack([g.float().square().sum() for g in state["gradients"]]).sum().sqrt()
    factor = torch.where(norm > state["largest"], state["largest"] / norm, 1.0)
    _ = [o.copy_(g.float() * factor) for o, g in zip(state["out"], state["gradients"])]
    return dict(norm=norm, flat=state["flat"])


# ---------------------------------------------------------------------------
# the call
# ---------------------------------------------------------------------------


def run(state):
    kind = state["kind"]
    if not own:
        return dict(tokens=_plain_tokens, experts=_plain_experts, clip=_plain_clip)[kind](state)
    import purin_amd as pa

    if kind == "tokens":
        routing = pa.route(state["weights"], state["slots"])
        rows = pa.dispatch(state["x"], routing)
        out = pa.combine(state["y"], routing)
        got = dict(experts=routing.experts, weights=routing.weights, offsets=routing.offsets,
                   place=routing.place, source=routing.source, rows=rows, out=out)
        if state["train"]:
            got["g_x"], got["g_weights"], got["g_y"] = torch.autograd.grad(
                (rows, out), (state["x"], state["weights"], state["y"]),
                (state["cot_rows"], state["cot_out"]))
        return got
    if kind == "experts":
        out = pa.expert_product(state["rows"], state["weight"], state["offsets"])
        if not state["train"]:
            return dict(out=out)
        g_rows, g_weight = torch.autograd.grad(out, (state["rows"], state["weight"]), state["cot"])
        return dict(out=out, g_rows=g_rows, g_weight=g_weight)
    norm = pa.clip_gradients(state["gradients"], state["largest"], out=state["out"])
    return dict(norm=norm, flat=state["flat"])


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    b = SIZES[case["dtype"]]
    if case["kind"] == "tokens":
        n, e, k, h = case["tokens"], case["experts"], case["slots"], case["width"]
        fill = 1.0
        if case["sparse"]:  # the mean share of the slots that positive weights fill
            p = _share(case)
            chance = [math.exp(math.lgamma(e + 1) - math.lgamma(i + 1) - math.lgamma(e - i + 1)
                               + i * math.log(max(p, 1e-300)) + (e - i) * math.log(max(1 - p, 1e-300)))
                      for i in range(e + 1)]
            fill = 0.98 * sum(min(i, k) * c for i, c in enumerate(chance)) / k
        used = n * k * fill
        # weights in; experts, chosen weights, places, sources and offsets out
        whole = n * e * 4 + n * k * 16 + (e + 1) * 4
        # tokens in, rows out; rows in, tokens out
        whole += n * h * b + n * k * h * b + used * h * b + n * h * b
        flops = 2.0 * used * h
        if case["train"]:
            # rows' gradients in, tokens' out; tokens' gradients and rows in, rows' out; weights' out
            whole += used * h * b + n * h * b + n * h * b + used * h * b + n * k * h * b + n * e * 4
            flops += 4.0 * used * h
        return {"bytes": float(whole), "flops": flops}
    if case["kind"] == "experts":
        p, e, k, n = case["rows"], case["experts"], case["inner"], case["outer"]
        used = max(1, int(p * case["used"]))
        # the experts that have a row, of rows that fall anywhere
        busy = e * (1.0 - (1.0 - 1.0 / e) ** used)
        whole, flops = (used * k + p * n + busy * k * n) * b, 2.0 * used * k * n
        if case["train"]:
            whole += (used * n + p * k + busy * k * n + used * (k + n) + e * k * n) * b
            flops *= 3.0
        return {"bytes": float(whole), "flops": flops}
    return {"bytes": 2.0 * b * case["elements"], "flops": 3.0 * case["elements"]}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "tokens":
        return _exact_tokens(state)
    if case["kind"] == "experts":
        rows, weight = state["rows"].detach(), state["weight"].detach()
        offsets = state["offsets"].tolist()
        got = dict(out=torch.zeros((rows.shape[0], weight.shape[2]), dtype=torch.float64, device=DEVICE))
        if state["train"]:
            got["g_rows"] = torch.zeros(rows.shape, dtype=torch.float64, device=DEVICE)
            got["g_weight"] = torch.zeros(weight.shape, dtype=torch.float64, device=DEVICE)
        for e, (a, z) in enumerate(zip(offsets, offsets[1:])):
            if a == z:
                continue
            w, r = weight[e].double(), rows[a:z].double()
            got["out"][a:z] = r @ w
            if state["train"]:
                g = state["cot"][a:z].double()
                got["g_rows"][a:z] = g @ w.T
                got["g_weight"][e] = r.T @ g
        return got
    total = sum(float(g.double().square().sum()) for g in state["gradients"])
    norm = math.sqrt(total)
    factor = min(1.0, state["largest"] / norm) if norm > 0 else 1.0
    flat = torch.zeros(state["flat"].shape, dtype=torch.float64, device=DEVICE)
    for o, g in zip(state["out"], state["gradients"]):
        at = o.storage_offset()
        flat[at:at + g.numel()] = g.double() * factor
    return dict(norm=torch.tensor(norm, dtype=torch.float64), flat=flat)


def _exact_tokens(state):
    k = state["slots"]
    w = state["weights"].detach().cpu().numpy()
    n, e = w.shape
    index = np.argsort(-w, axis=1, kind="stable")[:, :k]
    value = np.take_along_axis(w, index, 1)
    taken = value > 0
    token, slot = np.nonzero(taken)
    expert = index[token, slot]
    by = np.lexsort((slot, token, expert))
    place = np.full((n, k), -1)
    place[token[by], slot[by]] = np.arange(by.size)
    x, y = state["x"].detach().double(), state["y"].detach().double()
    h = x.shape[1]
    to = lambda a: torch.as_tensor(np.ascontiguousarray(a), device=DEVICE)  # noqa: E731
    rows = torch.zeros((n * k, h), dtype=torch.float64, device=DEVICE)
    rows[: by.size] = x[to(token[by])]
    chosen = to(np.where(taken, value, 0.0).astype(np.float64))
    out = torch.zeros((n, h), dtype=torch.float64, device=DEVICE)
    got = dict(experts=None, weights=chosen, offsets=None, place=None, source=None, rows=rows, out=out)
    if state["train"]:
        cot_rows, cot_out = state["cot_rows"].double(), state["cot_out"].double()
        g_x, g_y = torch.zeros_like(out), torch.zeros_like(rows)
        g_w = torch.zeros((n, e), dtype=torch.float64, device=DEVICE)
        got.update(g_x=g_x, g_y=g_y, g_weights=g_w)
    for j in range(k):
        t = to(np.nonzero(taken[:, j])[0])
        at = to(place[taken[:, j], j])
        out[t] += chosen[t, j, None] * y[at]
        if state["train"]:
            g_x[t] += cot_rows[at]
            g_y[at] = chosen[t, j, None] * cot_out[t]
            g_w[t, to(index[taken[:, j], j])] = (cot_out[t] * y[at]).sum(1)
    return got
