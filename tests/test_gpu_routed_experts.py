"""The example that runs the operators together with a projection layer."""

import numpy as np
import pytest

from tests._gpu import require_gpu

pytestmark = pytest.mark.gpu


def test_training_brings_the_loss_down():
    torch = require_gpu()
    from examples.routed_experts import train

    losses, norms, model = train(steps=40, log=None)
    print([round(float(v), 3) for v in losses[::8]], flush=True)
    assert torch.isfinite(losses).all() and torch.isfinite(norms).all()
    assert float(losses[-5:].mean()) < 0.7 * float(losses[:3].mean())


def test_the_layer_against_a_dense_one():
    """Output and gradients in f64 against every expert on every token, weighted: the weights
    are on the polytope, most are exactly zero, and slots for all of them lose nothing."""
    torch = require_gpu()
    from examples.routed_experts import RoutedExperts

    torch.manual_seed(1)
    group, groups, experts, width = 12, 5, 6, 10
    model = RoutedExperts(width, 16, experts, group, groups, experts, dtype=torch.float64)
    x = torch.randn(group * groups, width, device="cuda", dtype=torch.float64)
    w = model.weights(x).detach()
    # the layer's tolerance (1e-9) on the rows; bounds hold exactly
    assert (w >= 0).all() and float((w.sum(1) - 1).abs().max()) < 1e-7
    load = w.view(groups, group, experts).sum(1)
    assert float(load.max()) <= 1.25 * group / experts + 1e-7
    assert float((w == 0).double().mean()) > 0.3
    parameters = list(model.parameters())
    cot = torch.randn_like(x)

    def dense():
        w = model.weights(x)
        h = torch.relu(torch.matmul(x[None], model.inner))
        return (torch.matmul(h, model.outer) * w.T[:, :, None]).sum(0)

    out, want = model(x), dense()
    got_g = torch.autograd.grad(out, parameters, cot)
    want_g = torch.autograd.grad(want, parameters, cot)
    assert float((out - want).abs().max()) < 1e-12
    # the experts' gradients are the same sums; the router's pass the same implicit VJP, solved
    # to 1e-9, with a gradient of zero instead of any at the weights that are zero: the VJP of a
    # projection ignores what stays at its bound
    for name, a, b in zip(("router", "inner", "outer"), got_g, want_g):
        scale = float(b.abs().max())
        tol = 1e-5 if name == "router" else 1e-12
        assert float((a - b).abs().max()) <= tol * max(scale, 1.0), name
