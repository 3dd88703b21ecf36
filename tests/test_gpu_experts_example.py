"""The example with rows kept in 8 bits, and its layer served from packed weights."""

import numpy as np
import pytest

from oracle import experts as oe
from tests._gpu import require_gpu
from tests.test_gpu_train import _np

pytestmark = pytest.mark.gpu


def test_gradients_with_kept_rows_and_the_served_layer():
    """One step's gradients beside those without, within what 8 bits leave.  The served layer against
    the oracle on the weights in 4 bits."""
    torch = require_gpu()
    from examples.routed_experts import RoutedExperts
    from purin_amd import unpack

    group, groups, experts, width, hidden = 12, 5, 6, 40, 64
    torch.manual_seed(1)
    model = RoutedExperts(width, hidden, experts, group, groups, 3)
    x = torch.randn(group * groups, width, device="cuda")
    cot = torch.randn_like(x)
    plain = torch.autograd.grad(model(x), list(model.parameters()), cot)
    model.saved = "int8"
    kept = torch.autograd.grad(model(x), list(model.parameters()), cot)
    for a, b in zip(plain, kept):
        assert a.shape == b.shape and bool(torch.isfinite(b).all())
        # A relu's slope is lost where 0 < u < half a step.  With a block's largest below 4 root mean
        # squares the step is 2^-5 of one, and of normal u that are positive 2^-6 * 0.4 / 0.5 =
        # 1.25 % are lost: sqrt(0.0125) = 0.112 of the gradient's norm.  A row's elements are off by
        # at most 2^-6 root mean squares themselves, 2^-5 together with the second product's.
        assert float((a - b).norm()) <= (0.112 + 2.0 ** -5) * float(a.norm())
    with torch.no_grad():
        weights, packed = model.weights(x)[:8], model.packed()
    out = model.serve(x[:8], weights, packed)
    values = [_np(unpack(m)) for m in packed]
    rows = _np(x[:8].bfloat16())
    want, terms = oe.layer(rows, _np(weights), 3, *values, "relu")
    bound = 2.0 ** -8 * np.abs(want) + (2 * (width + hidden + 4) * 2.0 ** -24 + 2.0 ** -15) * terms
    assert (np.abs(_np(out) - want) <= bound + 2.0 ** -126).all()
