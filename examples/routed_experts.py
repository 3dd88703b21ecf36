"""A layer of experts whose routing weights are a projection, trained for a few steps.

The router's scores of a group of tokens are projected onto the routing polytope: a token's
weights are not negative and sum to one, and no expert takes more than its share of the group.
The projection leaves most weights exactly zero; the tokens with a weight for an expert go to it
and back, and the gradients of the weights go on through the projection's implicit VJP to the
router.  The gradients' global norm is limited before the step.

    python examples/routed_experts.py [--steps N]
"""

from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from purin_amd import (ChambollePockConfig, clip_gradients, combine, dispatch,  # noqa: E402
                       expert_product, prepare_projection, route)
from purin_amd.problems import CanonicalRows  # noqa: E402


def routing_polytope(tokens, experts, capacity):
    """The rows of one group: weights (tokens, experts) flattened, token-major.  Equalities: a
    token's weights sum to one; inequalities: an expert's load is at most ``capacity``, and every
    weight is at least zero (one-entry rows, which the layer takes as bounds)."""
    n = tokens * experts
    index = np.arange(n).reshape(tokens, experts)
    columns = np.concatenate((index.ravel(), index.T.ravel(), np.arange(n)))
    lengths = np.concatenate((np.full(tokens, experts), np.full(experts, tokens), np.ones(n, int)))
    values = np.concatenate((np.ones(2 * n), -np.ones(n)))
    rhs = np.concatenate((np.ones(tokens), np.full(experts, float(capacity)), np.zeros(n)))
    indptr = np.concatenate(([0], np.cumsum(lengths)))
    return CanonicalRows(n, tokens, experts + n, 0, indptr, columns.astype(np.int32), values, rhs,
                         np.zeros((rhs.size, 0)))


class RoutedExperts(torch.nn.Module):
    """Two matrices to an expert; ``group`` tokens share each expert's capacity."""

    def __init__(self, width, hidden, experts, group, groups, slots, slack=1.25,
                 dtype=torch.float32):
        super().__init__()
        self.experts, self.slots = experts, slots
        rows = routing_polytope(group, experts, slack * group / experts)
        self.layer = prepare_projection(
            rows, batch_size=groups, dtype=dtype,
            config=ChambollePockConfig(tolerance=1e-5 if dtype == torch.float32 else 1e-9,
                                       max_iterations=5000))
        make = lambda *shape: torch.nn.Parameter(  # noqa: E731
            torch.randn(shape, device="cuda", dtype=dtype) / shape[-2] ** 0.5)
        self.router = make(width, experts)
        self.inner = make(experts, width, hidden)
        self.outer = make(experts, hidden, width)

    def weights(self, x):
        """The routing weights (tokens, experts)."""
        return self.layer((x @ self.router).view(self.layer.batch_size, -1)).view(-1, self.experts)

    def forward(self, x):
        routing = route(self.weights(x), self.slots)
        rows = dispatch(x, routing)
        rows = torch.relu(expert_product(rows, self.inner, routing))
        return combine(expert_product(rows, self.outer, routing), routing)


def train(steps=50, seed=0, width=64, hidden=128, experts=8, group=32, groups=64, slots=4,
          largest=1.0, rate=0.2, log=print):
    """Losses and gradient norms of ``steps`` steps on tokens from a mixture: each kind of token
    has a linear map of its own to learn."""
    torch.manual_seed(seed)
    model = RoutedExperts(width, hidden, experts, group, groups, slots)
    parameters = list(model.parameters())
    centres = torch.randn(experts, width, device="cuda")
    maps = torch.randn(experts, width, width, device="cuda") / width ** 0.5
    losses, norms = [], []
    for step in range(steps):
        kind = torch.randint(experts, (group * groups,), device="cuda")
        x = centres[kind] + 0.3 * torch.randn(kind.numel(), width, device="cuda")
        target = torch.einsum("tw,twv->tv", x, maps[kind])
        loss = (model(x) - target).square().mean()
        gradients = torch.autograd.grad(loss, parameters)
        norm = clip_gradients(gradients, largest)
        with torch.no_grad():
            for p, g in zip(parameters, gradients):
                p -= rate * g
        losses.append(loss.detach())
        norms.append(norm)
        if log and (step % 10 == 0 or step == steps - 1):
            log(f"step {step}: loss {float(losses[-1]):.4f}, gradient norm {float(norm):.3f}")
    return torch.stack(losses), torch.stack(norms), model


if __name__ == "__main__":
    arguments = argparse.ArgumentParser()
    arguments.add_argument("--steps", type=int, default=50)
    train(arguments.parse_args().steps)
