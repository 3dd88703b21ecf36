"""Arguments of the experts' calls that are no tensors at all (CPU only): ValueError, as for any wrong
one, also where the argument cannot be hashed or listed."""

import pytest


def test_names_and_fields_of_other_types():
    torch = pytest.importorskip("torch")
    from purin_amd import Microscaled, activate, expert_layer, expert_product, pack, unpack

    t = torch.zeros((4, 64))
    m = Microscaled(t.byte(), t.byte(), "fp4", (4, 64), 1, torch.float32)
    part = lambda **kw: Microscaled(**{**m.__dict__, **kw})  # noqa: E731
    for f in (lambda: pack(t, ["fp4"]), lambda: pack(t, {}), lambda: activate(t, ["silu"]),
              lambda: activate(t, saved=["int8"]), lambda: expert_layer(t, t, 2, t, t, ["silu"]),
              lambda: unpack(part(kind=["fp4"])), lambda: unpack(part(shape=None)),
              lambda: expert_product(t, part(shape=None), t), lambda: expert_product(part(shape=5), m, t),
              lambda: expert_product(t, part(kind=[]), t),
              lambda: expert_layer(t, t, 2, part(shape=None), t),
              lambda: expert_layer(t, t, 2, t, part(shape=5)), lambda: expert_layer(t, t, 2, part(kind=[]), t)):
        with pytest.raises(ValueError):
            f()
