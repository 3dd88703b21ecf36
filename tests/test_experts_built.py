"""The built device code of products with packed weights and of the layer (CPU only): loads
straight into LDS leave their wait states, and no kernel spills."""

import os

import pytest

from purin_amd import build as B
from tests.test_build_guards import _code_objects, _disassemble, _need_tools
from tests.test_lds_load_hazards import hazards


@pytest.mark.parametrize("kernel", [b"k_product_packed", b"k_layer_up"])
def test_loads_into_lds_leave_their_wait_states(kernel, tmp_path):
    _need_tools()
    if not os.path.exists(B.LIB):
        pytest.skip("libpurin_cp.so is not built")
    loads = 0
    for k, obj in enumerate(_code_objects(B.LIB)):
        if kernel not in obj:
            continue
        text = _disassemble(obj, tmp_path, f"l{k}")
        n, bad = hazards(text)
        loads += n
        assert not bad, f"{len(bad)} of {n} loads, the first: {bad[0]}"
        assert "scratch_" not in text, "a kernel uses scratch memory"
    assert loads > 0, "no load into LDS found"
