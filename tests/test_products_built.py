"""The experts' products that the library holds are those that a call can reach (CPU only)."""

import os
import re

import pytest

from purin_amd import build as B
from tests.test_build_guards import LLVM, _code_objects, _kernel_metadata, _need_tools


def test_split_products_of_few_rows_have_one_height(tmp_path):
    """A contraction is split, and its parts written as 32-bit sums, only where tiles of 32 rows
    leave CUs idle; tiles of 64 rows are taken where they fill the CUs, and are never split."""
    _need_tools()
    if not os.path.exists(f"{LLVM}/llvm-readelf") or not os.path.exists(B.LIB):
        pytest.skip("llvm-readelf or the library is not there")
    names = [name for k, obj in enumerate(_code_objects(B.LIB)) if b"k_product_thin" in obj
             for name, _ in _kernel_metadata(obj, tmp_path, f"t{k}")]
    # (element type, type of the sums written, rows of a tile)
    built = set(re.findall(r"14k_product_thinI(DF16_|DF16b)(DF16_|DF16b|S2_|f)Li(\d+)ELi64E",
                           "\n".join(names)))
    heights = {(c == "f", int(rows)) for _, c, rows in built}
    assert heights == {(False, 32), (False, 64), (True, 32)}, sorted(built)
