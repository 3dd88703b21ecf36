"""What the C entry points of microscaled numbers, the activation and the layer refuse (CPU only:
every call here ends before a launch), and the struct's layout."""

import ctypes as C
import os
import shutil
import subprocess

import pytest

from purin_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
X = 256  # an address that nothing reads


def test_struct_and_codes_match_the_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "purin_train.h"',
             "int main(void) {", '  printf("%zu\\n", sizeof(purin_train_matrices));']
    for field, _ in _lib.TrainMatrices._fields_:
        lines.append(f'  printf("%zu\\n", offsetof(purin_train_matrices, {field}));')
    lines.append('  printf("%d %d %d %d %d %d %d\\n", PURIN_TRAIN_FP4, PURIN_TRAIN_INT8, '
                 "PURIN_TRAIN_RELU, PURIN_TRAIN_SILU, PURIN_TRAIN_GELU, PURIN_TRAIN_LAYER_TOKENS, "
                 "PURIN_TRAIN_LAYER_PAIRS);")
    lines += ["  return 0;", "}"]
    src, exe = tmp_path / "t.c", tmp_path / "t"
    src.write_text("\n".join(lines) + "\n")
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True, capture_output=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True,
                                          text=True).stdout.split()]
    want = [C.sizeof(_lib.TrainMatrices)]
    want += [getattr(_lib.TrainMatrices, f).offset for f, _ in _lib.TrainMatrices._fields_]
    want += [_lib.FP4, _lib.INT8, _lib.RELU, _lib.SILU, _lib.GELU, _lib.LAYER_TOKENS,
             _lib.LAYER_PAIRS]
    assert got == want


def test_pack_refusals():
    lib = _lib.load()

    def pack(dtype=2, kind=0, groups=1, rows=4, length=32, x=X, sg=0, sr=32, sl=1, codes=X, scales=X):
        return lib.purin_train_pack(None, dtype, kind, groups, rows, length, x, sg, sr, sl, codes,
                                    scales)

    assert pack(dtype=7) == _lib.ERR_ARG
    assert pack(dtype=_lib.F64) == _lib.ERR_UNSUPPORTED
    assert pack(kind=2) == _lib.ERR_ARG
    assert pack(rows=-1) == _lib.ERR_ARG and pack(length=-1) == _lib.ERR_ARG
    assert pack(length=1 << 31) == _lib.ERR_UNSUPPORTED
    assert pack(sr=2, sl=2) == _lib.ERR_ARG and pack(sr=-1) == _lib.ERR_ARG
    assert pack(x=None) == _lib.ERR_ARG and pack(codes=None) == _lib.ERR_ARG
    assert pack(codes=X + 8) == _lib.ERR_ARG and pack(scales=X + 2) == _lib.ERR_ARG
    assert pack(rows=0) == _lib.OK and pack(length=0) == _lib.OK

    def unpack(dtype=2, kind=1, rows=4, length=32, codes=X, scales=X, out=X, ldo=32):
        return lib.purin_train_unpack(None, dtype, kind, rows, length, codes, scales, out, ldo)

    assert unpack(dtype=_lib.F64) == _lib.ERR_UNSUPPORTED and unpack(kind=-1) == _lib.ERR_ARG
    assert unpack(ldo=31) == _lib.ERR_ARG and unpack(out=None) == _lib.ERR_ARG
    assert unpack(codes=X + 4) == _lib.ERR_ARG and unpack(rows=0) == _lib.OK


def test_activate_refusals():
    lib = _lib.load()

    def act(dtype=2, kind=1, gated=1, rows=4, hidden=8, u=X, ldu=16, out=X, codes=X, scales=X):
        return lib.purin_train_activate(None, dtype, kind, gated, rows, hidden, u, ldu, out, codes,
                                        scales)

    assert act(kind=3) == _lib.ERR_ARG and act(dtype=-1) == _lib.ERR_ARG
    assert act(ldu=15) == _lib.ERR_ARG and act(u=None) == _lib.ERR_ARG
    assert act(scales=None) == _lib.ERR_ARG and act(codes=None) == _lib.ERR_ARG
    assert act(dtype=_lib.F64) == _lib.ERR_UNSUPPORTED
    assert act(codes=X + 8) == _lib.ERR_ARG and act(rows=0) == _lib.OK

    def vjp(dtype=2, kind=1, gated=1, rows=4, hidden=8, u=X, ldu=16, codes=None, scales=None, g=X,
            ldg=8, g_u=X):
        return lib.purin_train_activate_vjp(None, dtype, kind, gated, rows, hidden, u, ldu, codes,
                                            scales, g, ldg, g_u)

    assert vjp(u=None) == _lib.ERR_ARG and vjp(g=None) == _lib.ERR_ARG
    assert vjp(ldg=7) == _lib.ERR_ARG and vjp(ldu=15) == _lib.ERR_ARG
    assert vjp(codes=X) == _lib.ERR_ARG
    assert vjp(dtype=_lib.F64, codes=X, scales=X) == _lib.ERR_UNSUPPORTED


def test_packed_product_refusals():
    lib = _lib.load()

    def product(dtype=2, rows=8, inner=32, outer=4, experts=2, a=X, lda=32, a_scales=None, codes=X,
                scales=X, ws=None, ws_bytes=0, ldo=4):
        return lib.purin_train_expert_product_packed(None, dtype, rows, inner, outer, experts, a, lda,
                                                     a_scales, codes, scales, X, ws, ws_bytes, X, ldo)

    assert product(dtype=_lib.F64) == _lib.ERR_UNSUPPORTED
    assert product(dtype=_lib.F32) == _lib.ERR_UNSUPPORTED
    assert product(dtype=_lib.F64, a_scales=X) == _lib.ERR_UNSUPPORTED
    assert product(lda=31) == _lib.ERR_ARG and product(ldo=3) == _lib.ERR_ARG
    assert product(codes=None) == _lib.ERR_ARG and product(codes=X + 8) == _lib.ERR_ARG
    assert product(scales=X + 1) == _lib.ERR_ARG
    assert product(a=X + 8, a_scales=X) == _lib.ERR_ARG
    assert product(experts=0) == _lib.ERR_ARG and product(experts=1025) == _lib.ERR_UNSUPPORTED
    assert product(rows=0) == _lib.OK
    # rows that are copied to other addresses need a workspace
    assert product() == _lib.ERR_ARG and b"workspace" in lib.purin_cp_last_error()
    size = lib.purin_train_expert_product_packed_workspace_bytes
    assert size(2, 0, 8, 32, 4, 2) > 0 and size(2, 1, 8, 32, 4, 2) == 0
    assert size(0, 0, 8, 32, 4, 2) < 0 and size(2, 0, -1, 32, 4, 2) < 0


def test_layer_refusals():
    lib = _lib.load()
    good = _lib.TrainMatrices(X, None, 64, 8, 1)

    def layer(dtype=2, wdtype=0, tokens=4, experts=2, slots=2, width=8, hidden=8, outer=8, act=1,
              gated=0, x=X, ldx=8, weights=X, ldw=2, a=good, b=good, ws=X, ws_bytes=1 << 20, out=X):
        return lib.purin_train_expert_layer(None, dtype, wdtype, tokens, experts, slots, width, hidden,
                                            outer, act, gated, x, ldx, weights, ldw, C.byref(a),
                                            C.byref(b), ws, ws_bytes, out)

    assert layer(dtype=_lib.F32) == _lib.ERR_UNSUPPORTED and layer(dtype=9) == _lib.ERR_ARG
    assert layer(wdtype=4) == _lib.ERR_ARG and layer(act=3) == _lib.ERR_ARG
    assert layer(slots=3) == _lib.ERR_ARG and layer(slots=0) == _lib.ERR_ARG
    assert layer(tokens=65) == _lib.ERR_UNSUPPORTED
    assert layer(tokens=64, slots=17, experts=17, ldw=17) == _lib.ERR_UNSUPPORTED
    assert layer(experts=1025) == _lib.ERR_UNSUPPORTED
    assert layer(ldx=7) == _lib.ERR_ARG and layer(ldw=1) == _lib.ERR_ARG
    assert layer(ldx=1 << 24) == _lib.ERR_UNSUPPORTED
    assert layer(width=1 << 21, ldx=1 << 21) == _lib.ERR_UNSUPPORTED
    assert layer(x=None) == _lib.ERR_ARG and layer(weights=None) == _lib.ERR_ARG
    assert layer(a=_lib.TrainMatrices(X, None, 64, 8, 2)) == _lib.ERR_ARG
    assert layer(a=_lib.TrainMatrices(X, None, -1, 8, 1)) == _lib.ERR_ARG
    assert layer(a=_lib.TrainMatrices(None, None, 64, 8, 1)) == _lib.ERR_ARG
    # two columns with a gate
    assert layer(a=_lib.TrainMatrices(X, None, 64, 8, 2), hidden=1, gated=1) == _lib.ERR_ARG
    assert layer(b=_lib.TrainMatrices(X + 8, X, 0, 0, 0)) == _lib.ERR_ARG
    assert layer(b=_lib.TrainMatrices(X, X + 1, 0, 0, 0)) == _lib.ERR_ARG
    assert layer(ws_bytes=16) == _lib.ERR_ARG and layer(ws=X + 4) == _lib.ERR_ARG
    assert layer(tokens=0) == _lib.OK
    size = lib.purin_train_expert_layer_workspace_bytes
    assert size(2, 4, 2, 2, 8, 8, 8) > 0 and size(2, 65, 2, 2, 8, 8, 8) < 0


def test_python_refusals_without_a_gpu():
    """Arguments that end before any tensor is looked at, and tensors that are not on the GPU."""
    torch = pytest.importorskip("torch")
    from purin_amd import Microscaled, activate, expert_layer, expert_product, pack, unpack
    from purin_amd.experts import expert_layer_workspace_bytes

    t = torch.zeros((4, 64))
    m = Microscaled(t.byte(), t.byte(), "fp4", (4, 64), 1, torch.float32)
    for f in (lambda: pack(t, "fp8"), lambda: pack(t, "fp4"), lambda: pack([1.0], "fp4"),
              lambda: pack(t, "int8", axis="0"), lambda: unpack(t), lambda: unpack(m),
              lambda: activate(t, "tanh"), lambda: activate(t), lambda: activate(t, saved="fp4"),
              lambda: activate([[1.0]]),
              lambda: expert_product(t, t, t, saved="int4"), lambda: expert_product(m, t, t),
              lambda: expert_product(t, m, t, saved="int8"),
              lambda: expert_layer(t, t, 2.0, t, t), lambda: expert_layer(t, t, 2, None, t),
              lambda: expert_layer(t, t, 2, t, t, "tanh"), lambda: expert_layer(t, t, 2, t, t)):
        with pytest.raises(ValueError):
            f()
    with pytest.raises(_lib.PurinError, match="64 tokens"):
        expert_layer_workspace_bytes(_lib.BF16, 65, 8, 2, 64, 64, 64)
