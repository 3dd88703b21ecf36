"""The C ABI of ``include/purin_train.h``: exports, the struct's layout, and what it refuses
(CPU only: every call here ends before a launch)."""

import ctypes as C
import os
import re
import shutil
import subprocess

import pytest

from purin_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def declared_functions():
    text = open(os.path.join(ROOT, "include", "purin_train.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(purin_train_\w+)\s*\(", text)))


def test_header_binding_and_library_agree():
    assert set(declared_functions()) == set(_lib.TRAIN_SYMBOLS)
    lib = C.CDLL(_lib.LIB_PATH)
    assert not [s for s in declared_functions() if not hasattr(lib, s)]


def test_struct_and_codes_match_the_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "purin_train.h"',
             "int main(void) {", '  printf("%zu\\n", sizeof(purin_train_tensor));']
    names = {"in_": "in"}
    for field, _ in _lib.TrainTensor._fields_:
        lines.append(f'  printf("%zu\\n", offsetof(purin_train_tensor, {names.get(field, field)}));')
    lines.append('  printf("%d %d %d %d %d\\n", PURIN_TRAIN_F32, PURIN_TRAIN_F64, '
                 "PURIN_TRAIN_BF16, PURIN_TRAIN_F16, PURIN_TRAIN_MAX_EXPERTS);")
    lines += ["  return 0;", "}"]
    src, exe = tmp_path / "t.c", tmp_path / "t"
    src.write_text("\n".join(lines) + "\n")
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True, capture_output=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True,
                                          text=True).stdout.split()]
    want = [C.sizeof(_lib.TrainTensor)]
    want += [getattr(_lib.TrainTensor, f).offset for f, _ in _lib.TrainTensor._fields_]
    want += [_lib.F32, _lib.F64, _lib.BF16, _lib.F16, _lib.MAX_EXPERTS]
    assert got == want


X = 256  # an address that nothing reads


def test_route_refusals():
    lib = _lib.load()

    def route(dtype=0, tokens=4, experts=8, slots=2, ld=8, weights=X, offsets=X):
        return lib.purin_train_route(None, dtype, tokens, experts, slots, weights, ld, None, 0,
                                     X, X, offsets, X, X)

    assert route(dtype=9) == _lib.ERR_ARG
    assert route(slots=9) == _lib.ERR_ARG and b"slots" in lib.purin_cp_last_error()
    assert route(slots=0) == _lib.ERR_ARG
    assert route(ld=7) == _lib.ERR_ARG
    assert route(weights=None) == _lib.ERR_ARG
    assert route(offsets=None) == _lib.ERR_ARG
    assert route(experts=1025, ld=1025) == _lib.ERR_UNSUPPORTED
    assert route(tokens=1 << 30) == _lib.ERR_UNSUPPORTED
    # a workspace that is missing
    assert route(tokens=1 << 20) == _lib.ERR_ARG and b"workspace" in lib.purin_cp_last_error()
    assert lib.purin_train_route_workspace_bytes(-1, 8, 2) < 0
    assert lib.purin_train_route_workspace_bytes(4, 0, 2) < 0


def test_row_refusals():
    lib = _lib.load()
    assert lib.purin_train_dispatch(None, 0, 4, 8, 2, 16, X, 15, X, X, X) == _lib.ERR_ARG
    assert lib.purin_train_dispatch(None, 0, 4, 8, 2, 16, None, 16, X, X, X) == _lib.ERR_ARG
    assert lib.purin_train_dispatch(None, 0, 4, 8, 2, -1, X, 16, X, X, X) == _lib.ERR_ARG
    assert lib.purin_train_combine(None, 0, 7, 4, 2, 16, X, 16, X, X, X) == _lib.ERR_ARG
    assert lib.purin_train_combine(None, 0, 0, 4, 2, 16, X, 3, X, X, X) == _lib.ERR_ARG
    assert lib.purin_train_combine_vjp(None, 0, 0, 4, 8, 2, 16, X, 16, X, 16, X, X, None, X,
                                       X) == _lib.ERR_ARG


def test_product_refusals():
    lib = _lib.load()

    def product(dtype=0, rows=8, inner=4, outer=4, experts=2, lda=4, we=16, wi=4, wo=1, ldo=4):
        return lib.purin_train_expert_product(None, dtype, rows, inner, outer, experts, X, lda, X,
                                              we, wi, wo, X, None, 0, X, ldo)

    assert product(dtype=4) == _lib.ERR_ARG
    assert product(experts=0) == _lib.ERR_ARG
    assert product(lda=3) == _lib.ERR_ARG
    assert product(ldo=3) == _lib.ERR_ARG
    assert product(wi=8, wo=2) == _lib.ERR_ARG
    assert product(we=-1) == _lib.ERR_ARG
    assert product(experts=1025) == _lib.ERR_UNSUPPORTED
    assert product(rows=1 << 31) == _lib.ERR_UNSUPPORTED
    assert lib.purin_train_expert_weights_vjp(None, 0, 8, 4, 4, 2, X, 3, X, 4, X, None, 0,
                                              X) == _lib.ERR_ARG


def test_clip_refusals():
    lib = _lib.load()
    need = lib.purin_train_clip_workspace_bytes(2)

    def clip(spans, largest=1.0, ws=X, ws_bytes=need, norm_dtype=0, norm=X, dtype=0):
        table = (_lib.TrainTensor * len(spans))()
        for row, (i, o, n) in zip(table, spans):
            row.in_, row.out, row.count, row.dtype = i, o, n, dtype
        return lib.purin_train_clip(None, len(spans), table, largest, ws, ws_bytes, norm_dtype,
                                    norm)

    apart = [(1 << 20, 1 << 20, 4), (1 << 21, 1 << 21, 4)]
    assert clip(apart, largest=float("nan")) == _lib.ERR_ARG
    assert clip(apart, dtype=5) == _lib.ERR_ARG
    assert clip(apart, norm_dtype=2) == _lib.ERR_ARG
    assert clip(apart, norm=None) == _lib.ERR_ARG
    assert clip(apart, ws_bytes=8) == _lib.ERR_ARG
    assert clip(apart, ws=X + 8) == _lib.ERR_ARG
    assert clip([(None, None, 4)]) == _lib.ERR_ARG
    assert clip([(1 << 20, 1 << 20, -1)]) == _lib.ERR_ARG
    # memory that is shared: twice in place, an output over an input, outputs over each other
    for spans in ([(4096, 4096, 4), (4096, 4096, 4)], [(4096, 4096, 8), (4112, 4112, 8)],
                  [(4096, 8192, 8), (8200, 16384, 8)], [(4096, 8192, 8), (12288, 8204, 8)],
                  [(4096, 4100, 8)]):
        assert clip(spans) == _lib.ERR_ARG, spans
        assert b"overlap" in lib.purin_cp_last_error()
