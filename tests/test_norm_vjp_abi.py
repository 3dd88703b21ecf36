"""What purin_train_norm_vjp refuses (CPU only: every call here ends before a launch)."""

from purin_amd import _lib

X = 256  # an address that nothing reads


def test_norm_vjp_refusals():
    lib = _lib.load()

    def vjp(spans, norm_dtype=0, norm=X, g_norm=X, dtype=0):
        table = (_lib.TrainTensor * max(len(spans), 1))()
        for row, (i, o, n) in zip(table, spans):
            row.in_, row.out, row.count, row.dtype = i, o, n, dtype
        return lib.purin_train_norm_vjp(None, len(spans), table, norm_dtype, norm, g_norm)

    apart = [(1 << 20, 1 << 20, 4), (1 << 21, 1 << 21, 4)]
    assert vjp([]) == _lib.OK
    assert vjp(apart, dtype=5) == _lib.ERR_ARG
    assert vjp(apart, norm_dtype=2) == _lib.ERR_ARG
    assert vjp(apart, norm=None) == _lib.ERR_ARG
    assert vjp(apart, g_norm=None) == _lib.ERR_ARG
    assert vjp([(1 << 20, None, 4)]) == _lib.ERR_ARG
    assert vjp([(None, 1 << 20, 4)]) == _lib.ERR_ARG
    assert vjp([(1 << 20, 1 << 20, -1)]) == _lib.ERR_ARG
    assert vjp([(4096, 8192, 8), (8200, 16384, 8)]) == _lib.ERR_ARG
    assert b"overlap" in lib.purin_cp_last_error()
    assert lib.purin_train_norm_vjp(None, -1, None, 0, X, X) == _lib.ERR_ARG
    assert lib.purin_train_norm_vjp(None, 1, None, 0, X, X) == _lib.ERR_ARG
