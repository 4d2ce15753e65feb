"""What the 8-bit product and its first steps write may not lie in what they read, in each other's outputs or in the
workspace: refused on the host, before any launch (no GPU).  Addresses are never touched."""
import ctypes

import pytest

from yolo_amd import _lib

from test_operators_host import linear

M = 1 << 28                                              # between the buffers below
X, W, T, B, S, OUT, WS = (M * i for i in range(1, 8))


def refused(rc):
    return rc == -1 and b"overlap" in _lib.load().y3_last_error()


@pytest.mark.parametrize("rows", [1, 4])
@pytest.mark.parametrize("dtype", [_lib.Y3_BF16, _lib.Y3_I8])
def test_product_outputs(lib, rows, dtype):
    d = linear(rows=rows, out_ld=70, dtype=dtype)        # rows of 50 floats, 280 bytes apart; k_pad 128, n_pad 64
    at = dict(x=X, s=S if dtype == _lib.Y3_I8 else None, w=W, t=T, b=B)
    last = (rows - 1) * 280

    def call(out, **kw):
        a = dict(at, **kw)
        return lib.y3_linear_i8(ctypes.byref(d), a["x"], a["s"], a["w"], a["t"], a["b"], out, None, 0, None)

    for out in (W, W + 128 * 64 - 4, W - last - 196, T, T + 196, T - last - 196, B, B + 196, B - last - 196):
        assert refused(call(out))
    if dtype == _lib.Y3_I8:
        for out in (S, S + rows * 4 - 4, S - last - 196):
            assert refused(call(out))
    if rows > 1:                                         # 50 floats of bias do not fit between two rows: they reach into one
        for b in (OUT + 200, OUT + 276, OUT + 84):
            assert refused(call(OUT, b=b))


def test_product_workspace(lib):
    d = linear(k=5000, n=50, x_ld=8192, out_ld=50, rows=3000)
    need = ctypes.c_int64(0)
    assert lib.y3_linear_i8_workspace_bytes(ctypes.byref(d), ctypes.byref(need)) == 0 and need.value > 1 << 20
    call = lambda ws, x=X: lib.y3_linear_i8(ctypes.byref(d), x, None, W, T, B, OUT, ws, need.value, None)  # noqa: E731
    for ws in (X, X + (3000 - 1) * 16384 + 9984, W, W + 5120 * 64 - 16, T, T + 192, B, B + 192, OUT, OUT + 3000 * 200 - 16):
        assert refused(call(ws))
    for end in (X, W, T, B, OUT):
        assert refused(call(end - need.value + 16))


def test_quantised_rows(lib):
    q = lambda x, out, scale, ld=40: lib.y3_quantize_rows_i8(0, x, 9, 40, ld, out, 48, scale, None)  # noqa: E731
    for scale in (X, X + 8 * 160 + 156, X - 32, OUT, OUT + 8 * 48 + 44, OUT - 32):
        assert refused(q(X, OUT, scale))
    assert refused(q(X, OUT, X + 168, 50))               # nine scales from 8 bytes into a gap of 40
    assert refused(q(X, X + 16, S))


@pytest.mark.parametrize("dtype,es", [(_lib.Y3_F32, 4), (_lib.Y3_BF16, 2), (_lib.Y3_I8, 1)])
def test_packed_weights(lib, dtype, es):
    d = linear()                                         # k 100, n 50
    pack = lambda packed, scale=T: lib.y3_linear_i8_pack(ctypes.byref(d), dtype, W, 104, packed, scale, None)  # noqa: E731
    for packed in (W, W + (49 * 104 + 96) * es // 16 * 16, W - 128 * 64 + 16):
        assert refused(pack(packed))
    if dtype != _lib.Y3_I8:
        for scale in (W, W + (49 * 104 + 99) * es // 4 * 4, W - 196, X, X + 128 * 64 - 4, X - 196):
            assert refused(pack(X, scale))
    for ld in (1 << 44, (1 << 62) + 1):
        assert lib.y3_linear_i8_pack(ctypes.byref(d), dtype, W, ld, X, T, None) == -1
