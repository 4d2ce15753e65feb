"""The 8-bit product's and the class probabilities' refusals at the C-ABI: everything here is decided on the host, before
any launch (no GPU)."""
import ctypes

import pytest

from yolo_amd import _lib

P = 1 << 12          # an aligned address nobody dereferences: every call below is refused first


def linear(**kw):
    d = _lib.LinearI8Desc()
    d.dtype, d.out_dtype, d.k, d.n, d.rows, d.x_ld, d.out_ld = _lib.Y3_BF16, _lib.Y3_F32, 100, 50, 4, 100, 50
    for k, v in kw.items():
        setattr(d, k, v)
    if 1 <= d.k <= 131071 and 1 <= d.n <= 1 << 24 and "k_pad" not in kw:
        assert _lib.load().y3_linear_i8_layout(ctypes.byref(d)) == 0
    return d


def test_linear_layout(lib):
    for k, n, kp, np_ in ((1, 1, 128, 16), (128, 16, 128, 16), (129, 17, 256, 32), (1024, 255, 1024, 256), (131071, 3, 131072, 16)):
        d = linear(k=k, n=n, x_ld=k, out_ld=n)
        assert (d.k_pad, d.n_pad) == (kp, np_)
    for bad in (dict(k=0), dict(k=131072), dict(n=0), dict(n=(1 << 24) + 1)):
        d = _lib.LinearI8Desc()
        d.k, d.n = 8, 8
        for k, v in bad.items():
            setattr(d, k, v)
        assert lib.y3_linear_i8_layout(ctypes.byref(d)) == -1
    assert lib.y3_linear_i8_layout(None) == -1


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(out_dtype=_lib.Y3_I8), dict(rows=-1), dict(rows=1 << 50), dict(x_ld=99), dict(out_ld=49),
                                dict(flags=2), dict(k_pad=64, n_pad=64)])
def test_linear_descriptor_refusals(lib, kw):
    d = linear(**kw)
    need = ctypes.c_int64(0)
    assert lib.y3_linear_i8_workspace_bytes(ctypes.byref(d), ctypes.byref(need)) == -1
    assert lib.y3_linear_i8(ctypes.byref(d), P, None, P, P, None, 1 << 30, P, 1 << 40, None) == -1
    with pytest.raises(ValueError):
        _lib.check(-1)


def test_linear_pointer_refusals(lib):
    d = linear()
    call = lambda *a: lib.y3_linear_i8(ctypes.byref(d), *a, None)  # noqa: E731
    big, out = 1 << 40, 1 << 30
    assert call(None, None, P, P, None, out, P, big) == -1
    assert call(P, None, None, P, None, out, P, big) == -1
    assert call(P, None, P, None, None, out, P, big) == -1
    assert call(P, None, P, P, None, None, P, big) == -1
    assert call(P, P, P, P, None, out, P, big) == -1                # scales with float rows
    assert call(P + 1, None, P, P, None, out, P, big) == -2
    assert call(P, None, P + 8, P, None, out, P, big) == -2
    assert call(P, None, P, P + 2, None, out, P, big) == -2
    assert call(P, None, P, P, P + 1, out, P, big) == -2
    assert call(P, None, P, P, None, out + 2, P, big) == -2
    assert call(P, None, P, P, None, P + 8, P, big) == -1           # overlaps x
    assert b"overlap" in lib.y3_last_error()
    d = linear(dtype=_lib.Y3_I8)
    assert call(P, None, P, P, None, out, None, 0) == -1             # 8-bit rows without scales
    d = linear(rows=0)
    assert call(None, None, None, None, None, None, None, 0) == 0


def test_quantize_and_pack_refusals(lib):
    q = lib.y3_quantize_rows_i8
    assert q(5, P, 1, 8, 8, 1 << 20, 16, P, None) == -1
    assert q(0, P, 1, 0, 8, 1 << 20, 16, P, None) == -1
    assert q(0, P, -1, 8, 8, 1 << 20, 16, P, None) == -1
    assert q(0, P, 1, 8, 7, 1 << 20, 16, P, None) == -1
    assert q(0, P, 1, 8, 8, 1 << 20, 8, P, None) == -2
    assert q(0, P, 1, 17, 17, 1 << 20, 16, P, None) == -2
    assert q(0, P, 1, 8, 8, (1 << 20) + 8, 16, P, None) == -2
    assert q(0, P, 1, 8, 8, P, 16, P, None) == -1
    assert q(0, P, 1, 8, 8, 1 << 20, 16, None, None) == -1
    assert q(0, None, 0, 8, 8, None, 16, None, None) == 0
    d = linear()
    pack = lambda *a: lib.y3_linear_i8_pack(ctypes.byref(d), *a, None)  # noqa: E731
    assert pack(7, P, 100, P, P) == -1
    assert pack(0, P, 99, P, P) == -1
    assert pack(0, P, 100, P + 4, P) == -2
    assert pack(0, P, 100, P, None) == -1
    assert pack(0, None, 100, P, P) == -1


O = P + (1 << 32)                                       # outputs, far from the logits


def probs(**kw):
    d = _lib.LogProbsDesc()
    d.dtype, d.classes, d.rows, d.group, d.group_ld, d.row_ld, d.top, d.extent = _lib.Y3_F32, 80, 10, 1, 85, 0, 3, 9 * 85 + 80
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw", [dict(dtype=2), dict(classes=0), dict(classes=(1 << 24) + 1), dict(rows=-1), dict(top=33), dict(top=-1),
                                dict(classes=2), dict(extent=9 * 85 + 79), dict(group=0), dict(group_ld=-1), dict(row_ld=-1), dict(rows=11),
                                dict(group=3, group_ld=256, row_ld=85, extent=3 * 256 + 79)])
def test_log_probs_descriptor_refusals(lib, kw):
    d = probs(**kw)
    assert lib.y3_log_probs(ctypes.byref(d), P, None, P, O, O, O, O, P, 1 << 40, None) == -1
    assert b"overlap" not in lib.y3_last_error()


def test_log_probs_pointer_refusals(lib):
    d = probs()
    call = lambda *a: lib.y3_log_probs(ctypes.byref(d), *a, P, 1 << 40, None)  # noqa: E731
    assert call(None, None, P, O, O, O, O) == -1
    assert call(P, None, None, O, O, O, O) == -1
    assert call(P, None, P, None, O, O, O) == -1
    assert call(P, None, P, O, O, None, O) == -1
    assert call(P + 2, None, P, O, O, O, O) == -2
    assert call(P, P + 4, P, O, O, O, O) == -2
    assert call(P, None, P + 2, O, O, O, O) == -2
    assert call(P, None, P, O + 1, O, O, O) == -2
    end = P + (9 * 85 + 80) * 4
    for i, n in enumerate((10, 10, 30, 30)):                         # outputs that reach into the logits
        for at in (P, end - 4, P - 4 * n + 4, P + 82 * 4):
            outs = [O] * 4
            outs[i] = at
            assert call(P, None, P, *outs) == -1 and b"overlap" in lib.y3_last_error()
    d = probs(rows=0)
    assert call(None, None, None, None, None, None, None) == 0


def test_linear_slices_of_one_buffer_are_not_an_overlap(lib):
    """Rows of 5000 bf16 and of 50 fp32 in one buffer of 16 KB a row: side by side they pass (the call is then refused for
    its workspace), four bytes into each other they do not."""
    need = ctypes.c_int64(0)
    d = linear(k=5000, n=50, x_ld=8192, out_ld=4096, rows=70000)          # k too long to be quantised on the way: a workspace
    assert lib.y3_linear_i8_workspace_bytes(ctypes.byref(d), ctypes.byref(need)) == 0 and need.value > 0
    call = lambda out: lib.y3_linear_i8(ctypes.byref(d), P, None, P, P, None, out, None, 0, None)  # noqa: E731
    for out in (P + 10000, P + 16384 - 200, P + 3 * 16384 + 12000):
        assert call(out) == -1 and b"workspace" in lib.y3_last_error()
    for out in (P + 9996, P + 16384 - 196, P, P + 3 * 16384 + 100):
        assert call(out) == -1 and b"overlap" in lib.y3_last_error()


def test_detection_rows_refusals(lib):
    d = _lib.DecodeDesc()
    d.batch, d.num_scales, d.num_classes, d.num_anchors = 2, 2, 80, 3
    for l in range(2):
        d.grid_h[l] = d.grid_w[l] = 13
        d.head_ld[l] = 256
    call = lambda *a: lib.y3_detection_rows(ctypes.byref(d), *a, None)  # noqa: E731
    assert call(None, P, 51, P, P) == -1 and call(P, None, 51, P, P) == -1 and call(P, P, 51, None, P) == -1 and call(P, P, 51, P, None) == -1
    assert call(P, P, 0, P, P) == -1 and call(P, P, 257, P, P) == -1
    assert call(P + 2, P, 51, P, P) == -2 and call(P, P, 51, P + 4, P) == -2
    for field, v in (("batch", 0), ("num_scales", 4), ("num_classes", 97), ("num_anchors", 0)):
        old = getattr(d, field)
        setattr(d, field, v)
        assert call(P, P, 51, P, P) == -1
        setattr(d, field, old)
    d.head_ld[1] = 254
    assert call(P, P, 51, P, P) == -1


def test_int8_network_wants_bf16():
    from yolo_amd import build_model, config
    with pytest.raises(ValueError, match="int8"):
        build_model.Network(config.yolov3_tiny_cfg_path, 80, dtype="fp32", device="cuda:0", int8=True)


@pytest.mark.parametrize("k", [-1, 33])
def test_alternatives_option_range(tmp_path, k):
    import argparse
    from yolo_amd import inference
    with pytest.raises(ValueError, match="alternatives"):
        inference.run_inference(str(tmp_path), str(tmp_path / "out"), argparse.Namespace(alternatives=k))
    assert not (tmp_path / "out").exists()
