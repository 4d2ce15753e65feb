"""What the class probabilities write may not lie in what they read, in each other's outputs or in the workspace: refused on
the host, before any launch (no GPU).  Addresses are never touched."""
import ctypes

import pytest

from yolo_amd import _lib

from test_operators_host import probs
from test_operators_overlap import B, OUT, S, W, X, refused


@pytest.mark.parametrize("ids_64", [0, 1])
def test_log_probs_outputs(lib, ids_64):
    d = probs(ids_64=ids_64)                             # 10 rows of 80, three alternatives
    outs = [OUT + i * 4096 for i in range(4)]
    size = (40, 40, 120, 120)

    def call(o, offsets=None):
        return lib.y3_log_probs(ctypes.byref(d), X, offsets, B, o[0], o[1], o[2], o[3], None, 0, None)

    for i in range(4):
        for at, n in [(B, 80 if ids_64 else 40)] + [(outs[j], size[j]) for j in range(4) if j != i]:
            for to in (at, at + n - 4, at - size[i] + 4):
                o = list(outs)
                o[i] = to
                assert refused(call(o))
        o = list(outs)
        o[i] = S + 76
        d.extent = 1 << 20
        assert refused(call(o, S))
        d.extent = 9 * 85 + 80


def test_log_probs_workspace(lib):
    d = probs(classes=40000, group_ld=40000, extent=400000)
    need = ctypes.c_int64(0)
    assert lib.y3_log_probs_workspace_bytes(ctypes.byref(d), ctypes.byref(need)) == 0 and need.value > 0
    outs = [OUT + i * 4096 for i in range(4)]
    for at, n in [(X, 1600000), (B, 40)] + list(zip(outs, (40, 40, 120, 120))):
        for ws in (at, (at + n - 4) // 16 * 16, (at - need.value) // 16 * 16 + 16):
            assert refused(lib.y3_log_probs(ctypes.byref(d), X, None, B, *outs, ws, need.value, None))


def test_detection_rows(lib):
    d = _lib.DecodeDesc()
    d.batch, d.num_scales, d.num_classes, d.num_anchors = 2, 2, 80, 3
    for l in range(2):
        d.grid_h[l] = d.grid_w[l] = 13
        d.head_ld[l] = 256
    cap = 2 * 80 * 51
    call = lambda offsets, classes: lib.y3_detection_rows(ctypes.byref(d), X, W, 51, offsets, classes, None)  # noqa: E731
    for offsets in (X, X + cap * 4 - 8, X - 2 * cap * 8 + 8, W, W + 640 - 8, W - 2 * cap * 8 + 8, B, B + cap * 4 - 8, B - 2 * cap * 8 + 8):
        assert refused(call(offsets, B))
    for classes in (X, X + cap * 4 - 4, X - cap * 4 + 4, W, W + 636, W - cap * 4 + 4, OUT):
        assert refused(call(OUT, classes))
