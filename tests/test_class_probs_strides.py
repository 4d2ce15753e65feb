"""How log_probs reads a tensor's strides (no GPU)."""
import pytest
import torch

from yolo_amd.class_probs import _two_strides


@pytest.mark.parametrize("shape,strides,want", [
    ((80,), (1,), (1, 1, 0, 0)),
    ((1, 1, 80), (7, 9, 1), (1, 1, 0, 0)),
    ((5, 80), (85, 1), (5, 1, 85, 0)),
    ((2, 5, 80), (5 * 85, 85, 1), (10, 1, 85, 0)),
    ((2, 5, 3, 80), (5 * 256, 256, 85, 1), (30, 3, 256, 85)),
    ((2, 5, 3, 80), (6 * 256, 256, 85, 1), None),
    ((4, 7, 80), (0, 100, 1), (28, 7, 0, 100)),
    ((2, (1 << 31) - 1, 1), (1 << 40, 1, 1), (2 * ((1 << 31) - 1), (1 << 31) - 1, 1 << 40, 1)),
    ((2, (1 << 31) + 8, 1), (1 << 40, 1, 1), None),            # not a group of 8 - 2^31
    ((2, 1 << 32, 1), (1 << 32, 1, 1), (1 << 33, 1, 1, 0)),
])
def test_two_strides(shape, strides, want):
    assert _two_strides(torch.empty_strided(shape, strides, dtype=torch.bfloat16, device="meta")) == want
