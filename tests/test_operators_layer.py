"""What may be done to a layer of the 8-bit product after it was made (no GPU)."""
import copy
import ctypes
import pickle

import pytest
import torch
from torch.autograd import forward_ad

from yolo_amd.linear_i8 import Int8Linear


@pytest.mark.parametrize("name", ["n", "k", "device", "leaky", "out_dtype", "bias", "scale"])
def test_attributes_are_read_only(name):
    """Calls keep descriptors (made with out_dtype and leaky) and pointers (of bias and scale): a float32 descriptor behind
    a bfloat16 output would store past its end."""
    lay = object.__new__(Int8Linear)
    setattr(lay, "_" + name, "value")
    with pytest.raises(AttributeError):
        setattr(lay, name, "other")
    assert getattr(lay, name) == "value"


@pytest.mark.parametrize("which", ["weight", "bias", "scale"])
def test_gradients_of_a_layer_are_refused(which):
    def make(track):
        t = {"weight": torch.ones(8, 32), "bias": torch.ones(8), "scale": None}
        if which == "scale":
            t["weight"], t["scale"] = torch.ones(8, 32, dtype=torch.int8), torch.ones(8)
        t[which] = track(t[which])
        return Int8Linear(t["weight"], bias=t["bias"], scale=t["scale"], device="cuda:0")

    with pytest.raises(ValueError, match="gradient"):
        make(lambda v: v.requires_grad_())
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="tangent"):
            make(lambda v: forward_ad.make_dual(v, torch.ones_like(v)))


@pytest.mark.parametrize("n,k", [(1, (1 << 32) + 5), ((1 << 32) + 5, 1), (1, 131072), ((1 << 24) + 1, 1)])
def test_sizes_past_32_bits_are_refused(n, k):
    """They are not taken for what is left of them in 32 bits."""
    with pytest.raises(ValueError, match="at most"):
        Int8Linear(torch.empty(n, k, dtype=torch.int8, device="meta"), scale=torch.empty(n, device="meta"), device="cuda:0")


@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, lambda v: pickle.loads(pickle.dumps(v))])
@pytest.mark.parametrize("with_bias", [False, True])
def test_a_copy_points_to_its_own_memory(how, with_bias):
    """... and not to that of the layer it was made of, which may be gone by then."""
    lay = object.__new__(Int8Linear)
    lay._packed, lay._scale = torch.arange(64, dtype=torch.int8), torch.rand(4)
    lay._bias = torch.rand(4) if with_bias else None
    lay._k = 3
    lay._weights = (lay._packed.data_ptr(), lay._scale.data_ptr(), lay._bias.data_ptr() if with_bias else None)
    lay._descs = {(0, 1, 2, 3): (ctypes.byref(ctypes.c_int(1)), 0)}
    new = how(lay)
    assert new._weights == (new._packed.data_ptr(), new._scale.data_ptr(), new._bias.data_ptr() if with_bias else None)
    assert new._descs == {} and new.k == 3 and torch.equal(new._packed, lay._packed) and torch.equal(new.scale, lay.scale)
    assert len(lay._descs) == 1
