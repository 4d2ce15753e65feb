"""What may be done to a layer of the 8-bit product after it was made (no GPU)."""
import pytest

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
