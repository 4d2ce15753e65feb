"""-m gpu: log probabilities of rows whose largest logits lie far from zero, by every kernel; above all those of chunks (more
than 1024 classes).

There the rounding of (maximum * log2 e), which every exponent of a fast sum has in it, is as large as the exponent's whole
range.  Such logits are multiples of a large power of two, so a class is either level with the maximum or impossible, and
the results are those of the level ones.  The bounds are test_gpu_class_probs.check's."""
import numpy as np
import pytest
import torch

from test_gpu_class_probs import DT, check
from yolo_amd.class_probs import log_probs

pytestmark = pytest.mark.gpu

FAR = [-2130706432.0, -4278190080.0, -2.9e9, -6.4e9, -5.58e9, 1728053248.0, 5.58e9, -1e9, 1e8, -1e8, 1e12, -1e30, 9e36, -9e36,
       1.1e37, -1.1e37]


def _agree(z, g):
    rows, C = z.shape
    ids = torch.randint(0, C, (rows,), generator=g)
    for top in (0, 5):
        check(log_probs(z.cuda(), ids.cuda(), top=top), z, ids, top)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("C", [80, 700, 1100, 2048, 4096, 5000, 32001])
def test_level_rows(C, dt):
    """All classes alike: log p = -log C, the entropy log C."""
    g = torch.Generator().manual_seed(C)
    _agree(torch.tensor(FAR)[:, None].expand(-1, C).contiguous().to(DT[dt]), g)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("C", [80, 700, 1100, 2048, 4096, 5000, 32001])
def test_masked_stretches(C, dt):
    """Ordinary logits with whole stretches at a mask's value, the other way round, and a scattering."""
    g = torch.Generator().manual_seed(C + 1)
    for v in FAR:
        z = 3 * torch.randn(4, C, generator=g)
        z[0, : C // 2] = v
        z[1, C // 3:] = v
        z[2, torch.rand(C, generator=g) < 0.9] = v
        z[3] += v
        _agree(z.to(DT[dt]), g)


def test_random_far_rows():
    g = torch.Generator().manual_seed(7)
    v = torch.cat([1.5e9 + 1.4e9 * torch.rand(400, generator=g), torch.exp(18 + 20 * torch.rand(400, generator=g))])
    v = torch.where(torch.rand(800, generator=g) < 0.5, v, -v)
    z = v[:, None].repeat(1, 1500)
    z[:, 700:] = torch.where(torch.rand(800, 1, generator=g) < 0.5, z[:, 700:], torch.nextafter(z[:, 700:], torch.full((), -np.inf)))
    _agree(z, g)
