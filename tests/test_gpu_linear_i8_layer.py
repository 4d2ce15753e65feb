"""-m gpu: a layer of the 8-bit product as an object: when its weights are there, and what may change about it later."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from oracle import darknet as od
from yolo_amd import build_model, config
from yolo_amd import darknet_weights as dw
from yolo_amd.class_probs import log_probs
from yolo_amd.linear_i8 import Int8Linear, quantize_rows

pytestmark = pytest.mark.gpu


def _busy(n=40):
    """Work queued on the current stream: the launches behind it start milliseconds later."""
    a = torch.zeros(4096, 4096, device="cuda")
    b = torch.empty_like(a)
    for _ in range(n):
        torch.mm(a, a, out=b)


@pytest.mark.parametrize("weights", ["f32", "i8", "cpu"])
def test_a_layer_made_behind_queued_work_is_called_on_another_stream(weights):
    n, k = 256, 640
    g = torch.Generator().manual_seed(1)
    x = torch.randn(300, k, generator=g).to(torch.bfloat16).cuda()
    w = torch.randint(-127, 128, (n, k), generator=g).to(torch.int8) if weights == "i8" else torch.randn(n, k, generator=g)
    kw = dict(scale=torch.rand(n, generator=g).cuda()) if weights == "i8" else {}
    w = w if weights == "cpu" else w.cuda()
    bias = torch.ones(n, device="cuda")                      # (copies from the host would wait for the queue)
    ref = Int8Linear(w, bias=bias, **kw)(x)
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(one):
        for size in (n * k, 4 * n):                          # what the layer's allocations would otherwise find
            for dirt in [torch.full((size,), 101, dtype=torch.uint8, device="cuda") for _ in range(4)]:
                del dirt
        _busy()
        lay = Int8Linear(w, bias=bias, **kw)
    with torch.cuda.stream(two):
        got = lay(x)
    torch.cuda.synchronize()
    assert torch.equal(got, ref)


def test_a_network_packs_on_one_stream_and_runs_on_another():
    """The 1x1 weights are packed while the first plan is built and serve every later plan."""
    cfg = config.yolov3_tiny_cfg_path
    params = dw.random_params(od.parse_layers(cfg, 80)[0], seed=4)
    x = torch.rand(3, 160, 160, 3, device="cuda")
    nets = []
    for _ in range(2):
        net = build_model.Network(cfg, 80, dtype="bf16", int8=True)
        net.set_params(params)
        nets.append(net)
    ref = [h.clone() for h in nets[0](x)]
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(one):
        _busy()
        first = nets[1](x[:1])
    with torch.cuda.stream(two):
        got = nets[1](x)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, ref)) and all(torch.equal(a, b[:1]) for a, b in zip(first, ref))


def test_a_layer_made_inside_a_capture():
    n, k = 64, 200
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn(50, k, generator=g).cuda(), torch.randn(n, k, generator=g).cuda()
    Int8Linear(w)(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = Int8Linear(w)(x)
    for seed in range(3):
        w.copy_(torch.randn(n, k, generator=g))
        ref = Int8Linear(w)(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ref)


def test_a_layer_keeps_its_own_scale_and_bias():
    n, k = 40, 100
    g = torch.Generator().manual_seed(3)
    x = torch.randn(7, k, generator=g).cuda()
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8).cuda()
    scale, bias = torch.rand(n, generator=g).cuda(), torch.randn(n, generator=g).cuda()
    lay = Int8Linear(w, scale=scale, bias=bias)
    ref = lay(x)
    for t in (w, scale, bias):
        t.zero_()
    assert torch.equal(lay(x), ref)
    wide = torch.randn(n, 2, generator=g).double()           # other types and strides are copied as they were
    a, b = Int8Linear(w, scale=wide[:, 0], bias=wide[:, 1]), Int8Linear(w, scale=wide[:, 0].float().cuda(), bias=wide[:, 1].float().cuda())
    assert torch.equal(a(x), b(x))


def test_gradients_of_a_call_are_refused():
    """Of every tensor that a call takes, in both directions of differentiation; without gradients they all pass."""
    lay = Int8Linear(torch.ones(8, 32), out_dtype=torch.float32)
    x, q, s, y = torch.ones(4, 32).cuda(), torch.ones(4, 32, dtype=torch.int8).cuda(), torch.ones(4).cuda(), torch.empty(4, 8).cuda()
    lq = Int8Linear(torch.ones(8, 32, dtype=torch.int8), scale=torch.ones(8), out_dtype=torch.float32)
    ids = torch.zeros(4, dtype=torch.int64).cuda()
    calls = [(x, lambda t: lay(t)), (x, lambda t: quantize_rows(t)), (s, lambda t: lq(q, scale=t)), (y, lambda t: lay(x, out=t)),
             (x, lambda t: log_probs(t, ids, top=2)), (s, lambda t: log_probs(x, ids, out=(t, torch.empty(4, device="cuda"), None, None))),
             (s, lambda t: log_probs(x, ids, out=(torch.empty(4, device="cuda"), t, None, None)))]
    for t, call in calls:
        call(t)
        track = t.clone().requires_grad_()
        with pytest.raises(ValueError, match="gradient"):
            call(track)
        with torch.no_grad():
            call(track)
        with forward_ad.dual_level():
            call(t)
            with pytest.raises(ValueError, match="tangent"):
                call(forward_ad.make_dual(t, torch.ones_like(t)))


def test_vectors_between_the_rows_of_an_output():
    """Scales and bias in the padding of the output's own buffer, the input in another slice of it: nothing overlaps."""
    rows, k, n = 33, 24, 16
    g = torch.Generator().manual_seed(5)
    buf = torch.randn(rows, 64, generator=g).cuda()
    x, out = buf[:, :k], buf[:, k:k + n]
    lay = Int8Linear(torch.randn(n, k, generator=g), out_dtype=torch.float32)
    ref = lay(x.contiguous())
    before = buf.clone()
    scale = buf[5, 44:44 + n]                                # between rows 5 and 6 of `out`
    scale.copy_(lay.scale)
    lay._weights = (lay._packed.data_ptr(), scale.data_ptr(), None)
    lay(x, out=out)
    before[5, 44:44 + n] = lay.scale
    before[:, k:k + n] = ref
    assert torch.equal(buf, before)


def test_rows_past_32_bits_are_refused():
    """5 or 80 values are what 32 bits hold of these lengths."""
    one = torch.zeros(1, 1, dtype=torch.bfloat16, device="cuda")
    z, off = torch.zeros(400, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad in (lambda: quantize_rows(one.expand(1, (1 << 32) + 5)), lambda: log_probs(one.expand(1, (1 << 32) + 80)),
                lambda: log_probs(z, rows=off, classes=(1 << 32) + 80), lambda: log_probs(z, rows=off, classes=(1 << 24) + 1)):
        with pytest.raises(ValueError):
            bad()
