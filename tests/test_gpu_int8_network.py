"""-m gpu: the 8-bit products and the class probabilities as a detector runs them: Network(..., int8=True), its detections
and their alternatives, eager, captured, and through the command."""
import numpy as np
import pytest
import torch

from oracle import darknet as od
from yolo_amd import _lib, build_model, config, graph, inference
from yolo_amd import darknet_weights as dw
from yolo_amd.postprocess import PostProcessor

from test_gpu_linear_i8 import close, rule, want

pytestmark = pytest.mark.gpu


def _network(cfg, seed, **kw):
    layers, _ = od.parse_layers(cfg, 80)
    net = build_model.Network(cfg, 80, dtype="bf16", **kw)
    net.set_params(dw.random_params(layers, seed=seed))
    return net


def _view(cp, ref, heads, rows, c):
    f32 = ref["buf"][0] != "arena"
    base = heads[ref["buf"][1]].reshape(-1) if f32 else cp.arena[ref["buf"][1]:].view(torch.bfloat16)
    return torch.as_strided(base, (rows, c), (ref["ld"], 1), base.storage_offset() + ref["off"])


@pytest.mark.parametrize("cfg,size,batch,least", [("yolov3", 160, 2, 20), ("yolov3", 416, 5, 20), ("yolov3-tiny", 416, 3, 3), ("yolov3-spp", 160, 1, 20)])
def test_every_8_bit_launch_of_a_network(cfg, size, batch, least):
    """Each 8-bit launch of the real plans against the definition, on the input it found: the real shapes, strides, channel
    slices and heads.  Every other launch is the bf16 network's."""
    cfg = {"yolov3": config.yolov3_cfg_path, "yolov3-tiny": config.yolov3_tiny_cfg_path, "yolov3-spp": config.yolov3_spp_cfg_path}[cfg]
    net = _network(cfg, 11, int8=True)
    plain = build_model.Network(cfg, 80, dtype="bf16")
    plain.set_params(net.params)
    cp, other = net.plan_for(batch, size, size), plain.plan_for(batch, size, size)
    x = torch.rand(batch, size, size, 3, device="cuda")
    heads = [torch.zeros((batch, hd["h"], hd["w"], hd["ld"]), device="cuda") for hd in cp.plan.heads]
    env = {"in": x.data_ptr(), "stream": torch.cuda.current_stream().cuda_stream, "heads": [h.data_ptr() for h in heads]}
    cp.begin_pass()
    seen = 0
    for op, ref, launch in zip(cp.plan.ops, other.plan.ops, cp.launchers):
        if not op.get("int8"):
            assert op["kind"] == ref["kind"] and op.get("kernel") == ref.get("kernel")
            _lib.check(launch(env))
            continue
        rows = batch * op["out_hw"][0] * op["out_hw"][1]
        xin = _view(cp, op["x"], heads, rows, op["in_c"]).float().cpu().numpy()
        _lib.check(launch(env))
        got = _view(cp, op["y"], heads, rows, op["out_c"])
        kernel, bias = dw.fold_batch_norm(net.params[op["layer"]])
        w, t = rule(kernel[0, 0].T)
        q, s = rule(xin)
        close(got, *want(q, s, w, t, bias.astype(np.float32), op["leaky"]), "f32" if op["out_f32"] else "bf16")
        seen += 1
    assert seen >= least


def _check_alternatives(alt, heads, det, anchors_per_scale, num_classes, top):
    """Against log_softmax in 64 bits of the logits that the kept indices name."""
    B, C = det.kept_idx.shape[:2]
    kept, count = det.kept_idx.cpu().numpy(), det.kept_count.cpu().numpy()
    flat = torch.cat([h.reshape(B, -1, anchors_per_scale, 5 + C)[..., 5:].reshape(B, -1, C) for h in heads], 1).double().cpu()
    lp = torch.log_softmax(flat, -1)
    H = -(lp.exp() * lp).sum(-1)
    order = torch.sort(flat, dim=-1, descending=True, stable=True).indices
    rows = 0
    tol = 2.0 ** -24 * 80                                # (the bound of the kernel for at most 96 classes, logits below 100)
    for b in range(B):
        r = 0
        for c in range(C):
            for k in range(count[b, c]):
                p = kept[b, c, k]
                for got, ref in ((alt.logp[b, r], lp[b, p, c]), (alt.entropy[b, r], H[b, p])):
                    assert abs(float(got) - float(ref)) <= tol * (1 + abs(float(ref)))
                assert torch.equal(alt.top_ids[b, r].cpu().long(), order[b, p, :top])
                ref = lp[b, p][order[b, p, :top]]
                assert (((alt.top_logp[b, r].cpu().double() - ref).abs()) <= tol * (1 + ref.abs())).all()
                r += 1
        assert r == int(det.count[b])
        assert (alt.top_ids[b, r:] == -1).all() and (alt.logp[b, r:] == 0).all() and (alt.entropy[b, r:] == 0).all()
        rows += r
    return rows


@pytest.mark.parametrize("cfg,size,batch", [("yolov3", 160, 3), ("yolov3-tiny", 416, 2)])
def test_int8_detections_and_their_alternatives(cfg, size, batch):
    """The run as it is used: images -> 8-bit network -> decode -> NMS -> what each detection could be instead."""
    tiny = "tiny" in cfg
    net = _network(config.yolov3_tiny_cfg_path if tiny else config.yolov3_cfg_path, 21, int8=True)
    anchors = inference.read_anchors(config.tiny_anchors_path if tiny else config.anchors_path)
    pp = PostProcessor(anchors, 80, (size, size), 0.3, 0.3, 51)
    x = torch.rand(batch, size, size, 3, device="cuda")
    det, heads = pp.detect(net, x, (size, size), want_heads=True)
    plain = pp(net(x), (size, size))                     # (the same buffers: the 8-bit network gives the same bits again)
    assert plain.boxes is det.boxes
    alt = pp.alternatives(heads, det, top=5)
    assert _check_alternatives(alt, heads, det, 3, 80, 5) > 10
    one = pp.alternatives([h.contiguous() for h in heads], det, top=1)
    assert torch.equal(one.top_ids[..., 0], alt.top_ids[..., 0]) and torch.equal(one.logp, alt.logp)
    for bad in (lambda: pp.alternatives(heads, det, top=0), lambda: pp.alternatives(heads, det, top=33), lambda: pp.alternatives(heads[:-1], det),
                lambda: pp.alternatives([h[:1] for h in heads], det)):
        with pytest.raises(ValueError):
            bad()


def test_int8_network_in_a_graph_and_in_chunks():
    """Captured and replayed on several inputs, and in chunks of another size: the bits of the eager run."""
    net = _network(config.yolov3_cfg_path, 5, int8=True)
    anchors = inference.read_anchors(config.anchors_path)
    g = graph.GraphedDetector(net, anchors, 80, (160, 160), batch=3, score_threshold=0.3)
    pp = PostProcessor(anchors, 80, (160, 160), 0.3, 0.3, 51)
    xs = [torch.rand(3, 160, 160, 3, device="cuda") for _ in range(3)]
    ref = []
    for x in xs:
        heads = [h.clone() for h in net(x)]
        ref.append(heads)
        for a, b in zip(net.forward(x, chunk=2), heads):
            assert torch.equal(a, b)
    for i in (1, 2, 0):
        g.images.copy_(xs[i])
        det = g()
        other = net(xs[(i + 1) % 3])                     # eager work between the replays
        torch.cuda.synchronize()
        for a, b in zip(g.heads, ref[i]):
            assert torch.equal(a, b)
        for a, b in zip(other, ref[(i + 1) % 3]):
            assert torch.equal(a, b)
        alt = g.pp.alternatives(g.heads, det, top=2)
        assert _check_alternatives(alt, [h.clone() for h in g.heads], det, 3, 80, 2) == int(det.count.sum())


@pytest.mark.parametrize("kw", [dict(batch=1, graph=False), dict(batch=2, graph=False), dict(batch=2, graph=True)])
def test_command_with_int8_and_alternatives(tmp_path, kw):
    """run_inference with --int8 --alternatives 3: the label files as before, and one line per detection beside them."""
    import argparse
    import os
    from PIL import Image
    from yolo_amd import planner
    rng = np.random.default_rng(5)
    img_dir, out_dir = tmp_path / "imgs", tmp_path / "out"
    img_dir.mkdir()
    for i, hw in enumerate([(120, 160), (200, 150), (96, 96)]):
        Image.fromarray(rng.integers(0, 256, hw + (3,), dtype=np.uint8), mode="RGB").save(str(img_dir / ("im%d.png" % i)))
    cfg = config.yolov3_tiny_cfg_path
    layers, _ = od.parse_layers(cfg, 80)
    wpath = str(tmp_path / "tiny.weights")
    dw.write_weights(wpath, planner.parse_cfg(cfg, 80)[0], dw.random_params(layers, seed=3))
    args = argparse.Namespace(cfg=cfg, weights=wpath, input_shape=416, dtype="bf16", darknet_model="1", int8=True, alternatives=3, **kw)
    results = inference.run_inference(str(img_dir), str(out_dir), args)
    assert sum(len(r[2]) for r in results) > 0
    for i in range(3):
        labels = open(str(out_dir / "labels" / ("im%d.txt" % i))).read().splitlines()
        lines = open(str(out_dir / "alternatives" / ("im%d.txt" % i))).read().splitlines()
        assert len(lines) == len(labels) == len(results[i][2])
        for lab, line in zip(labels, lines):
            cls, logp, entropy, *alts = line.split(",")
            assert cls == lab.split(",")[4] and len(alts) == 3 and float(entropy) >= 0
            ids, lps = zip(*[(int(a.split(":")[0]), float(a.split(":")[1])) for a in alts])
            assert len(set(ids)) == 3 and list(lps) == sorted(lps, reverse=True) and lps[0] <= 0
            if int(cls) in ids:
                assert lps[ids.index(int(cls))] == float(logp)
    assert os.path.exists(str(out_dir / "images" / "im0.png"))
