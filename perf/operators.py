"""Workloads of two operators: the matrix product in 8-bit integers with a scale per row (pixel or token) and per
channel (yolo_amd.linear_i8), and the log probabilities of given classes with entropy and top alternatives
(yolo_amd.class_probs).

`run` computes them in their plain form, elementary torch operations in 32 bits, or, where `own` is set, through the
package.  `exact` gives the same from the definitions in 64 bits.

The product.  A row x of the input is held as 8-bit integers q = round_half_even(x * (127 / a)) with one scale s = a / 127,
a = max(max_j |x_j|, 127 * 2^-126); a weight row w_n likewise, once, when the layer is loaded.  Then
    y[m, n] = act(s[m] * t[n] * sum_k q[m, k] * w[n, k] + b[n]),     act = identity or max(v, 0.1 v).
The log probabilities.  For a row of C logits z and a class c:  log p_c = z_c - log sum_j exp(z_j), the entropy
- sum_j p_j log p_j, and the classes of the `top` largest logits (ties: the lowest class) with their log p.
"""
import math

import torch

own = False

TINY = 127.0 * 2.0 ** -126          # the smallest magnitude a row's scale is made for
F32, F64 = torch.float32, torch.float64
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- the cases ---------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token through a square projection: the weights are read once for one row, latency and HBM bound
        dict(name="product 1 row", op="product", rows=1, k=4096, n=4096, x="bf16", out="bf16", bias=False, leaky=False),
        # a few dozen rows (a small serving batch) through a narrowing projection
        dict(name="product 24 rows", op="product", rows=24, k=8192, n=2048, x="bf16", out="bf16", bias=True, leaky=False),
        # YOLOv3 at 608, one image: the 1x1 convolutions 1024 -> 512 on the 19 x 19 map
        dict(name="product 19x19 b1", op="product", rows=361, k=1024, n=512, x="bf16", out="bf16", bias=True, leaky=True),
        # the same, batch 64
        dict(name="product 19x19 b64", op="product", rows=23104, k=1024, n=512, x="bf16", out="bf16", bias=True, leaky=True),
        # YOLOv3 at 608, batch 64: the 1x1 convolutions 512 -> 256 of the 38 x 38 residual stage
        dict(name="product 38x38 b64", op="product", rows=92416, k=512, n=256, x="bf16", out="bf16", bias=True, leaky=True),
        # ... and the head of the 76 x 76 scale, 16 images: 255 channels of fp32
        dict(name="product head 76x76 b16", op="product", rows=92416, k=256, n=255, x="bf16", out="f32", bias=True, leaky=False),
        # a large product of rows that are 8-bit already (one quantisation, several products): matrix-core bound
        dict(name="product 8192 i8", op="product", rows=8192, k=8192, n=8192, x="i8", out="bf16", bias=False, leaky=False),
        # nothing a multiple of anything, fp32 in and out
        dict(name="product odd f32", op="product", rows=1777, k=1003, n=777, x="f32", out="f32", bias=True, leaky=False),
        # one row over a large vocabulary, twenty alternatives: latency bound
        dict(name="probs 1 x 128000", op="probs", rows=1, classes=128000, dtype="bf16", pad=0, top=20, ids=True),
        # scoring a few thousand given tokens over an odd vocabulary (rows start at odd addresses)
        dict(name="probs 4096 x 32001", op="probs", rows=4096, classes=32001, dtype="bf16", pad=0, top=5, ids=True),
        # every box of the 76 x 76 scale, 64 images at 608: 80 class logits inside [.., 3 x (5 + 80)] cells of 256 floats
        dict(name="probs boxes 76x76 b64", op="boxes", cells=64 * 5776, anchors=3, classes=80, top=3),
        # the class posterior of 64 images' kept detections, gathered from that head; a third of the rows lie in the
        # other scales and stay as they are
        dict(name="probs kept boxes", op="kept", rows=4096, cells=64 * 5776, anchors=3, classes=80, top=5),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.6:
        rows, k, n = _log_int(rng, 1, 16384), _log_int(rng, 48, 8192), _log_int(rng, 16, 8192)
        if rng.random() < 0.5:                                  # channel counts of real layers, as often as odd ones
            k, n = (k + 31) // 32 * 32, (n + 31) // 32 * 32
        return dict(op="product", rows=rows, k=k, n=n, x=rng.choice(["bf16", "bf16", "f32", "i8"]),
                    out=rng.choice(["bf16", "f32"]), bias=rng.random() < 0.5, leaky=rng.random() < 0.5)
    if rng.random() < 0.3:
        return dict(op="kept", rows=_log_int(rng, 1, 16384), cells=_log_int(rng, 64, 64 * 5776), anchors=rng.choice([2, 3]),
                    classes=rng.randint(1, 96), top=rng.randint(1, 8))
    classes = _log_int(rng, 20, 160000)
    rows = _log_int(rng, 1, max(1, min(65536, 120_000_000 // classes)))
    return dict(op="probs", rows=rows, classes=classes, dtype=rng.choice(["bf16", "f32"]), pad=rng.choice([0, 0, 1, 7, 64]),
                top=min(classes, rng.choice([0, 1, 5, 20])), ids=True)


# ---- the inputs --------------------------------------------------------------------------------------------------
def _activations(rows, k, g, leaky):
    """Rows as they reach a product: each channel with a gain of its own, some far above the rest, each row with a
    magnitude of its own; behind a leaky activation the negative half is a tenth."""
    gain = torch.exp(0.7 * torch.randn(k, device="cuda", generator=g))
    gain = torch.where(torch.rand(k, device="cuda", generator=g) < 0.01, gain * 8, gain)
    x = torch.randn(rows, k, device="cuda", generator=g) * gain * torch.exp(0.5 * torch.randn(rows, 1, device="cuda", generator=g))
    return torch.where(x > 0, x, 0.1 * x) if leaky else x


def _quantized(x):
    a = x.abs().amax(-1, keepdim=True).clamp(min=TINY)
    return torch.round(x * (127.0 / a)), a / 127.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "product":
        rows, k, n = case["rows"], case["k"], case["n"]
        x = _activations(rows, k, g, case["leaky"])
        if case["x"] == "i8":
            q, sc = _quantized(x)
            s["x"], s["x_scale"] = q.to(torch.int8), sc.reshape(-1).contiguous()
        else:
            s["x"], s["x_scale"] = x.to(DTYPES[case["x"]]), None
        w, ws = _quantized(torch.randn(n, k, device="cuda", generator=g) * torch.exp(0.5 * torch.randn(n, 1, device="cuda", generator=g)) / math.sqrt(k))
        s["w"], s["w_scale"] = w.to(torch.int8), ws.reshape(-1).contiguous()
        s["b"] = 0.2 * torch.randn(n, device="cuda", generator=g) if case["bias"] else None
        if own:                                                 # the layer, its weights laid out once
            from yolo_amd.linear_i8 import Int8Linear
            s["layer"] = Int8Linear(s["w"], bias=s["b"], scale=s["w_scale"], leaky=case["leaky"], out_dtype=DTYPES[case["out"]])
        return s
    if case["op"] == "probs":
        rows, c = case["rows"], case["classes"]
        z = 2.5 * torch.randn(rows, c + case["pad"], device="cuda", generator=g) + 6.0 * (torch.rand(rows, c + case["pad"], device="cuda", generator=g) < 4.0 / c)
        s["z"] = z.to(DTYPES[case["dtype"]])[:, :c]
        s["rows"] = None
        likely = s["z"].argmax(-1)
        other = torch.randint(0, c, (rows,), device="cuda", generator=g)
        s["ids"] = torch.where(torch.rand(rows, device="cuda", generator=g) < 0.6, likely, other).to(torch.int32) if case["ids"] else None
        return s
    # a head tensor: cells of `anchors` boxes, each x, y, w, h, confidence and the class logits; cells are padded to 8 floats
    c, a = case["classes"], case["anchors"]
    ld = (a * (5 + c) + 7) // 8 * 8
    head = torch.randn(case["cells"], ld, device="cuda", generator=g) * 2 - 3
    hot = torch.randint(0, c, (case["cells"] * a,), device="cuda", generator=g)
    at = torch.arange(case["cells"] * a, device="cuda")
    flat = head.view(-1)
    flat[(at // a) * ld + (at % a) * (5 + c) + 5 + hot] += 7.0 * torch.rand(at.numel(), device="cuda", generator=g)
    s["head"] = head
    s["z"] = head.as_strided((case["cells"], a, c), (ld, 5 + c, 1), 5)
    s["rows"] = None
    n = case["cells"] * a
    if case["op"] == "kept":
        pick = torch.randint(0, n, (case["rows"],), device="cuda", generator=g)
        off = (pick // a) * ld + (pick % a) * (5 + c) + 5
        s["rows"] = torch.where(torch.rand(case["rows"], device="cuda", generator=g) < 1 / 3, torch.full_like(off, -1), off)
        n = case["rows"]
    s["ids"] = torch.randint(0, c, (n,), device="cuda", generator=g).to(torch.int32)
    if case["op"] == "boxes":
        s["ids"] = s["ids"].view(case["cells"], a)
    else:                                                       # what the rows of other scales hold already
        s["out"] = (torch.full((n,), -1.0, device="cuda"), torch.full((n,), -2.0, device="cuda"),
                    torch.full((n, case["top"]), -3, dtype=torch.int32, device="cuda"), torch.full((n, case["top"]), -4.0, device="cuda"))
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------
def _order(z, bits):
    """Integers that order like (logit, then the lower class first)."""
    b = (z.float() + 0.0).view(torch.int32)
    b = torch.where(b < 0, b ^ 0x7fffffff, b).to(torch.int64)
    return (b << bits) - torch.arange(z.shape[-1], device=z.device)


def _log_probs(z, ids, top):
    """logp of `ids`, entropy, the `top` alternatives and their logp, of logits [..., C]."""
    x = z.float()
    d = x - x.amax(-1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    logp = d - torch.log(total)
    entropy = -torch.where(e > 0, e * logp, 0.0).sum(-1) / total[..., 0]
    got = [torch.gather(logp, -1, ids.long()[..., None])[..., 0] if ids is not None else None, entropy]
    if top:
        at = torch.topk(_order(z, 20), top, dim=-1).indices
        got += [at.to(torch.int32), torch.gather(logp, -1, at)]
    return got


def _plain(s):
    if s["op"] == "product":
        if s["x_scale"] is None:
            q, sc = _quantized(s["x"].float())
        else:
            q, sc = s["x"].float(), s["x_scale"][:, None]
        y = torch.matmul(q, s["w"].float().t()) * s["w_scale"] * sc
        if s["b"] is not None:
            y = y + s["b"]
        if s["leaky"]:
            y = torch.where(y > 0, y, 0.1 * y)
        return y.to(DTYPES[s["out"]])
    if s["rows"] is None:
        return _log_probs(s["z"], s["ids"], s["top"])
    rows = s["rows"]
    z = s["head"].view(-1)[rows.clamp(min=0)[:, None] + torch.arange(s["classes"], device=rows.device)]
    got = _log_probs(z, s["ids"], s["top"])
    keep = rows >= 0
    return [torch.where(keep.view(-1, *[1] * (new.dim() - 1)), new, old) for new, old in zip(got, s["out"])]


def run(state):
    if not own:
        return _plain(state)
    if state["op"] == "product":
        return state["layer"](state["x"], scale=state["x_scale"])
    from yolo_amd.class_probs import log_probs
    if state["rows"] is None:
        got = log_probs(state["z"], state["ids"], top=state["top"])
    else:
        got = log_probs(state["head"], state["ids"], top=state["top"], rows=state["rows"], classes=state["classes"], out=state["out"])
    return [v for v in got if v is not None]


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def work(case):
    size = {"bf16": 2, "f32": 4, "i8": 1}
    if case["op"] == "product":
        m, k, n = case["rows"], case["k"], case["n"]
        b = m * k * size[case["x"]] + (4 * m if case["x"] == "i8" else 0) + n * k + 4 * n + m * n * size[case["out"]]
        return {"bytes": b + (4 * n if case["bias"] else 0), "flops": 2 * m * k * n}
    if case["op"] == "probs":
        n, es = case["rows"], size[case["dtype"]]
    else:
        n, es = case["rows"] if case["op"] == "kept" else case["cells"] * case["anchors"], 4
    read = n * (2 / 3 if case["op"] == "kept" else 1) * case["classes"] * es + (8 * n if case["op"] == "kept" else 0)
    return {"bytes": read + n * (4 + 4 + 4 + 8 * case["top"]), "flops": 6 * n * case["classes"]}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "product":
        if s["x_scale"] is None:
            # the integers follow the rule's own 32-bit product x * (127 / a): a value next to the border of two could
            # otherwise be either
            a = torch.linalg.vector_norm(s["x"].to(F32), ord=math.inf, dim=1).clamp(min=TINY)
            q, unit = torch.round(s["x"].to(F32) * (127.0 / a)[:, None]).to(F64), a.to(F64) / 127
        else:
            q, unit = s["x"].to(F64), s["x_scale"].to(F64)
        y = (q @ s["w"].to(F64).T).mul_(unit[:, None]).mul_(s["w_scale"].to(F64)[None])
        if s["b"] is not None:
            y += s["b"].to(F64)
        return torch.maximum(y, 0.1 * y) if case["leaky"] else y
    z = s["z"]
    if s["rows"] is not None:
        idx = torch.nonzero(s["rows"] >= 0)[:, 0]
        first = s["rows"][idx]
        z = torch.stack([s["head"].view(-1)[first + j] for j in range(case["classes"])], 1)
        ids = s["ids"][idx]
    else:
        ids = s["ids"]
    x = z.to(F64)
    lp = x - torch.logsumexp(x, -1, keepdim=True)
    p = torch.exp(lp)
    got = [lp.take_along_dim(ids.long()[..., None], -1)[..., 0], -(p * lp).sum(-1)]
    del p
    if case["top"]:
        v, at = torch.sort(x, dim=-1, descending=True, stable=True)
        got += [at[..., :case["top"]].to(torch.int32), lp.take_along_dim(at[..., :case["top"]], -1)]
    if s["rows"] is None:
        return got
    full = []
    for new, old in zip(got, s["out"]):
        o = old.to(new.dtype)
        o[idx] = new
        full.append(o)
    return full
