"""-m gpu: the 8-bit product (y3_quantize_rows_i8, y3_linear_i8*) against its definition.

The integers are compared exactly (the rule's own 32-bit arithmetic in numpy), the outputs against int64 sums and 64-bit
scaling.  Roundings of an output: the integer sum to fp32, times t_n, the fused multiply-add with s_m and b_n, the leaky
product (2^-24 of the product or the result each), and half a step of the output type."""
import numpy as np
import pytest
import torch

from yolo_amd import _lib
from yolo_amd.linear_i8 import Int8Linear, quantize_rows

pytestmark = pytest.mark.gpu
TINY = np.float32(127 * 2.0 ** -126)
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
U = 2.0 ** -24


def rule(x):
    """(q, s) of float32 rows by the definition, in float32 like the definition."""
    x = np.asarray(x, dtype=np.float32)
    a = np.maximum(np.abs(x).max(axis=1), TINY)
    with np.errstate(invalid="ignore", over="ignore"):
        q = np.rint(x * (np.float32(127) * (np.float32(1) / a))[:, None])
    bad = ~np.isfinite(x).all(axis=1)
    q[bad] = 0
    s = a / np.float32(127)
    s[bad] = np.nan
    return q.astype(np.int64), s


def want(q, s, w, t, b, leaky):
    """64-bit result (the sums are whole numbers below 2^53: exact) and the magnitude that its roundings refer to."""
    p = (q.astype(np.float64) @ w.T.astype(np.float64)) * t.astype(np.float64)[None] * s.astype(np.float64)[:, None]
    y = p + (b.astype(np.float64)[None] if b is not None else 0.0)
    return (np.where(y > 0, y, 0.1 * y) if leaky else y), np.abs(p) + np.abs(y)


def close(got, y, size, out):
    got = got.float().cpu().numpy().astype(np.float64)
    half = 2.0 ** -8 if out == "bf16" else U
    bound = 4 * U * size + half * np.abs(y) * (1 + 4 * U) + 2.0 ** -133
    assert np.array_equal(np.isnan(got), np.isnan(y))
    off = np.abs(got - y) - bound
    assert not (off > 0).any(), "worst %g over the bound at %r" % (np.nanmax(off), np.unravel_index(np.nanargmax(off), off.shape))


def layer_of(rng, n, k, bias, leaky, out):
    w = rng.integers(-127, 128, (n, k)).astype(np.int64)
    t = (np.exp(rng.normal(size=n)) / 127 / np.sqrt(k)).astype(np.float32)
    b = rng.normal(size=n).astype(np.float32) if bias else None
    lay = Int8Linear(torch.from_numpy(w.astype(np.int8)), bias=b, scale=t, leaky=leaky, out_dtype=DT[out])
    return lay, w, t, b


def rows_of(rng, rows, k):
    return (rng.normal(size=(rows, k)) * np.exp(rng.normal(size=(1, k))) * np.exp(rng.normal(size=(rows, 1)))).astype(np.float32)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 7), (5, 64), (17, 255), (33, 512), (2, 1000), (9, 2047), (4, 4096), (2, 20003)])
def test_quantize_rows(dt, rows, k):
    rng = np.random.default_rng(rows * 1000 + k)
    x = torch.from_numpy(rows_of(rng, rows, k)).to(DT[dt])
    if rows > 2:
        x[1] = 0                                            # a row of zeros
        x[2] = 1e-39 if dt == "f32" else 1e-38              # ... and one below the smallest scale
    q, s = quantize_rows(x.cuda())
    wq, ws = rule(x.float().numpy())
    assert q.dtype == torch.int8 and q.shape == (rows, k) and s.shape == (rows,)
    np.testing.assert_array_equal(q.cpu().numpy(), wq)
    np.testing.assert_array_equal(s.cpu().numpy(), ws)
    # what the pair stands for is within half a step of x (127 steps, four roundings of the quotient)
    step = ws.astype(np.float64)[:, None]
    assert (np.abs(wq * step - x.double().numpy()) <= step * (0.5 + 127 * 4 * U)).all()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_quantize_rows_ties_nonfinite_strides(dt):
    x = torch.zeros(8, 40)
    x[0, :5] = torch.tensor([127.0, 0.5, 1.5, -0.5, -2.5])   # scale 1: halves go to the even integer
    x[1, 3] = float("nan")
    x[2, 39] = float("inf")
    x[3, 0] = float("-inf")
    x[4] = torch.finfo(DT[dt]).max
    x[5, 1::2] = -3e38
    x = x.to(DT[dt])
    wide = torch.full((8, 57), 9.0, dtype=DT[dt], device="cuda")
    wide[:, 11:51] = x.cuda()                               # rows at odd addresses
    for t in (x.cuda(), wide[:, 11:51], x.cuda().t().contiguous().t(), x.cuda().view(2, 4, 40)):
        q, s = quantize_rows(t)
        wq, ws = rule(x.float().numpy())
        np.testing.assert_array_equal(q.cpu().numpy().reshape(8, 40), wq)
        np.testing.assert_array_equal(s.cpu().numpy().reshape(8), ws)


SHAPES = [(1, 1, 1), (1, 64, 16), (2, 63, 15), (3, 129, 17), (15, 1000, 255), (16, 4096, 33), (17, 128, 64), (31, 300, 100),
          (64, 256, 255), (65, 512, 256), (100, 1024, 512), (130, 777, 300), (257, 128, 257), (300, 2048, 48), (513, 640, 520),
          (1, 8192, 200), (40, 5000, 96), (700, 1500, 700)]


@pytest.mark.parametrize("rows,k,n", SHAPES)
@pytest.mark.parametrize("x,out", [("f32", "f32"), ("bf16", "bf16"), ("i8", "f32"), ("i8", "bf16"), ("bf16", "f32")])
def test_product(rows, k, n, x, out):
    rng = np.random.default_rng(rows + 7 * k + 11 * n)
    bias, leaky = (rows + n) % 2 == 1, (k + n) % 3 != 0
    lay, w, t, b = layer_of(rng, n, k, bias, leaky, out)
    xs = torch.from_numpy(rows_of(rng, rows, k))
    if x == "i8":
        q = rng.integers(-128, 128, (rows, k))
        s = np.exp(rng.normal(size=rows)).astype(np.float32)
        got = lay(torch.from_numpy(q.astype(np.int8)).cuda(), scale=torch.from_numpy(s).cuda())
    else:
        xs = xs.to(DT[x])
        q, s = rule(xs.float().numpy())
        got = lay(xs.cuda())
    assert got.dtype == DT[out] and got.shape == (rows, n)
    close(got, *want(q, s, w, t, b, leaky), out)


@pytest.mark.parametrize("rows,k,n,x,out", [(33000, 512, 256, "bf16", "bf16"), (32769, 256, 255, "bf16", "f32"), (40000, 128, 128, "bf16", "bf16"),
                                            (32768, 300, 200, "f32", "bf16"), (50001, 100, 64, "f32", "f32"), (33001, 768, 128, "bf16", "bf16"),
                                            (35000, 650, 77, "bf16", "f32"), (33333, 384, 128, "bf16", "bf16"), (32800, 511, 129, "f32", "f32"),
                                            (60000, 64, 255, "bf16", "bf16"), (34000, 768, 250, "bf16", "bf16"), (33007, 256, 255, "f32", "f32"),
                                            (33005, 500, 129, "bf16", "bf16"), (32801, 128, 1, "bf16", "f32"), (33003, 40, 3, "f32", "bf16")])
def test_product_of_very_many_rows(rows, k, n, x, out):
    """Panels of rows under weights that stay where they are; wide rows, ragged last panels, odd channels."""
    rng = np.random.default_rng(rows)
    bias, leaky = n % 2 == 1, k % 3 != 0
    lay, w, t, b = layer_of(rng, n, k, bias, leaky, out)
    wide = torch.zeros(rows, k + 24, dtype=DT[x], device="cuda")
    xs = torch.from_numpy(rows_of(rng, rows, k)).to(DT[x])
    xs[5, 3] = float("nan")
    wide[:, 16:16 + k] = xs.cuda()
    q, s = rule(xs.float().numpy())
    got = lay(wide[:, 16:16 + k])
    ref, size = want(q, s, w, t, b, leaky)
    close(got, ref, size, out)
    assert torch.isnan(got[5]).all() and not torch.isnan(got[6:]).any()
    assert torch.equal(lay(xs.cuda()[rows - 70:]), got[rows - 70:])


@pytest.mark.parametrize("rows,k,n", [(10001, 200, 520), (16500, 700, 3001), (9003, 120, 1000), (5000, 130, 1500), (3700, 2300, 1040), (10100, 600, 300),
                                     (500, 500, 2000), (731, 6624, 352), (200, 6600, 352), (731, 4096, 500), (5690, 2704, 48),
                                     (1700, 3669, 176), (700, 3000, 256), (300, 9000, 30),
                                     (130, 2600, 4000), (6000, 400, 200)])
@pytest.mark.parametrize("x,out", [("bf16", "bf16"), ("i8", "f32"), ("f32", "f32")])
def test_product_of_the_middle_range(rows, k, n, x, out):
    """Blocks of 32, 48 and 64 rows by one to four blocks of channels a wave; ragged last ones."""
    rng = np.random.default_rng(rows + n)
    bias, leaky = rows % 2 == 1, k % 200 == 0
    lay, w, t, b = layer_of(rng, n, k, bias, leaky, out)
    if x == "i8":
        q = rng.integers(-128, 128, (rows, k))
        s = np.exp(rng.normal(size=rows)).astype(np.float32)
        got = lay(torch.from_numpy(q.astype(np.int8)).cuda(), scale=torch.from_numpy(s).cuda())
    else:
        xs = torch.from_numpy(rows_of(rng, rows, k)).to(DT[x])
        q, s = rule(xs.float().numpy())
        got = lay(xs.cuda())
    close(got, *want(q, s, w, t, b, leaky), out)


@pytest.mark.parametrize("rows,k,n", [(4100, 640, 2100), (3000, 512, 3001), (8200, 1037, 1025), (2300, 4096, 4100)])
@pytest.mark.parametrize("x,out", [("bf16", "bf16"), ("i8", "f32"), ("i8", "bf16"), ("f32", "f32")])
def test_product_of_many_rows_and_channels(rows, k, n, x, out):
    """Enough 256 x 256 tiles to fill the card; odd numbers of k-steps, ragged last tiles, more tiles than CUs."""
    rng = np.random.default_rng(rows + n)
    bias, leaky = n % 2 == 1, k % 2 == 0
    lay, w, t, b = layer_of(rng, n, k, bias, leaky, out)
    if x == "i8":
        q = rng.integers(-128, 128, (rows, k))
        s = np.exp(rng.normal(size=rows)).astype(np.float32)
        got = lay(torch.from_numpy(q.astype(np.int8)).cuda(), scale=torch.from_numpy(s).cuda())
    else:
        xs = torch.from_numpy(rows_of(rng, rows, k)).to(DT[x])
        q, s = rule(xs.float().numpy())
        got = lay(xs.cuda())
    close(got, *want(q, s, w, t, b, leaky), out)


@pytest.mark.parametrize("rows,k,n", [(1, 64, 32), (20, 100, 30), (70, 256, 255), (400, 300, 77), (300, 1024, 256)])
@pytest.mark.parametrize("x", ["f32", "bf16", "i8"])
def test_product_strides_and_guard(rows, k, n, x):
    """Rows inside wider buffers at odd offsets, outputs inside a wider buffer: nothing beside them is written."""
    rng = np.random.default_rng(rows)
    lay, w, t, b = layer_of(rng, n, k, True, True, "f32")
    if x == "i8":
        q = rng.integers(-127, 128, (rows, k))
        s = np.exp(rng.normal(size=rows)).astype(np.float32)
        wide = torch.full((rows, k + 13), 77, dtype=torch.int8, device="cuda")
        wide[:, 5:5 + k] = torch.from_numpy(q.astype(np.int8)).cuda()
        scale = torch.from_numpy(s).cuda()
    else:
        xs = torch.from_numpy(rows_of(rng, rows, k)).to(DT[x])
        q, s = rule(xs.float().numpy())
        wide = torch.full((rows, k + 13), 7.0, dtype=DT[x], device="cuda")
        wide[:, 5:5 + k] = xs.cuda()
        scale = None
    buf = torch.full((rows + 2, n + 9), -5.0, device="cuda")
    view = buf[1:-1, 3:3 + n]
    got = lay(wide[:, 5:5 + k], scale=scale, out=view)
    assert got is view
    close(got, *want(q, s, w, t, b, True), "f32")
    rest = buf.clone()
    rest[1:-1, 3:3 + n] = -5.0
    assert (rest == -5.0).all()


def test_product_rows_are_independent_and_nan_stays_in_its_row():
    rng = np.random.default_rng(5)
    for rows, k, n in [(6, 256, 48), (200, 512, 128), (3, 5000, 64), (700, 1500, 600)]:
        lay, w, t, b = layer_of(rng, n, k, True, False, "bf16")
        x = torch.from_numpy(rows_of(rng, rows, k)).to(torch.bfloat16).cuda()
        y = lay(x)
        bad = x.clone()
        bad[1, k - 1] = float("nan")
        bad[2, 0] = float("inf")
        z = lay(bad)
        assert torch.isnan(z[1:3]).all()
        keep = [0] + list(range(3, rows))
        assert torch.equal(z[keep], y[keep])
        assert torch.equal(lay(x[rows - 1:]), y[rows - 1:])     # alone, whichever kernel that takes: same bits
        assert torch.equal(lay(x.view(1, rows, k)), y.view(1, rows, n))


def test_product_from_one_quantisation_equals_the_product_of_rows():
    rng = np.random.default_rng(6)
    for rows, k in [(1, 100), (50, 256), (300, 1000)]:
        a, b = layer_of(rng, 96, k, True, True, "bf16")[0], layer_of(rng, 33, k, False, False, "f32")[0]
        x = torch.from_numpy(rows_of(rng, rows, k)).cuda()
        r = quantize_rows(x)
        assert torch.equal(a(x), a(r.values, scale=r.scale))
        assert torch.equal(b(x), b(r.values, scale=r.scale))


@pytest.mark.parametrize("rows,k,n", [(1, 17, 5), (2, 4141, 1048), (11, 9001, 40), (100, 5001, 64), (300, 65, 257), (7195, 1742, 178), (400, 1003, 2000),
                                      (3000, 300, 600), (9000, 100, 300), (40, 20001, 16), (5000, 601, 2100)])
@pytest.mark.parametrize("first,extra", [(0, 0), (1, 2), (16, 15), (5, 16)])
def test_eight_bit_rows_anywhere(rows, k, n, first, extra):
    """8-bit rows at odd addresses and pitches, the last one up to the end of its buffer."""
    rng = np.random.default_rng(rows + k)
    lay, w, t, b = layer_of(rng, n, k, True, False, "f32")
    q = rng.integers(-128, 128, (rows, k))
    s = np.exp(rng.normal(size=rows)).astype(np.float32)
    flat = torch.full((first + rows * (k + extra) - extra,), 99, dtype=torch.int8, device="cuda")
    x = flat[first:].as_strided((rows, k), (k + extra, 1))
    x.copy_(torch.from_numpy(q.astype(np.int8)))
    close(lay(x, scale=torch.from_numpy(s).cuda()), *want(q, s, w, t, b, False), "f32")


def test_float_weights_are_quantised_per_channel():
    rng = np.random.default_rng(7)
    w = rows_of(rng, 40, 200)
    w[3] = 0
    for dt in ("f32", "bf16"):
        wt = torch.from_numpy(w).to(DT[dt])
        lay = Int8Linear(wt, out_dtype=torch.float32)
        wq, ws = rule(wt.float().numpy())
        np.testing.assert_array_equal(lay.scale.cpu().numpy(), ws)
        x = torch.from_numpy(rows_of(rng, 10, 200))
        q, s = rule(x.numpy())
        close(lay(x.cuda()), *want(q, s, wq, ws, None, False), "f32")


def test_more_rows_than_a_grid():
    rows, k = (1 << 27) + 77, 16
    x = torch.randint(-128, 128, (rows, k), dtype=torch.int8, device="cuda")
    for n in (1, 40):
        if n == 40:
            x = x[: (1 << 23) + 5]
        w = torch.arange(n * k).view(n, k) % 7 - 3
        lay = Int8Linear(w.to(torch.int8), scale=torch.full((n,), 2.0 ** -8), out_dtype=torch.bfloat16)
        got = lay(x, scale=torch.ones(x.shape[0], device="cuda"))
        for lo in range(0, x.shape[0], 1 << 24):
            part = x[lo:lo + (1 << 24)].float() @ w.float().cuda().t() * 2.0 ** -8           # (integers below 2^24: exact)
            assert torch.equal(got[lo:lo + (1 << 24)], part.bfloat16())


@pytest.mark.parametrize("rows,k,n,x", [(1200007, 2048, 16, "bf16"), (17500001, 128, 64, "bf16"), (70001, 32768, 16, "bf16"), (9000001, 128, 256, "f32"),
                                        (540001, 8192, 300, "i8"), (9, 100, 40, "bf16")])
def test_rows_past_32_bits(rows, k, n, x):
    """Inputs of more than 4 GB, of which the first and last rows are looked at; few rows on a pitch of 2^30 elements."""
    rng = np.random.default_rng(k)
    lay, w, t, b = layer_of(rng, n, k, True, True, "f32")
    if rows == 9:
        xs = torch.zeros(9 << 30, dtype=torch.bfloat16, device="cuda").as_strided((9, k), (1 << 30, 1))
    else:
        xs = torch.zeros(rows, k, dtype=torch.int8 if x == "i8" else DT[x], device="cuda")
    m = min(rows, 100)
    head, tail = torch.from_numpy(rows_of(rng, m, k)), torch.from_numpy(rows_of(rng, m, k))
    if x == "i8":
        head, tail = (torch.from_numpy(rng.integers(-128, 128, (m, k)).astype(np.int8)) for _ in range(2))
    head, tail = head.to(xs.dtype), tail.to(xs.dtype)
    xs[:m], xs[-m:] = head.cuda(), tail.cuda()
    if rows == m:
        head = tail
    s = torch.full((rows,), 0.5, device="cuda") if x == "i8" else None
    got = lay(xs, scale=s)
    for part, y in ((head, got[:m]), (tail, got[-m:])):
        q, sc = (part.numpy(), np.full(m, 0.5, np.float32)) if x == "i8" else rule(part.float().numpy())
        close(y, *want(q, sc, w, t, b, True), "f32")


def test_tiles_past_32_bits():
    rows, k, n = 40001, 512, 60001
    w = torch.randint(-128, 128, (n, k), dtype=torch.int8, device="cuda")
    x = torch.randint(-128, 128, (rows, k), dtype=torch.int8, device="cuda")
    got = Int8Linear(w, scale=torch.full((n,), 2.0 ** -6, device="cuda"))(x, scale=torch.ones(rows, device="cuda"))
    for lo in range(0, rows, 8000):
        part = x[lo:lo + 8000].float() @ w.float().t() * 2.0 ** -6                           # (integers below 2^24: exact)
        assert torch.equal(got[lo:lo + 8000], part.bfloat16())


@pytest.mark.parametrize("k", [130, 20])
def test_very_many_channels(k):
    """2^24 channels: weights and outputs past 32-bit offsets."""
    n, rows = 1 << 24, 65
    if k == 130:                                             # 8-bit weights
        w = torch.randint(-128, 128, (n, k), dtype=torch.int8, device="cuda")
        lay = Int8Linear(w, scale=torch.full((n,), 2.0 ** -6, device="cuda"))
    else:                                                    # float weights that are their own 8-bit values
        w = torch.randint(-126, 127, (n, k), dtype=torch.int8, device="cuda")
        w[:, 3] = 127
        lay = Int8Linear(w.float() * 2.0 ** -6, out_dtype=torch.bfloat16)
        assert torch.equal(lay.scale, torch.full((n,), 2.0 ** -6, device="cuda"))
    x = torch.randint(-128, 128, (rows, k), dtype=torch.int8, device="cuda")
    got = lay(x, scale=torch.ones(rows, device="cuda"))
    for lo in range(0, n, 1 << 22):
        part = x.float() @ w[lo:lo + (1 << 22)].float().t() * 2.0 ** -6                      # (integers below 2^24: exact)
        assert torch.equal(got[:, lo:lo + (1 << 22)], part.bfloat16())


def test_sum_at_the_ends_of_32_bits():
    k = 131071
    for xv, wv in ((-128, -128), (127, -128), (-128, 127)):
        lay = Int8Linear(torch.full((17, k), wv, dtype=torch.int8), scale=torch.full((17,), 2.0 ** -20), out_dtype=torch.float32)
        y = lay(torch.full((2, k), xv, dtype=torch.int8, device="cuda"), scale=torch.ones(2, device="cuda"))
        assert (y.cpu() == np.float32(xv * wv * k) * np.float32(2.0 ** -20)).all()


def test_empty_and_refusals():
    lay = Int8Linear(torch.ones(8, 32), out_dtype=torch.float32)
    assert lay(torch.empty(0, 32, device="cuda")).shape == (0, 8)
    x = torch.ones(4, 32, device="cuda")
    s = torch.ones(4, device="cuda")
    for bad in (lambda: lay(x[:, :31]), lambda: lay(x.half()), lambda: lay(x.cpu()), lambda: lay(x, scale=s),
                lambda: lay(x.to(torch.int8)), lambda: lay(x.to(torch.int8), scale=s[:3]), lambda: lay(x.to(torch.int8).view(2, 2, 32), scale=s.view(1, 4)),
                lambda: lay(x, out=torch.empty(4, 8, dtype=torch.bfloat16, device="cuda")),
                lambda: lay(x, out=torch.empty(4, 9, device="cuda")), lambda: lay(x, out=torch.empty(8, 4, device="cuda").t()),
                lambda: lay(x.clone().requires_grad_()), lambda: Int8Linear(torch.ones(8, 32), scale=torch.ones(8)),
                lambda: Int8Linear(torch.ones(8, 32).to(torch.int8)), lambda: Int8Linear(torch.ones(8, 32), out_dtype=torch.float16),
                lambda: Int8Linear(torch.ones(8, 32), bias=torch.ones(7)), lambda: Int8Linear(torch.ones(8)),
                lambda: quantize_rows(x.half()), lambda: quantize_rows(x.cpu())):
        with pytest.raises(ValueError):
            bad()
    buf = torch.zeros(4 * 40, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        lay(buf[:128].view(4, 32), out=buf[100:132].view(4, 8))


@pytest.mark.parametrize("rows,k,n", [(1, 4096, 512), (30, 8192, 64), (361, 1024, 512), (3000, 256, 255), (1200, 2500, 600), (33000, 256, 128)])
def test_streams_and_graph_replays(rows, k, n):
    """Two layers of one input on two streams at once, then a captured run replayed on changing inputs, eager work between."""
    rng = np.random.default_rng(rows)
    a, b = layer_of(rng, n, k, True, True, "bf16")[0], layer_of(rng, n, k, False, False, "f32")[0]
    xs = [torch.from_numpy(rows_of(rng, rows, k)).to(torch.bfloat16).cuda() for _ in range(4)]
    wa, wb = [a(x) for x in xs], [b(x) for x in xs]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for x in xs:
        with torch.cuda.stream(s1):
            ya = a(x)
        with torch.cuda.stream(s2):
            yb = b(x)
        got.append((ya, yb))
    torch.cuda.synchronize()
    for (ya, yb), ra, rb in zip(got, wa, wb):
        assert torch.equal(ya, ra) and torch.equal(yb, rb)
    x = xs[0].clone()
    graphs = []
    for lay in (a, b):                                       # two graphs that replay one after the other
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = lay(x)
        graphs.append((g, y))
    for i in (1, 2, 3, 0):
        x.copy_(xs[i])
        graphs[0][0].replay()
        other = a(xs[(i + 1) % 4])                           # eager work between the replays
        graphs[1][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], wa[i]) and torch.equal(graphs[1][1], wb[i]) and torch.equal(other, wa[(i + 1) % 4])


def test_layer_is_called_from_two_threads():
    import threading
    rng = np.random.default_rng(9)
    lay = layer_of(rng, 128, 300, True, True, "f32")[0]
    xs = [torch.from_numpy(rows_of(rng, 50 + i, 300)).cuda() for i in range(2)]
    ref = [lay(x) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                y = lay(xs[i])
                torch.cuda.current_stream().synchronize()
                if not torch.equal(y, ref[i]):
                    bad.append(i)
    th = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in th]
    [t.join() for t in th]
    assert not bad


def test_workspace_too_small_is_refused():
    import ctypes
    lib = _lib.load()
    d = _lib.LinearI8Desc()
    d.dtype, d.out_dtype, d.k, d.n, d.rows, d.x_ld, d.out_ld = _lib.Y3_F32, _lib.Y3_F32, 5000, 64, 3000, 5000, 64
    _lib.check(lib.y3_linear_i8_layout(ctypes.byref(d)))
    need = ctypes.c_int64(0)
    _lib.check(lib.y3_linear_i8_workspace_bytes(ctypes.byref(d), ctypes.byref(need)))
    assert need.value > 0
    t = torch.zeros(16, device="cuda")
    p = t.data_ptr()
    assert lib.y3_linear_i8(ctypes.byref(d), p, None, p, p, None, p + (1 << 40), p, need.value - 1, None) == -1      # (never touched)
    assert b"workspace" in lib.y3_last_error()
