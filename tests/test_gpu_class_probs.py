"""-m gpu: y3_log_probs against the formulas in 64 bits.

Bounds, with u = 2^-24 and L = 1 + log C: an exponential is off by at most (3 |d| + 3) u of itself (d and its product with
log2 e rounded, the constant, the instruction), and sum(e |d|) / Z <= L, so Z is off by (3 L + 3 + adds) u of itself with at
most C / 64 + 8 additions on the way of a term; log Z adds 2 u log Z, the differences u of their result.  S = sum e d has
the same with one factor |d| more (sum e d^2 / Z <= L^2 + 1)."""
import numpy as np
import pytest
import torch

from yolo_amd.class_probs import log_probs

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def plain(z, ids, top):
    """64 bits, on the CPU: logp, entropy, top ids, top logp (rows of -inf and NaN by the definition)."""
    z = z.double().cpu()
    C = z.shape[-1]
    lp = torch.log_softmax(z, -1)
    dead = (z == -np.inf).all(-1)
    lp[dead] = -np.inf
    p = lp.exp()
    H = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    nan = torch.isnan(z).any(-1) | (z == np.inf).any(-1)
    H[nan] = np.nan
    lp[nan] = np.nan
    at = torch.sort(z, dim=-1, descending=True, stable=True).indices[..., :top]
    idc = ids.long().cpu()
    logp = torch.gather(lp, -1, idc.clamp(0, C - 1)[..., None])[..., 0]
    logp = torch.where(idc < 0, torch.zeros_like(logp), torch.where(idc >= C, torch.full_like(logp, np.nan), logp))
    return logp, H, at, torch.gather(lp, -1, at), lp


def check(got, z, ids, top):
    C = z.shape[-1]
    logp, H, at, tlp, _ = plain(z, ids, top)
    L = 1 + np.log(C)
    adds = C / 64 + 8

    def near(a, b, size):
        a = a.double().cpu()
        assert a.shape == b.shape
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a == -np.inf, b == -np.inf)
        fine = torch.isfinite(b)
        off = (a[fine] - b[fine]).abs() - U * (3 * L + 3 + adds + 2 * L + 3 * b[fine].abs()) * size
        assert not (off > 0).any(), off.max()
    near(got.logp, logp, 1)
    near(got.entropy, H, 1 + 2 * L)
    if top:
        assert torch.equal(got.top_ids.cpu().long(), at)
        near(got.top_logp, tlp, 1)
    else:
        assert got.top_ids is None and got.top_logp is None


CLASSES = [1, 2, 3, 7, 15, 16, 17, 20, 63, 64, 65, 80, 81, 127, 128, 200, 255, 256, 300, 512, 777, 1000, 1024, 1025, 2047, 4096,
           5000, 8193, 20000, 32001, 70001, 131072]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("C", CLASSES)
def test_sizes(C, dt):
    g = torch.Generator().manual_seed(C)
    rows = 5 if C > 1000 else 37
    z = (3 * torch.randn(rows, C, generator=g)).to(DT[dt])
    ids = torch.randint(0, C, (rows,), generator=g)
    top = min(C, [1, 5, 20, 32][C % 4])
    check(log_probs(z.cuda(), ids.cuda(), top=top), z, ids, top)
    check(log_probs(z.cuda(), ids.int().cuda()), z, ids, 0)


@pytest.mark.parametrize("rows,C,top", [(1, 80, 3), (2, 50000, 32), (64, 32000, 5), (300, 6000, 1), (1000, 1500, 8), (5000, 80, 5),
                                        (3, 130001, 20), (700, 257, 32), (700, 520, 31), (700, 1023, 20)])
def test_rows(rows, C, top):
    g = torch.Generator().manual_seed(rows)
    z = 4 * torch.randn(rows, C, generator=g)
    ids = torch.randint(0, C, (rows,), generator=g)
    check(log_probs(z.cuda(), ids.cuda(), top=top), z, ids, top)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("C", [5, 80, 300, 700, 1024, 1500, 3000, 6000, 40000])
def test_hard_rows(C, dt):
    """Ties, masks of -inf and of the type's lowest value, rows that a mask leaves empty, NaN and infinities, large offsets,
    one class far above the rest, all mass in one lane's stretch, rising and falling rows."""
    low = torch.finfo(DT[dt]).min
    g = torch.Generator().manual_seed(C)
    z = torch.randn(18, C, generator=g)
    z[0] = 0
    z[1] = torch.randint(0, 3, (C,), generator=g).float()
    z[2] = -np.inf
    z[3] = -np.inf
    z[3, C // 2] = 1.5
    z[4] = low
    z[5, ::2] = low
    z[6, torch.rand(C, generator=g) < 0.7] = -np.inf
    z[7, C - 1] = np.nan
    z[8, 0] = np.inf
    z[9] += 3e4
    z[10, C // 3] = 90.0
    z[11] = torch.arange(C) * (8.0 / C)
    z[12] = -torch.arange(C) * (8.0 / C)
    z[13] = torch.where(torch.arange(C) < 8, 5.0, -5.0)
    z[14] = torch.finfo(DT[dt]).max
    z[15] = torch.where(torch.arange(C) % 2 == 0, 0.0, -0.0)
    z[16] = np.nan
    z[17, : C // 2] = -np.inf
    z[17, 1] = np.nan
    z = z.to(DT[dt])
    ids = torch.randint(0, C, (18,), generator=g)
    ids[0] = -1
    ids[1] = C
    ids[2] = 0
    ids[3] = C // 2
    ids[10] = C // 3
    top = min(C, 12)
    got = log_probs(z.cuda(), ids.cuda(), top=top)
    finite = [i for i in range(18) if i not in (7, 8, 16, 17)]
    pick = torch.tensor(finite)
    check(type(got)(*[v[pick.cuda()] for v in got]), z[pick], ids[pick], top)
    for i in (7, 8, 16, 17):
        assert torch.isnan(got.logp[i]) and torch.isnan(got.entropy[i]) and torch.isnan(got.top_logp[i]).all()
        assert ((got.top_ids[i] >= 0) & (got.top_ids[i] < C)).all() and got.top_ids[i].unique().numel() == top


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("C", [8192, 16384, 32768, 32775, 41221, 65537])
def test_rows_a_little_longer_than_whole_chunks(C, dt):
    g = torch.Generator().manual_seed(C)
    z = (3 * torch.randn(9, C + 3, generator=g)).to(DT[dt])
    z[4, C - 20:] = 9.0
    z[5, : C - 20] = -np.inf
    ids = torch.randint(0, C, (9,), generator=g)
    for top in (1, 20, 32):
        check(log_probs(z.cuda()[:, 3:], ids.cuda(), top=top), z[:, 3:], ids, top)
        check(log_probs(z.cuda()[:, :C], ids.cuda(), top=top), z[:, :C], ids, top)


@pytest.mark.parametrize("top", [1, 2, 7])
@pytest.mark.parametrize("C", [80, 777, 1030, 4117, 9000, 33000])
def test_equal_largest_logits(C, top):
    """Several classes with the row's largest logit: the first ones, whatever ran on the card before."""
    g = torch.Generator().manual_seed(C)
    rows = 500
    z = torch.randn(rows, C, generator=g).to(torch.bfloat16)
    for r in range(rows):
        z[r, torch.randperm(C, generator=g)[: r % 12]] = 6.0
    ids = torch.randint(0, C, (rows,), generator=g)
    zc, ic = z.cuda(), ids.cuda()
    for before in (100.0, -100.0):
        log_probs(torch.full((4096, max(C, 2000)), before, device="cuda"), None, top=32)
        check(log_probs(zc, ic, top=top), z, ids, top)


@pytest.mark.parametrize("rows,C,ld", [(34001, 65536, 65536), (30000001, 80, 80), (5, 700, 1 << 30), (5, 5000, 1 << 30)])
def test_rows_past_32_bits(rows, C, ld):
    """More than 2^31 logits, of which the first and last rows are looked at."""
    g = torch.Generator().manual_seed(C)
    z = torch.zeros(rows * ld, dtype=torch.bfloat16, device="cuda").as_strided((rows, C), (ld, 1))
    m = min(rows, 50)
    ends = [(3 * torch.randn(m, C, generator=g)).to(torch.bfloat16) for _ in range(2)]
    z[:m], z[-m:] = ends[0].cuda(), ends[1].cuda()
    if rows == m:
        ends[0] = ends[1]
    ids = torch.randint(0, C, (rows,), generator=g).int().cuda()
    got = log_probs(z, ids, top=3)
    for part, at in ((ends[0], slice(0, m)), (ends[1], slice(rows - m, rows))):
        check(type(got)(*[v[at] for v in got]), part, ids[at].cpu(), 3)


def test_strides():
    g = torch.Generator().manual_seed(1)
    C = 80
    head = 2 * torch.randn(6, 5, 4, 256, generator=g)
    boxes = head[..., :255].view(6, 5, 4, 3, 85)[..., 5:]
    ids = torch.randint(0, C, boxes.shape[:-1], generator=g)
    dev = head.cuda()
    view = dev[..., :255].unflatten(-1, (3, 85))[..., 5:]
    assert not view.is_contiguous()
    for top in (0, 4):
        check(log_probs(view, ids.cuda(), top=top), boxes, ids, top)
    for t, ref in ((view[:, 0], boxes[:, 0]), (view[2:3, 1:2, 0, 1], boxes[2:3, 1:2, 0, 1]), (view[0, 0, 0, 0], boxes[0, 0, 0, 0]),
                   (view.permute(3, 0, 1, 2, 4), boxes.permute(3, 0, 1, 2, 4)), (view[0, 0, 0, :1].expand(7, C), boxes[0, 0, 0, :1].expand(7, C)),
                   (view[0, 0].transpose(0, 2), boxes[0, 0].transpose(0, 2))):
        i = torch.randint(0, ref.shape[-1], ref.shape[:-1], generator=g)
        check(log_probs(t, i.cuda(), top=2), ref, i, 2)
    wide = torch.randn(9, 3001, generator=g).to(torch.bfloat16)
    i = torch.randint(0, 2990, (9,), generator=g)
    check(log_probs(wide.cuda()[:, 7:2997], i.cuda(), top=9), wide[:, 7:2997], i, 9)
    assert log_probs(wide.cuda()[:0], i.cuda()[:0], top=2).top_ids.shape == (0, 2)


@pytest.mark.parametrize("C", [80, 3000])
def test_rows_by_offset(C):
    """Gathered rows: the same row twice, skipped rows left as they were, rows that reach behind the tensor."""
    g = torch.Generator().manual_seed(C)
    base = torch.randn(50 * C + 13, generator=g)
    off = torch.randint(0, base.numel() - C + 1, (200,), generator=g)
    off[3] = off[4]
    off[5] = base.numel() - C
    off[7::11] = -1
    far = [9, 20]
    off[9], off[20] = base.numel() - C + 1, 1 << 60
    ids = torch.randint(0, C, (200,), generator=g)
    out = (torch.full((200,), -1.0).cuda(), torch.full((200,), -2.0).cuda(), torch.full((200, 5), -3, dtype=torch.int32).cuda(),
           torch.full((200, 5), -4.0).cuda())
    got = log_probs(base.cuda(), ids.cuda(), top=5, rows=off.cuda(), classes=C, out=out)
    assert all(a is b for a, b in zip(got, out))
    skip = off < 0
    for v, fill in zip(got, (-1, -2, -3, -4)):
        assert (v.cpu()[skip] == fill).all()
    assert torch.isnan(got.logp.cpu()[far]).all() and torch.isnan(got.entropy.cpu()[far]).all()
    assert (got.top_ids.cpu()[far] == -1).all() and torch.isnan(got.top_logp.cpu()[far]).all()
    ok = ~skip
    ok[far] = False
    pick = ok.nonzero()[:, 0]
    z = torch.stack([base[o:o + C] for o in off[pick].tolist()])
    check(type(got)(*[v[pick.cuda()] for v in got]), z, ids[pick], 5)
    fresh = log_probs(base.cuda(), ids.cuda(), top=5, rows=off.cuda(), classes=C)
    assert (fresh.top_ids.cpu()[skip] == -1).all() and (fresh.logp.cpu()[skip] == 0).all()
    assert torch.equal(fresh.logp.cpu()[ok], got.logp.cpu()[ok])


def test_refusals():
    z = torch.zeros(4, 80, device="cuda")
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    rows = torch.zeros(4, dtype=torch.int64, device="cuda")
    f = torch.zeros(4, device="cuda")
    for bad in (lambda: log_probs(z.cpu(), ids), lambda: log_probs(z.half(), ids), lambda: log_probs(z, ids[:3]), lambda: log_probs(z, ids.float()),
                lambda: log_probs(z, ids, top=33), lambda: log_probs(z, ids, top=-1), lambda: log_probs(z[:, :3], ids, top=4),
                lambda: log_probs(z, ids, rows=rows), lambda: log_probs(z, ids, classes=80), lambda: log_probs(z, ids, rows=rows.int(), classes=80),
                lambda: log_probs(z.t(), ids, rows=rows, classes=4), lambda: log_probs(z[:, :0], ids), lambda: log_probs(z.requires_grad_(), ids),
                lambda: log_probs(z.detach(), ids, out=(f[:3], f, None, None)), lambda: log_probs(z.detach(), ids, out=(None, f, None, None)),
                lambda: log_probs(z.detach(), ids, top=1, out=(f, f, None, None))):
        with pytest.raises(ValueError):
            bad()


def test_outputs_in_the_logits_are_refused():
    buf = torch.zeros(40 * 85, device="cuda")
    z = buf.view(40, 85)[:, :80]
    good = [torch.empty(40, device="cuda"), torch.empty(40, device="cuda"), None, None]
    log_probs(z, torch.zeros(40, dtype=torch.int64, device="cuda"), out=tuple(good))
    good[1] = buf[85 * 39 + 40 - 1:][:40]
    with pytest.raises(ValueError, match="overlap"):
        log_probs(z, torch.zeros(40, dtype=torch.int64, device="cuda"), out=tuple(good))


@pytest.mark.parametrize("rows,C", [(1, 128000), (16, 40000), (3000, 80)])
def test_streams_and_graph_replays(rows, C):
    g = torch.Generator().manual_seed(rows)
    zs = [torch.randn(rows, C, generator=g).cuda() for _ in range(4)]
    ids = torch.randint(0, C, (rows,), generator=g).cuda()
    ref = [log_probs(z, ids, top=6) for z in zs]
    torch.cuda.synchronize()
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))  # noqa: E731
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, z in enumerate(zs * 3):
        with torch.cuda.stream(streams[i % 2]):
            got.append(log_probs(z, ids, top=6))
    torch.cuda.synchronize()
    assert all(same(r, ref[i % 4]) for i, r in enumerate(got))
    z = zs[0].clone()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            r = log_probs(z, ids, top=6)
        graphs.append((gr, r))
    for i in (1, 2, 3, 0):
        z.copy_(zs[i])
        graphs[0][0].replay()
        other = log_probs(zs[(i + 1) % 4], ids, top=6)
        graphs[1][0].replay()
        torch.cuda.synchronize()
        assert same(graphs[0][1], ref[i]) and same(graphs[1][1], ref[i]) and same(other, ref[(i + 1) % 4])
