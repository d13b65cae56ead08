"""linear_xent on the GPU against its definition in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

import tail_ref as ref

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def rows_apart(t, dev, pad, off=0, fill=math.nan):
    """t on the device, its rows pad elements apart and off elements behind a boundary, `fill` between them."""
    r, c = t.shape
    buf = torch.full((off + r * (c + pad),), fill, dtype=t.dtype, device=dev)
    v = buf[off:].view(r, c + pad)[:, :c]
    v.copy_(t)
    return v


def problem(r, v, d, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn((v, d), generator=g) * (1.5 / math.sqrt(d))
    labels = torch.randint(0, v, (r,), generator=g, dtype=torch.int32)
    x = spread * torch.randn((r, d), generator=g) + 4.0 * torch.rand((r, 1), generator=g) * w[labels.long()]
    return x.to(DT[dtype]), w.to(DT[dtype]), labels, g


def call(C, dev, x, w, labels, rw=None, outs="all", piece=0, pad=0, off=0, dw_type=None, stream=0, w_pad=None,
         w_off=0):
    """(loss, dX, dW, row loss) on the CPU; outputs behind and between rows must stay as they were."""
    r, d = x.shape
    v = w.shape[0]
    dt = x.dtype
    xd = rows_apart(x, dev, pad, off)
    wd = rows_apart(w, dev, pad if w_pad is None else w_pad, w_off)
    n = C.linear_xent_scratch(max(r, 1), v, d, dt, outs != "loss", piece)
    if (pad or off or w_pad or w_off) and d % 8 == 0:  # room for a copy of a piece's rows of W
        n += (piece or v + 256) * (-(-d // 64) * 64) * 4
    scratch = torch.full((n // 4,), math.nan, device=dev)
    loss, rl = torch.full((1,), math.nan, device=dev), torch.full((r,), math.nan, device=dev)
    mark = 7.0
    dx = rows_apart(torch.full((r, d), math.nan, dtype=dt), dev, pad, off, mark)
    dw = rows_apart(torch.full((v, d), math.nan, dtype=dw_type or dt), dev, pad, off, mark)
    o = {"loss": [loss, rl], "dx": [loss, dx, rl], "all": [loss, dx, dw, rl]}[outs] + [scratch]
    ins = [xd, wd, labels.to(dev)] + ([rw.to(dev)] if rw is not None else [])
    C.op_call(C.OpKind.LinearXent, ins, o, 0, b"", stream)
    if pad or off:
        for t in (dx, dw):
            whole = t._base
            inside = torch.zeros_like(whole, dtype=torch.bool)
            inside[off:].view(t.shape[0], d + pad)[:, :d] = True
            assert (whole[~inside] == mark).all()
    return loss.cpu(), dx.cpu(), dw.cpu(), rl.cpu()


def check(got, x, w, labels, rw=None, outs="all"):
    loss, dx, dw, rl, bt, bx, bw, bl = ref.linear_xent(x, w, labels, rw)
    far = (got[3].double() - rl).abs()
    assert (far <= bl).all(), (far / bl.clamp(min=1e-300)).max()
    assert abs(float(got[0]) - float(loss)) <= bt
    if outs == "loss":
        return
    far, b = (got[1].double() - dx).abs(), ref.rounded(bx, dx, x.dtype)
    assert (far <= b).all(), ((far / b).max(), (far > b).sum())
    if outs == "all":
        far, b = (got[2].double() - dw).abs(), ref.rounded(bw, dw, got[2].dtype)
        assert (far <= b).all(), ((far / b).max(), (far > b).sum())


SIZES = [(1, 1, 1), (1, 5, 3), (2, 300, 64), (5, 129, 7), (32, 1000, 96), (33, 700, 128), (64, 513, 200), (65, 257, 64),
         (128, 2049, 192), (130, 1003, 72), (257, 4099, 128)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("r,v,d", SIZES)
def test_sizes(C, dev, r, v, d, dtype):
    x, w, labels, _ = problem(r, v, d, dtype, r + v + d)
    for outs in ("loss", "dx", "all"):
        check(call(C, dev, x, w, labels, outs=outs), x, w, labels, outs=outs)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_rows_that_do_not_count(C, dev, dtype):
    """Labels out of range and weights of 0, with NaN and infinities in those rows; weights of either sign."""
    for r, v, d in ((7, 300, 64), (70, 1030, 100), (300, 2000, 64)):
        x, w, labels, g = problem(r, v, d, dtype, r)
        rw = torch.randn(r, generator=g)
        labels[0], labels[3], labels[4] = -1, v, 2 ** 31 - 1
        labels[5] = -2 ** 31
        rw[1], rw[6] = 0.0, -0.0
        xx = x.clone()
        xx[[0, 3, 4, 5]] = math.nan
        xx[1, 0], xx[6, :] = math.inf, -math.inf
        for out in ("loss", "all"):
            got = call(C, dev, xx, w, labels, rw, outs=out)
            check(got, x, w, labels, rw, outs=out)
            assert (got[3][[0, 1, 3, 4, 5, 6]] == 0).all()
            if out == "all":
                assert (got[1][[0, 1, 3, 4, 5, 6]] == 0).all()
        xx = x.clone()
        xx[[0, 3, 4, 5]] = math.nan
        check(call(C, dev, xx, w, labels), x, w, labels)  # the mean over the others


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_no_row_counts(C, dev, dtype):
    x, w, labels, _ = problem(40, 500, 64, dtype, 1)
    x[:] = math.nan
    for rw, lab in ((None, torch.full_like(labels, -1)), (torch.zeros(40), labels)):
        got = call(C, dev, x, w, lab, rw)
        assert all((t == 0).all() for t in got)
    got = call(C, dev, x[:0], w, labels[:0])  # and no row at all
    assert float(got[0]) == 0 and (got[2] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("r,v,d,piece", [(40, 1003, 64, 256), (200, 2100, 128, 512), (3, 3000, 72, 1024),
                                         (300, 1300, 100, 256), (64, 5000, 192, 4864)])
def test_pieces(C, dev, r, v, d, piece, dtype):
    """Scratch for a part of the classes: the others' logits are computed twice."""
    x, w, labels, g = problem(r, v, d, dtype, piece)
    rw = torch.rand(r, generator=g) + 0.1
    labels[0], labels[1], labels[2] = v - 1, piece - 1, piece
    check(call(C, dev, x, w, labels, rw, piece=piece), x, w, labels, rw)
    check(call(C, dev, x, w, labels, rw, "dx", piece=piece), x, w, labels, rw, "dx")
    check(call(C, dev, x, w, labels, rw, "loss", piece=piece), x, w, labels, rw, "loss")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("pad,off", [(8, 0), (1, 0), (3, 5), (64, 16)])
def test_rows_apart(C, dev, pad, off, dtype):
    """Rows any distance apart at any element, NaN between them; nothing between the outputs' rows is written."""
    for r, v, d, piece in ((40, 700, 64, 0), (150, 600, 128, 256), (33, 300, 50, 256)):
        x, w, labels, _ = problem(r, v, d, dtype, pad + off)
        check(call(C, dev, x, w, labels, pad=pad, off=off, piece=piece), x, w, labels)
        check(call(C, dev, x, w, labels, piece=piece, w_pad=pad, w_off=off), x, w, labels)


def test_repeated_rows(C, dev):
    """X and W as broadcast views: every row the same memory."""
    x, w, labels, _ = problem(20, 300, 64, "bf16", 4)
    xd, wd = x[:1].to(dev).expand(20, 64), w[:1].to(dev).expand(300, 64)
    n = C.linear_xent_scratch(20, 300, 64, torch.bfloat16) // 4 + 512 * 64
    outs = [torch.empty(1, device=dev), torch.empty((20, 64), device=dev, dtype=torch.bfloat16),
            torch.empty((300, 64), device=dev, dtype=torch.bfloat16), torch.empty(20, device=dev)]
    C.op_call(C.OpKind.LinearXent, [xd, wd, labels.to(dev)], outs + [torch.empty(n, device=dev)])
    check([o.cpu() for o in outs], xd.cpu().contiguous(), wd.cpu().contiguous(), labels)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_f32_weight_gradient(C, dev, dtype):
    for r, v, d, pad in ((70, 1003, 64, 0), (300, 900, 100, 3)):
        x, w, labels, _ = problem(r, v, d, dtype, 5)
        got = call(C, dev, x, w, labels, dw_type=torch.float32, pad=pad)
        assert got[2].dtype == torch.float32
        check(got, x, w, labels)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("r,v,d", [(600, 25000, 64), (1025, 13001, 256), (4096, 4096, 96), (129, 70000, 64),
                                   (2500, 3001, 512)])
def test_large_tiles(C, dev, r, v, d, dtype):
    """Enough rows and classes for the largest tiles, whole and in pieces; the definition on the device."""
    x, w, labels, g = problem(r, v, d, dtype, r)
    labels[::5] = -1
    want = [t.cpu() if isinstance(t, torch.Tensor) else t
            for t in ref.linear_xent(*(t.to(dev) for t in (x, w)), labels.to(dev))]
    for piece in (0, -(-v // 512) * 256):
        got = call(C, dev, x, w, labels, piece=piece)
        loss, dx, dw, rl, bt, bx, bw, bl = want
        assert ((got[3].double() - rl).abs() <= bl).all() and abs(float(got[0]) - float(loss)) <= bt
        assert ((got[1].double() - dx).abs() <= ref.rounded(bx, dx, x.dtype)).all()
        assert ((got[2].double() - dw).abs() <= ref.rounded(bw, dw, x.dtype)).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_logits_far_from_zero(C, dev, dtype):
    """Every logit of a row shifted by some hundreds, whole tiles far below the rest, certain labels."""
    r, v, d = 48, 1500, 64
    x, w, labels, g = problem(r, v, d, dtype, 3)
    shift = torch.linspace(-300, 300, r)
    x[:, 0], w[:, 0] = shift.to(x.dtype), 1.0
    w[256:800, 1], x[:, 1] = -200.0, 1.0
    w[labels[:8].long(), 2] = 60.0
    x[:8, 2], x[8:, 2] = 1.0, 0.0
    check(call(C, dev, x, w, labels), x, w, labels)
    check(call(C, dev, x, w, labels, piece=512), x, w, labels)


def test_infinite_and_missing_logits(C, dev):
    """Classes of logit -inf have probability 0; a row of nothing else, a NaN and +inf give a NaN row and its label's share."""
    r, v, d = 40, 700, 64
    for dtype in ("bf16", "f32"):
        x, w, labels, g = problem(r, v, d, dtype, 6)
        x[:, 3], w[:, 3] = 0.0, 0.0
        x[:, 3] = 1.0
        w[300:600, 3] = -math.inf  # masked classes: whole tiles and parts of tiles
        labels[:] = torch.randint(0, 300, (r,), generator=g, dtype=torch.int32)
        for piece in (0, 256):
            got = call(C, dev, x, w, labels, piece=piece)
            # dX in every column but the masking one (0 times infinity there), dW of the classes that are not masked
            keep = [c for c in range(d) if c != 3]
            ok = torch.ones(v, dtype=torch.bool)
            ok[300:600] = False
            loss, dx, dw, rl, bt, bx, bw, bl = ref.linear_xent(x, w[ok], labels)
            assert ((got[3].double() - rl).abs() <= bl).all() and abs(float(got[0]) - float(loss)) <= bt
            assert ((got[1].double() - dx).abs() <= ref.rounded(bx, dx, x.dtype))[:, keep].all()
            assert ((got[2].double()[ok] - dw).abs() <= ref.rounded(bw, dw, x.dtype)).all()
            assert (got[2][~ok] == 0).all()
        x, w, labels, g = problem(r, v, d, dtype, 7)
        x[2, 5] = math.nan
        got = call(C, dev, x, w, labels)
        assert got[3][2].isnan() and got[1][2].isnan().all() and got[0].isnan() and got[2].isnan().all()
        rest = [i for i in range(r) if i != 2]
        assert not got[3][rest].isnan().any() and not got[1][rest].isnan().any()
        w[5, :], x, labels = -math.inf, x[rest].abs() + 0.1, labels[rest]  # class 5 is impossible
        labels[0] = 5
        got = call(C, dev, x, w, labels, outs="loss")
        assert got[3][0] == math.inf and not got[3][1:].isnan().any()


def test_gradient_against_differences(C, dev):
    """dX and dW against the loss, by central differences along random directions of length h.  The loss is off by
    bt on either side; the third derivative along a direction that moves each logit by at most s is at most 2 s^3."""
    r, v, d = 24, 500, 48
    x, w, labels, g = problem(r, v, d, "f32", 8)
    rw = torch.rand(r, generator=g)
    _, dx, dw, _ = call(C, dev, x, w, labels, rw)
    h = 2.0 ** -6
    bt = ref.linear_xent(x, w, labels, rw)[4]
    for k in range(4):
        a = torch.sign(torch.randn((r, d), generator=g)) * (k % 2 == 0) / d
        b = torch.sign(torch.randn((v, d), generator=g)) * (k % 2 == 1) / d
        up = call(C, dev, x + h * a, w + h * b, labels, rw, "loss")[0].double()
        down = call(C, dev, x - h * a, w - h * b, labels, rw, "loss")[0].double()
        slope = (dx.double() * a).sum() + (dw.double() * b).sum()
        s = h * max((a.abs() @ w.abs().t()).max(), (x.abs() @ b.abs().t()).max())
        moved = (x + h * a - x - h * a).abs().max() + (w + h * b - w - h * b).abs().max()  # roundings of the points
        off = float(moved) * (float(dx.abs().sum()) + float(dw.abs().sum())) / h
        assert abs((up - down) / (2 * h) - slope) <= (2 * bt / (2 * h) + 2 * s ** 3 * rw.sum() / (6 * h) + off
                                                      + 1e-5 * slope.abs() + 1e-6)


def test_same_bits_again_and_on_another_stream(C, dev):
    for dtype, r, v, d, piece in (("bf16", 300, 3000, 128, 0), ("f16", 20, 5000, 64, 1024), ("f32", 70, 900, 40, 0)):
        x, w, labels, _ = problem(r, v, d, dtype, 9)
        one = call(C, dev, x, w, labels, piece=piece)
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            two = call(C, dev, x, w, labels, piece=piece)
        s.synchronize()
        for a, b in zip(one, two):
            assert torch.equal(a, b)


def test_two_captured_calls(C, dev):
    """Two graphs with scratch of their own, replayed in turn with new rows, labels and numbers of rows that count."""
    r, v, d = 70, 1500, 128
    sets = []
    for k in range(2):
        x, w, labels, g = problem(r, v, d, "bf16", 20 + k)
        ins = [x.to(dev), w.to(dev), labels.to(dev)]
        outs = [torch.empty(1, device=dev), torch.empty((r, d), device=dev, dtype=torch.bfloat16),
                torch.empty((v, d), device=dev, dtype=torch.bfloat16), torch.empty(r, device=dev)]
        sc = torch.empty(C.linear_xent_scratch(r, v, d, torch.bfloat16, True, 768 if k else 0) // 4, device=dev)
        h = C.graph_create()
        C.op_call(C.OpKind.LinearXent, ins, outs + [sc], 0, b"", C.graph_begin_h(h))
        C.graph_end_h(h)
        sets.append((h, ins, outs))
    for i in range(4):
        for k, (h, ins, outs) in enumerate(sets):
            x, w, labels, g = problem(r, v, d, "bf16", 100 * i + k)
            labels[: 20 * i] = -1
            for t, n in zip(ins, (x, w, labels)):
                t.copy_(n)
            for t in outs:
                t.fill_(math.nan)
            C.graph_launch_h(h)
            piece = 768 if k else 0
            eager = call(C, dev, x, w, labels, piece=piece)
            torch.cuda.synchronize()
            for a, b in zip(outs, eager):
                assert torch.equal(a.cpu(), b)
    for h, _, _ in sets:
        C.graph_destroy(h)


def test_other_device_and_types_are_refused(C, dev):
    x, w, labels, _ = problem(8, 50, 64, "bf16", 1)
    outs = [torch.empty(1, device=dev), torch.empty(8, device=dev), torch.empty(1 << 20, device=dev)]
    with pytest.raises(RuntimeError):
        C.op_call(C.OpKind.LinearXent, [x.to(dev), w.float().to(dev), labels.to(dev)], outs)
    with pytest.raises(RuntimeError):
        C.op_call(C.OpKind.LinearXent, [x.to(dev), w.to(dev), labels.to(dev)], outs[:2] + [outs[2][:64]])
    with pytest.raises(RuntimeError):
        C.op_call(C.OpKind.LinearXent, [x, w.to(dev), labels.to(dev)], outs)


@pytest.mark.parametrize("dtype,dw_type", [("bf16", None), ("f16", None), ("f32", None), ("bf16", torch.float32)])
@pytest.mark.parametrize("r,v,d,piece", [(200, 4099, 128, 512), (250, 3001, 512, 256), (256, 6000, 1024, 1536),
                                         (129, 5003, 200, 768), (500, 9001, 320, 256), (1, 2000, 64, 256)])
def test_gradient_held_in_dw(C, dev, r, v, d, piece, dtype, dw_type):
    """Few classes in scratch, and dW with room for more until its rows are written: some, half or all of the others,
    behind W in place and behind copies of its rows."""
    x, w, labels, g = problem(r, v, d, dtype, r + piece)
    rw = torch.rand(r, generator=g) + 0.1
    rw[r // 2] = 0.0
    check(call(C, dev, x, w, labels, rw, piece=piece, dw_type=dw_type), x, w, labels, rw)
    check(call(C, dev, x, w, labels, rw, piece=piece, dw_type=dw_type, w_pad=8, w_off=3), x, w, labels, rw)


@pytest.mark.parametrize("dtype,dw_type", [("bf16", None), ("f16", None), ("f16", torch.float32)])
@pytest.mark.parametrize("r,v,d,pad", [(1, 63, 8, 0), (3, 65, 520, 0), (31, 1000, 1024, 8), (64, 4100, 1032, 0),
                                       (65, 129, 504, 16), (128, 2050, 1536, 0), (129, 13000, 1000, 0),
                                       (256, 24600, 512, 0), (200, 17001, 776, 24)])
def test_few_rows(C, dev, r, v, d, pad, dtype, dw_type):
    """Up to 256 rows: dW by blocks of 64 classes, columns and classes that end inside a block."""
    x, w, labels, g = problem(r, v, d, dtype, r + d)
    rw = torch.rand(r, generator=g) + 0.1
    labels[r // 2] = v - 1
    if r > 4:
        labels[r - 1], rw[0] = -1, 0.0
    check(call(C, dev, x, w, labels, rw, pad=pad, dw_type=dw_type), x, w, labels, rw)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("r,v,d", [(1, 700, 64), (5, 3001, 136), (64, 2000, 256), (100, 5000, 72), (128, 4096, 128)])
def test_few_rows_keep_the_labels_values(C, dev, r, v, d, dtype):
    """To 128 rows the label's value of G counts with the bits of f32: a row of dW with one label is off by its own
    rounding, by that of the other rows' probabilities (twice half a step) and by f32's, here 2^-16 in all."""
    x, w, labels, g = problem(r, v, d, dtype, r + v)
    w = w / 4  # (no row is sure of another class)
    labels = torch.randperm(v, generator=g)[:r].to(torch.int32)
    rw = torch.rand(r, generator=g) + 0.3
    got = call(C, dev, x, w, labels, rw)
    _, dx, dw, _, _, _, _, _ = ref.linear_xent(x, w, labels, rw)
    p = torch.softmax(x.double() @ w.double().t(), 1) * rw.double()[:, None]
    at = labels.long()
    p[torch.arange(r), at] = 0.0
    h = ref.HALF_STEP[x.dtype]
    slack = 2.0 ** -16 * (rw.double()[:, None] * x.double().abs()) + 2.0 ** -36 * x.double().abs().sum(0)
    bound = h * dw[at].abs() + 3 * h * (p[:, at].t() @ x.double().abs()) + slack + ref.TINY[x.dtype]
    assert ((got[2].double()[at] - dw[at]).abs() <= bound).all()
    slack = 2.0 ** -16 * (rw.double()[:, None] * w.double()[at].abs()) + 2.0 ** -36 * w.double().abs().sum(0)
    bound = h * dx.abs() + 3 * h * (p @ w.double().abs()) + slack + ref.TINY[x.dtype]
    assert ((got[1].double() - dx).abs() <= bound).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_equal_weights_are_not_rounded(C, dev, dtype):
    """The mean over any number of rows: 1 / rows is in no product, so dW of a label keeps all but the rounding of
    the probabilities."""
    for r in (3, 131, 700):
        x, w, labels, g = problem(r, 2003, 64, dtype, r)
        w = w / 64  # probabilities of about 1 / 2003
        labels = torch.randperm(2003, generator=g)[:r].to(torch.int32)
        for rw in (None, torch.full((r,), 1.0 / r)):
            got = call(C, dev, x, w, labels, rw)
            _, _, dw, _, _, _, _, _ = ref.linear_xent(x, w, labels, rw)
            p = torch.softmax(x.double() @ w.double().t(), 1)
            at, h = labels.long(), ref.HALF_STEP[x.dtype]
            own = p[torch.arange(r), at]
            # label: 1 - p lies in [1/2, 1], off by at most a quarter of a step of 1 and at most by p itself
            far = torch.minimum(torch.full_like(own, h / 2), own)[:, None] * x.double().abs()
            p[torch.arange(r), at] = 0.0
            far = far + 3 * h * (p[:, at].t() @ x.double().abs()) + 2.0 ** -16 * x.double().abs()
            bound = h * dw[at].abs() + far / r + ref.TINY[x.dtype] + 2.0 ** -36 / r * x.double().abs().sum(0)
            assert ((got[2].double()[at] - dw[at]).abs() <= bound * (1 + h)).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("r,v,d", [(3, 700, 8), (20, 1000, 40), (60, 900, 72), (100, 3000, 136), (300, 2600, 200),
                                   (600, 25000, 72), (1025, 13001, 264), (4096, 4096, 104), (2000, 9001, 2056)])
def test_rows_of_w_that_end_inside_a_k_step(C, dev, r, v, d, dtype):
    """W read in place: what lies behind a row is the next one, here with infinities where no other row may see them
    (classes of probability 0)."""
    x, w, labels, g = problem(r, v, d, dtype, r + d)
    x[:, 0] = x[:, 0].abs() + 0.5
    dead = torch.arange(1, v, 7)
    w[dead, 0] = -math.inf
    w[dead, 1:] = 0.0
    labels[(labels.long() % 7) == 1] -= 1
    loss, rl = call(C, dev, x, w, labels, outs="loss")[0::3]
    ws, xs, alive = w.clone(), x, torch.ones(v, dtype=torch.bool)
    alive[dead] = False
    at = torch.cumsum(alive, 0) - 1  # the same classes without the dead ones
    want, _, _, wl, bt, _, _, bl = ref.linear_xent(xs, ws[alive], at[labels.long()].to(torch.int32))
    assert ((rl.double() - wl).abs() <= bl).all()
    assert abs(float(loss) - float(want)) <= bt
    w[dead] = 0.0
    w[dead, 0] = -4.0
    check(call(C, dev, x, w, labels, outs="all"), x, w, labels)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("r", [32768, 32769, 70001])
def test_many_rows(C, dev, r, dtype):
    """Rows counted by every workgroup, and above 32768 by one."""
    x, w, labels, g = problem(r, 300, 64, dtype, r)
    rw = torch.rand(r, generator=g) + 0.1
    rw[::5] = 0.0
    labels[2::3], labels[r - 1] = -1, 299
    check(call(C, dev, x, w, labels, rw), x, w, labels, rw)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [2.0 ** -105, 2.0 ** -95, -2.0 ** -20, 2.0 ** 90, -2.0 ** 101])
def test_weights_of_any_scale(C, dev, scale, dtype):
    """On both sides of where the largest weight is divided out."""
    for r in (30, 150):
        x, w, labels, g = problem(r, 600, 64, dtype, r)
        rw = (torch.rand(r, generator=g) + 0.5) * scale
        check(call(C, dev, x, w, labels, rw), x, w, labels, rw)
