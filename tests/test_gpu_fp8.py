"""quant_fp8 and gemm_fp8 on the GPU against their definitions in 64 bits."""
from __future__ import annotations

import math
import struct

import pytest
import torch

import head_ref as ref

pytestmark = pytest.mark.gpu
QFP8 = int.from_bytes(b"QFP8", "little")
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def strided(rows, cols, dtype, dev, pad=0, off=0, fill=None):
    """A [rows, cols] view with rows cols + pad apart, off elements into its buffer."""
    buf = torch.empty(rows * (cols + pad) + off + 64, device=dev, dtype=torch.uint8 if dtype.itemsize == 1 else dtype)
    if dtype.itemsize == 1:
        buf.fill_(0x7F)  # NaN around the matrix
        buf = buf.view(dtype)
    else:
        buf.fill_(math.nan if fill is None else fill)
    return buf[off:off + rows * (cols + pad)].view(rows, cols + pad)[:, :cols], buf


def quant(C, x, fp8, by, pow2, transposed, pad=0, off=0):
    dev, (r, c) = x.device, x.shape
    shape = lambda n, m: (n if by == "rows" else ref.blocks(n), ref.blocks(m))  # noqa: E731
    outs, bufs = [], []
    for n, m in ((r, c), (c, r))[:1 + transposed]:
        q, buf = strided(n, m, ref.FP8[fp8], dev, pad, off)
        outs += [q, torch.full(shape(n, m), math.nan, device=dev)]
        bufs.append((buf, n, m))
    C.op_call(C.OpKind.QuantFp8, [x], outs, QFP8, struct.pack("<i", int(pow2)))
    for buf, n, m in bufs:  # nothing around the codes is written
        raw = buf.view(torch.uint8).cpu()
        at = torch.ones(raw.numel(), dtype=torch.bool)
        at[off:off + n * (m + pad)].view(n, m + pad)[:, :m] = False
        assert (raw[at] == 0x7F).all()
    return outs


@pytest.mark.parametrize("by", ["rows", "blocks"])
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("dtype,fp8,pow2", [("bf16", "e4m3", False), ("f16", "e5m2", False), ("f32", "e4m3", True),
                                            ("f32", "e5m2", False), ("bf16", "e4m3", True)])
@pytest.mark.parametrize("r,c", [(1, 1), (3, 5), (1, 640), (128, 128), (129, 255), (257, 1000), (640, 130)])
def test_quant(C, dev, r, c, dtype, fp8, pow2, by, transposed):
    g = torch.Generator().manual_seed(r * 1000 + c)
    x = (torch.randn((r, c), generator=g) * torch.exp2(torch.randint(-8, 8, (r, 1), generator=g))).to(DT[dtype])
    pad, off = (0, 0) if (r + c) % 2 else (3, 1)
    xd, _ = strided(r, c, DT[dtype], dev, pad, off)
    xd.copy_(x)
    outs = quant(C, xd, fp8, by, pow2, transposed, pad, off)
    for k, y in enumerate((x, x.t().contiguous())[:1 + transposed]):
        q, s = outs[2 * k].cpu(), outs[2 * k + 1].cpu()
        wq, ws = ref.quant(y, fp8, by, pow2)
        if by == "rows" and r == 1 and not transposed:
            ws = ws.view_as(s)
        assert torch.equal(s, ws)
        assert torch.equal(q.view(torch.uint8), wq.view(torch.uint8))
        # against x itself: half a step of the 8-bit type, and the rounding of 1 / s and of the product
        e = ref.spread(s.double(), *y.shape)
        half, sub = (2.0 ** -4, 2.0 ** -10) if fp8 == "e4m3" else (2.0 ** -3, 2.0 ** -17)
        far = (q.float().double() * e - y.double()).abs()
        assert (far <= torch.maximum(half * y.double().abs(), sub * e) * (1 + 8 * ref.U)).all()


def test_quant_zero_tiny_and_not_finite(C, dev):
    x = torch.zeros((130, 384))
    x[0, 5], x[1, 130], x[2, 300] = math.nan, math.inf, -math.inf
    x[3, 0:3] = torch.tensor([1e-45, -1e-40, 2.0 ** -126])
    x[4, 256:] = 3.3e38
    for by in ("rows", "blocks"):
        for pow2 in (False, True):
            for k, y in enumerate((x, x.t().contiguous())):
                got = quant(C, x.to(dev), "e4m3", by, pow2, True)
                q, s = got[2 * k].cpu().float(), got[2 * k + 1].cpu()
                wq, ws = ref.quant(y, "e4m3", by, pow2)
                assert torch.equal(s.isnan(), ws.isnan()) and torch.equal(s.nan_to_num(7.0), ws.nan_to_num(7.0))
                assert torch.equal(q.isnan(), wq.float().isnan())
                assert torch.equal(q.nan_to_num(7.0), wq.float().nan_to_num(7.0))


def codes(r, c, fp8, by, g, dev, pad=0, off=0):
    q = (torch.randn((r, c), generator=g) * (ref.FMAX[fp8] / 4)).clamp(-ref.FMAX[fp8], ref.FMAX[fp8]).to(ref.FP8[fp8])
    s = torch.rand((r if by == "rows" else ref.blocks(r), ref.blocks(c)), generator=g) + 0.1
    qd, _ = strided(r, c, ref.FP8[fp8], dev, pad, off)
    qd.copy_(q)
    return q, s, qd, s.to(dev)


def check_gemm(C, dev, m, n, k, a8="e4m3", b8="e4m3", a_by="rows", b_by="blocks", out="f32", bias=False, pad=0, off=0,
               cpad=0, s_t=False, seed=0):
    g = torch.Generator().manual_seed(m * 7 + n * 3 + k + seed)
    a, sa, ad, sad = codes(m, k, a8, a_by, g, dev, pad, off)
    b, sb, bd, sbd = codes(n, k, b8, b_by, g, dev, pad, off)
    if s_t:  # scales stored column by column
        sad, sbd = sad.t().contiguous().t(), sbd.t().contiguous().t()
    bi = torch.randn(n, generator=g) * 100 if bias else None
    c, buf = strided(m, n, DT[out], dev, cpad, cpad)
    ins = [ad, sad, bd, sbd] + ([bi.to(dev)] if bias else [])
    C.op_call(C.OpKind.GemmFp8, ins, [c])
    want, mag = ref.gemm(a, sa, b, sb, bi)
    bound = ref.gemm_bound(want, mag, k, DT[out], None if out == "f32" else ref.group_max(a, sa, b, sb))
    got = c.cpu().double()
    far = (got - want).abs()
    ok = far <= bound
    if out == "f16":
        # 65520 and more (65504 is the largest, half a step above it) rounds to infinity; what the f32 sum
        # leaves open there may do either
        over = want.abs() + bound >= 65520
        ok = torch.where(over, (got == want.sign() * math.inf) | (ok & (want.abs() - bound < 65520)), ok)
    assert ok.all(), (far / bound)[~ok].max()
    if cpad:
        rest = torch.ones(buf.numel(), dtype=torch.bool)
        rest[cpad:cpad + m * (n + cpad)].view(m, n + cpad)[:, :n] = False
        assert buf.cpu()[rest].isnan().all()
    return c


SIZES = [(1, 1, 1), (1, 16, 128), (1, 257, 1000), (5, 40, 129), (16, 4096, 512), (17, 100, 640), (33, 65, 127),
         (64, 64, 256), (100, 130, 784), (128, 128, 128), (130, 300, 144), (255, 257, 1024), (300, 512, 2049),
         (513, 700, 384), (1024, 1024, 256)]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_gemm_sizes(C, dev, m, n, k):
    pad = -k % 16  # rows on 16-byte steps
    check_gemm(C, dev, m, n, k, pad=pad)
    check_gemm(C, dev, m, n, k, a_by="blocks", b_by="rows", out="bf16", bias=True, pad=pad, cpad=3)
    check_gemm(C, dev, m, n, k, a_by="rows", b_by="rows", out="f16", pad=pad + 16, s_t=True)


@pytest.mark.parametrize("m,n,k", [(1, 40, 300), (40, 50, 260), (200, 300, 513), (300, 300, 1000)])
def test_gemm_any_alignment(C, dev, m, n, k):
    """Rows that start at any byte, NaN codes beside and between the rows."""
    for pad, off in ((0, 0), (1, 0), (0, 3), (5, 9)):
        check_gemm(C, dev, m, n, k, pad=pad, off=off, cpad=1)


@pytest.mark.parametrize("a8", ["e4m3", "e5m2"])
@pytest.mark.parametrize("b8", ["e4m3", "e5m2"])
@pytest.mark.parametrize("m,n,k", [(3, 200, 256), (70, 60, 300), (300, 520, 640)])
def test_gemm_types(C, dev, a8, b8, m, n, k):
    check_gemm(C, dev, m, n, k, a8, b8, b_by="rows", pad=-k % 16)
    check_gemm(C, dev, m, n, k, a8, b8, a_by="blocks", out="bf16", pad=-k % 16)


def test_gemm_nan_stays_in_its_row_and_column(C, dev):
    for m, n, k in ((4, 40, 256), (300, 400, 384)):
        g = torch.Generator().manual_seed(3)
        a, sa, ad, sad = codes(m, k, "e4m3", "rows", g, dev)
        b, sb, bd, sbd = codes(n, k, "e4m3", "rows", g, dev)
        ad.view(torch.uint8)[2, 7] = 0x7F
        sbd[11, 1] = math.nan
        c = torch.empty((m, n), device=dev)
        C.op_call(C.OpKind.GemmFp8, [ad, sad, bd, sbd], [c])
        nan = torch.zeros((m, n), dtype=torch.bool)
        nan[2], nan[:, 11] = True, True
        assert torch.equal(c.isnan().cpu(), nan)


def test_gemm_same_bits_whatever_else_runs(C, dev):
    """A row's result does not depend on the other rows' values, and a call repeated gives its bits."""
    one = check_gemm(C, dev, 300, 512, 1024, out="f32")
    two = check_gemm(C, dev, 300, 512, 1024, out="f32")
    assert torch.equal(one, two)


def test_quantised_linear_and_its_gradients(C, dev):
    """A Linear layer in 8 bits, forward and backward, as a training step
    runs it: x and dy quantised both ways, w by blocks; against the same
    quantised values multiplied in 64 bits."""
    g = torch.Generator().manual_seed(5)
    B, din, dout = 200, 300, 260
    x, w, dy = (torch.randn(s, generator=g) for s in ((B, din), (dout, din), (B, dout)))
    pad = lambda n: -n % 16  # noqa: E731

    def both(t, by, fp8="e4m3"):
        r, c = t.shape
        f = lambda n: n if by == "rows" else ref.blocks(n)  # noqa: E731
        q, _ = strided(r, c, ref.FP8[fp8], dev, pad(c))
        qt, _ = strided(c, r, ref.FP8[fp8], dev, pad(r))
        s, st = torch.empty((f(r), ref.blocks(c)), device=dev), torch.empty((f(c), ref.blocks(r)), device=dev)
        C.op_call(C.OpKind.QuantFp8, [t.to(dev).to(torch.bfloat16)], [q, s, qt, st], QFP8, struct.pack("<i", 0))
        return q, s, qt, st

    xq, xs, xqt, xst = both(x, "rows")
    wq, ws, wqt, wst = both(w, "blocks")
    dq, ds, dqt, dst = both(dy, "rows", "e5m2")
    for ins, exact, rel in (([xq, xs, wq, ws], x @ w.t(), 0.06), ([dq, ds, wqt, wst], dy @ w, 0.1),
                            ([dqt, dst, xqt, xst], dy.t() @ x, 0.1)):
        c = torch.empty((ins[0].shape[0], ins[2].shape[0]), device=dev)
        C.op_call(C.OpKind.GemmFp8, ins, [c])
        want, mag = ref.gemm(*[t.cpu() for t in ins])
        assert ((c.cpu().double() - want).abs() <= ref.gemm_bound(want, mag, ins[0].shape[1], torch.float32)).all()
        # a code is off by half a step, 2^-4 (e4m3) or 2^-3 (e5m2): the product of two by at most 2^-4 + 2^-4
        # (2^-3 + 2^-4) of its terms' magnitudes, in the norm of many terms with either sign well below that
        assert (c.cpu() - exact).norm() <= rel * exact.norm()


def test_captured_and_on_another_stream(C, dev):
    """quant + gemm captured once, replayed over changing inputs, with eager work between the replays."""
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.empty((64, 512), device=dev, dtype=torch.bfloat16)
    q, s = torch.empty((64, 512), device=dev, dtype=torch.float8_e4m3fn), torch.empty((64, 4), device=dev)
    w = torch.randn((300, 512), device=dev, generator=g).to(torch.float8_e4m3fn)
    ws = torch.rand((3, 4), device=dev, generator=g) + 0.5
    c = torch.empty((64, 300), device=dev)

    def calls(stream=0):
        C.op_call(C.OpKind.QuantFp8, [x], [q, s], QFP8, struct.pack("<i", 0), stream)
        C.op_call(C.OpKind.GemmFp8, [q, s, w, ws], [c], stream=stream)

    h = C.graph_create()
    calls(C.graph_begin_h(h))
    C.graph_end_h(h)
    for i in range(4):
        x.copy_(torch.randn((64, 512), device=dev, generator=g))
        c.fill_(math.nan)
        C.graph_launch_h(h)
        got = c.clone()
        torch.cuda.synchronize()
        c.fill_(math.nan)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            calls()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, c) and not got.isnan().any()
    C.graph_destroy(h)


def test_empty(C, dev):
    q, s = torch.empty((0, 256), device=dev, dtype=torch.float8_e4m3fn), torch.empty((0, 2), device=dev)
    C.op_call(C.OpKind.QuantFp8, [torch.empty((0, 256), device=dev)], [q, s], QFP8, struct.pack("<i", 0))
    w, ws = torch.zeros((5, 256), device=dev).to(torch.float8_e4m3fn), torch.ones((1, 2), device=dev)
    C.op_call(C.OpKind.GemmFp8, [q, s, w, ws], [torch.empty((0, 5), device=dev)])


def test_refusals_name_the_op(C, dev):
    x = torch.zeros((8, 256), device=dev)
    q, s = torch.empty((8, 256), device=dev, dtype=torch.float8_e4m3fn), torch.empty((8, 2), device=dev)
    with pytest.raises(RuntimeError, match="quant_fp8"):
        C.op_call(C.OpKind.QuantFp8, [x], [q, s[:, :1]], QFP8, struct.pack("<i", 0))
    with pytest.raises(RuntimeError, match="quant_fp8"):
        C.op_call(C.OpKind.QuantFp8, [x.t()], [q, s], QFP8, struct.pack("<i", 0))
    with pytest.raises(RuntimeError, match="gemm_fp8"):
        C.op_call(C.OpKind.GemmFp8, [q, s, q, s], [torch.empty((8, 9), device=dev)])
    with pytest.raises(RuntimeError, match="dtype"):
        C.op_call(C.OpKind.GemmFp8, [q, s.double(), q, s], [torch.empty((8, 8), device=dev)])
