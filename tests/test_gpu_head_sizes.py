"""The 8-bit and vocabulary-head ops where a kernel's form changes and where
offsets pass 32 bits, against their definitions in 64 bits; refusals of sizes
beyond them."""
from __future__ import annotations

import math
import struct

import pytest
import torch

import head_ref as ref
from aicf_cuda import abi
from test_gpu_fp8 import DT, QFP8, check_gemm, codes
from test_gpu_head import check, distill, student
from test_head_ops import DISTILL, I32, At, refused

gpu = pytest.mark.gpu
DTOP = int.from_bytes(b"DTOP", "little")


# rows in registers of 64 .. 1024 threads, in 16 bits and f32; read in each pass beyond
@gpu
@pytest.mark.parametrize("v,dtype", [(v + d, t) for v in (512, 1024, 2048, 4096, 8192, 16384) for d in (0, 1)
                                     for t in ("bf16", "f32")]
                         + [(v + d, "f32") for v in (28672, 57344) for d in (-1, 0, 1)]
                         + [(v + d, "f16") for v in (32768, 65536, 131072) for d in (-7, 0, 1)] + [(300007, "bf16")])
def test_distill_row_forms(C, dev, v, dtype):
    z, t, ids, g = student(2, v, 8, dtype, v)
    labels = torch.randint(0, v, (2,), generator=g, dtype=torch.int32)
    labels[1] = v - 1
    ids[0, 0], ids[1, 0] = v - 1, 0
    for scratch, pad in ((0, 0), (0, 1), (64, 0)):
        check(distill(C, dev, z, t, ids, 2.0, 0.5, labels, scratch=scratch, pad=pad), z, t, ids, 2.0, 0.5, labels)


@gpu
@pytest.mark.parametrize("r,p,v", [(1, 2, 49152), (1, 64, 49151), (3, 5, 50021), (1, 64, 70000), (40, 64, 49153),
                                   (48, 3, 49999), (49, 64, 49999)])
def test_distill_shared_rows(C, dev, r, p, v):
    """A row shared by as many workgroups as the scratch and the rows allow."""
    z, t, ids, _ = student(r, v, 4, "bf16", r)
    check(distill(C, dev, z, t, ids, 1.0, 0.0, scratch=p), z, t, ids, 1.0, 0.0)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 50, 0.9, 0.02), (1.3, 0, 0.3, 0.1),
            (0.0, 0, 1.0, 0.0), (1.0, 256, 0.95, 0.0), (1.0, 257, 1.0, 0.0), (2.0, 1025, 0.99, 0.0),
            (1.0, 4000, 1.0, 0.0), (1.0, 0, 1.0, 0.2), (5.0, 0, 0.999, 0.0)]


def draw(C, dev, z, u, sets, scratch, off=0):
    r = z.shape[0]
    col = lambda i, dt=torch.float32: torch.tensor([s[i] for s in sets], dtype=dt, device=dev)  # noqa: E731
    tok, lp = torch.full((r,), -9, dtype=torch.int32, device=dev), torch.full((r,), math.nan, device=dev)
    outs = [tok, lp]
    if scratch:
        outs.append(torch.full((r * scratch + off,), -1, dtype=torch.int32, device=dev)[off:].view(r, scratch))
    C.op_call(C.OpKind.SampleRow, [z, u.to(dev), col(0), col(1, torch.int32), col(2), col(3)], outs)
    return tok.cpu(), lp.cpu()


def as_f32(s):
    return tuple(x if isinstance(x, int) else struct.unpack("<f", struct.pack("<f", x))[0] for x in s)


@gpu
@pytest.mark.parametrize("v,dtype", [(8191, "f32"), (8192, "bf16"), (8193, "f32"), (32003, "f16"), (32768, "f16"), (50021, "bf16"), (131072, "bf16"),

                                     (524288, "f32"), (524289, "bf16"), (1500001, "f32")])
def test_sample_forms(C, dev, v, dtype):
    """Rows of all settings together, whole and shared by workgroups."""
    g = torch.Generator().manual_seed(v)
    z = (torch.randn((len(SETTINGS), v), generator=g) * 2).to(DT[dtype])
    z[:, ::911] += 4
    u = torch.rand(len(SETTINGS), generator=g)
    want = [ref.sample(z[i], u[i].item(), *as_f32(s)) for i, s in enumerate(SETTINGS)]
    zd = z.to(dev)
    for scratch, at in ((0, 0), (8192, 0), (8194, 1), (8193, 0)):  # (an odd length or address is left unused)
        tok, lp = draw(C, dev, zd, u, SETTINGS, scratch, at)
        assert tok.tolist() == [t for t, _ in want]
        # v weights, each rounded to a multiple of 2^-S beside a sum of 1 or more; one rounding to f32
        off = v * 2.0 ** -(min(51, 62 - (v - 1).bit_length()) + 1)
        assert all(abs(a - b) <= 2.0 ** -24 * abs(b) + off for a, (_, b) in zip(lp.tolist(), want))


@gpu
def test_sample_of_many_long_rows(C, dev):
    """Several rows a CU: 256 threads go through rows longer than 16384 classes too."""
    for r, v in ((520, 20011), (513, 16385)):
        g = torch.Generator().manual_seed(v)
        z = (torch.randn((r, v), generator=g) * 2).bfloat16()
        z[::7, : v // 2] = 0.0
        u = torch.rand(r, generator=g)
        sets = [SETTINGS[i % len(SETTINGS)] for i in range(r)]
        tok, _ = draw(C, dev, z.to(dev), u, sets, 0)
        assert tok.tolist() == [ref.sample(z[i], u[i].item(), *as_f32(s))[0] for i, s in enumerate(sets)]


@gpu
def test_sample_shared_rows_of_equal_logits(C, dev):
    """More classes at the cut than any list holds; few finite ones; one; none."""
    v = 40000
    z = torch.full((6, v), 1.5)
    z[1, 100:] = -math.inf
    z[2] = -math.inf
    z[2, 31111] = -3.0
    z[3] = -math.inf
    z[4, ::2] = 1.0
    z[5] = math.nan
    z[5, 7::5000] = 2.0
    u = torch.tensor([0.999, 0.5, 0.2, 0.3, 0.7, 0.6])
    for s in SETTINGS:
        sets = [s] * 6
        want = [ref.sample(z[i], u[i].item(), *as_f32(s))[0] for i in range(6)]
        for scratch in (0, 8192):
            assert draw(C, dev, z.to(dev), u, sets, scratch)[0].tolist() == want, s


@gpu
@pytest.mark.parametrize("m,n,k", [(1, 8192, 256), (1, 8208, 272), (16, 8209, 256), (17, 4096, 300), (17, 4112, 300),
                                   (32, 4100, 1023), (32, 9001, 512), (33, 4100, 256), (5, 16384, 255)])
def test_gemm_of_few_rows(C, dev, m, n, k):
    """Workgroups of 16 columns, and tiles of 32 rows from some hundreds of those on."""
    for out, b_by in (("f32", "rows"), ("bf16", "blocks"), ("f16", "rows")):
        check_gemm(C, dev, m, n, k, b_by=b_by, out=out, bias=out != "f32", pad=-k % 16, cpad=1)
    check_gemm(C, dev, m, n, k, "e5m2", a_by="blocks", out="f32", pad=-k % 16, s_t=True)


@gpu
def test_many_rows(C, dev):
    """More rows than one launch takes, than a grid has workgroups for in one pass."""
    g = torch.Generator(device=dev).manual_seed(5)
    rnd = lambda *s: torch.randn(s, device=dev, generator=g)  # noqa: E731
    r, v = (1 << 21) + 5, 4
    z, t = rnd(r, v), rnd(r, 1)
    ids = torch.randint(-1, v, (r, 1), device=dev, generator=g).to(torch.int32)
    labels = torch.randint(-1, v + 1, (r,), device=dev, generator=g).to(torch.int32)
    w = torch.rand(r, device=dev, generator=g)
    loss, dz, rl = torch.empty(1, device=dev), torch.empty_like(z), torch.empty(r, device=dev)
    C.op_call(C.OpKind.DistillTopk, [z, t, ids, labels, w], [loss, dz, rl], DTOP, struct.pack("<ff", 1.0, 0.25))
    q = torch.log_softmax(z.double(), -1)
    col = torch.arange(v, device=dev)
    soft, hard = (ids >= 0), (labels >= 0)[:, None] & (labels < v)[:, None]
    at_t, at_l = (col == ids).double(), (col == labels[:, None]).double()
    want = w.double()[:, None] * (0.75 * soft * (q.exp() - at_t) + 0.25 * hard * (q.exp() - at_l))
    rows = -0.75 * (q * at_t).sum(-1) - 0.25 * (q * at_l).sum(-1)
    rows[w == 0] = 0  # (a row of weight 0 is left out: there is one)
    # terms of at most 1, some ten roundings each; a row's loss: log q of at most 12, as many
    assert ((dz.double() - want).abs() <= 16 * ref.U * w.double()[:, None]).all()
    assert ((rl.double() - rows).abs() <= 16 * ref.U * (rows + 1)).all()
    # the weighted rows are added in 64 bits
    total = (w.double() * rows).sum()
    assert abs(loss.item() - total) <= 16 * ref.U * (w.double() * (rows + 1)).sum() + ref.U * total

    x = rnd(5_000_001, 3)
    out, s = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=dev), torch.empty((x.shape[0], 1), device=dev)
    C.op_call(C.OpKind.QuantFp8, [x], [out, s], QFP8, struct.pack("<i", 0))
    for part in (slice(0, 1000), slice(4_999_001, None)):
        wq, ws = ref.quant(x[part].cpu(), "e4m3", "rows", False)
        assert torch.equal(out[part].cpu().view(torch.uint8), wq.view(torch.uint8)) and torch.equal(s[part].cpu(), ws)
    assert ((out.float() * s - x).abs() <= 2.0 ** -4 * x.abs() * (1 + 8 * ref.U) + 2.0 ** -10 * s).all()

    r = 100_003
    z, u = rnd(r, 3), torch.rand(r, device=dev, generator=g)
    one = torch.ones(r, device=dev)
    tok = torch.empty(r, dtype=torch.int32, device=dev)
    C.op_call(C.OpKind.SampleRow, [z, u, one, torch.zeros_like(tok), one, 0 * one], [tok])
    cum = torch.softmax(z.double(), -1).cumsum(-1)
    want = (cum[:, :2] <= u.double()[:, None]).sum(-1)
    near = ((cum[:, :2] - u.double()[:, None]).abs() < 1e-12).any(-1)  # (64-bit sums either way there)
    assert (near | (tok == want)).all()


@gpu
@pytest.mark.parametrize("m,n,k", [(70001, 1, 272), (1, 70001, 272), (33, 1, 256), (2, 1, 300)])
def test_gemm_of_one_row_or_column(C, dev, m, n, k):
    for out in ("f32", "bf16"):
        check_gemm(C, dev, m, n, k, b_by="rows", out=out, bias=True, pad=-k % 16)


@gpu
def test_scales_of_any_strides(C, dev):
    """One scale for all blocks, scales shared by rows, every second word; the same matrix as both operands."""
    g = torch.Generator().manual_seed(4)
    for m, k in ((9, 300), (200, 512)):
        a, sa, ad, sad = codes(m, k, "e4m3", "rows", g, dev, -k % 16)
        nb = ref.blocks(k)
        wide = torch.rand((m, 2 * nb), generator=g).to(dev)
        for s in (torch.full((1, 1), 0.5, device=dev).expand(m, nb), sad[:1].expand(m, nb), sad[:, :1].expand(m, nb),
                  wide[:, ::2]):
            c = torch.empty((m, m), device=dev)
            C.op_call(C.OpKind.GemmFp8, [ad, s, ad, s], [c])
            want, mag = ref.gemm(a, s.cpu(), a, s.cpu())
            assert ((c.cpu().double() - want).abs() <= ref.gemm_bound(want, mag, k, torch.float32)).all()
    for by in ("rows", "blocks"):  # scales written column by column, with a gap
        x = torch.randn((130, 500), generator=g)
        f = (lambda n: n) if by == "rows" else ref.blocks
        q, qt = (torch.empty(s, dtype=torch.float8_e5m2, device=dev) for s in ((130, 500), (500, 130)))
        s, st = (torch.full((b, r + 3), math.nan, device=dev).t()[:r] for b, r in ((4, f(130)), (2, f(500))))
        for outs in ([q, s], [q, s, qt, st]):
            C.op_call(C.OpKind.QuantFp8, [x.to(dev)], outs, QFP8, struct.pack("<i", 1))
            for i, y in enumerate((x, x.t().contiguous())[:len(outs) // 2]):
                wq, ws = ref.quant(y, "e5m2", by, True)
                assert torch.equal(outs[2 * i].cpu().view(torch.uint8), wq.view(torch.uint8))
                assert torch.equal(outs[2 * i + 1].cpu(), ws)
                behind = torch.as_strided(outs[2 * i + 1], (3, ws.shape[1]), outs[2 * i + 1].stride(), ws.shape[0])
                assert behind.isnan().all()


@gpu
def test_distill_of_rows_that_share_logits(C, dev):
    """Logits, teacher and classes of one row for all (row stride 0)."""
    for v in (700, 50001):
        z, t, ids, g = student(1, v, 6, "f16", v)
        r = 4
        labels = torch.randint(0, v, (r,), generator=g, dtype=torch.int32)
        loss, rl, dz = torch.empty(1, device=dev), torch.empty(r, device=dev), torch.empty((r, v), device=dev).half()
        ins = [x.to(dev).expand(r, -1) for x in (z, t, ids)] + [labels.to(dev)]
        C.op_call(C.OpKind.DistillTopk, ins, [loss, dz, rl, torch.empty((r, 8, 4), device=dev)], DTOP,
                  struct.pack("<ff", 1.5, 0.5))
        check((loss.cpu(), dz.cpu(), rl.cpu()), z.expand(r, -1), t.expand(r, -1), ids.expand(r, -1), 1.5, 0.5, labels)


FAR = 1_200_000_000  # elements between rows: the third starts beyond 2^31 of them


def far_apart(t, dev):
    """Three rows on the device, FAR elements (rounded to 16) apart."""
    ld = FAR // 16 * 16
    n = 2 * ld + t.shape[1]
    buf = torch.empty(n, dtype=torch.uint8 if t.dtype.itemsize == 1 else t.dtype, device=dev).view(t.dtype)
    v = torch.as_strided(buf, t.shape, (ld, 1))
    v.copy_(t)
    return v


@gpu
def test_offsets_past_32_bits(C, dev):
    g = torch.Generator().manual_seed(2)
    z, t, ids, _ = student(3, 1000, 5, "bf16", 3)
    zd, loss, rl = far_apart(z, dev), torch.empty(1, device=dev), torch.empty(3, device=dev)
    C.op_call(C.OpKind.DistillTopk, [zd, t.to(dev), ids.to(dev)], [loss, zd, rl], DTOP, struct.pack("<ff", 1.0, 0.0))
    check((loss.cpu(), zd.cpu(), rl.cpu()), z, t, ids, 1.0, 0.0)
    zd.copy_(z)
    u = torch.rand(3, generator=g)
    tok, _ = draw(C, dev, zd, u, SETTINGS[1:4], 0)
    assert tok.tolist() == [ref.sample(z[i], u[i].item(), *as_f32(SETTINGS[1 + i]))[0] for i in range(3)]
    del zd
    x = torch.randn((3, 300), generator=g).to(torch.bfloat16)
    xd = far_apart(x, dev)
    q, s = far_apart(torch.zeros((3, 300)).to(torch.float8_e4m3fn), dev), torch.empty((3, 3), device=dev)
    C.op_call(C.OpKind.QuantFp8, [xd], [q, s], QFP8, struct.pack("<i", 0))
    wq, ws = ref.quant(x, "e4m3", "rows", False)
    assert torch.equal(q.cpu().view(torch.uint8), wq.view(torch.uint8)) and torch.equal(s.cpu(), ws)
    b, sb, bd, sbd = codes(40, 300, "e4m3", "rows", g, dev)
    for rows in (False, True):  # far rows of A and C, far rows of B
        a8, b8 = ([bd, sbd], [q, s]) if rows else ([q, s], [bd, sbd])
        c = torch.empty((40, 3), device=dev) if rows else far_apart(torch.zeros((3, 40)), dev)
        C.op_call(C.OpKind.GemmFp8, a8 + b8, [c])
        want, mag = ref.gemm(b, sb, wq, ws) if rows else ref.gemm(wq, ws, b, sb)
        assert ((c.cpu().double() - want).abs() <= ref.gemm_bound(want, mag, 300, torch.float32)).all()


@gpu
def test_quant_of_more_than_2_31_elements(C, dev):
    """70000 x 32768: both ways by blocks and by rows; the last rows and columns are checked."""
    m, k = 70000, 32768
    x = torch.zeros((m, k), dtype=torch.bfloat16, device=dev)
    g = torch.Generator().manual_seed(6)
    tail = torch.randn((368, k), generator=g).to(torch.bfloat16)  # from row 544 x 128 on
    x[m - 368:].copy_(tail)
    for by in ("rows", "blocks"):
        f = (lambda n: n) if by == "rows" else ref.blocks
        q, s = torch.empty((m, k), dtype=torch.float8_e4m3fn, device=dev), torch.empty((f(m), ref.blocks(k)), device=dev)
        qt = torch.empty((k, m), dtype=torch.float8_e4m3fn, device=dev)
        st = torch.empty((f(k), ref.blocks(m)), device=dev)
        wq, ws = ref.quant(tail, "e4m3", by, False)
        wqt, wst = ref.quant(tail.t().contiguous(), "e4m3", by, False)
        for outs in ([q, s], [q, s, qt, st]):
            for o in outs:
                o.view(torch.uint8 if o.dtype.itemsize == 1 else o.dtype).fill_(1)
            C.op_call(C.OpKind.QuantFp8, [x], outs, QFP8, struct.pack("<i", 0))
            assert torch.equal(q[m - 368:].cpu().view(torch.uint8), wq.view(torch.uint8))
            assert torch.equal(s[-ws.shape[0]:].cpu(), ws)
        assert torch.equal(qt[:, m - 368:].cpu().view(torch.uint8), wqt.view(torch.uint8))
        assert torch.equal(st[:, -wst.shape[1]:].cpu(), wst)
        assert not q[:1000].view(torch.uint8).any() and not qt[:, :1000].contiguous().view(torch.uint8).any()


def test_classes_beyond_the_limits_are_refused():
    d = At()
    for v in ((1 << 28) + 1, (1 << 31) - 1, 1 << 31):
        refused(abi.load(), DISTILL, [d((2, v)), d((2, 4)), d((2, 4), I32)], [d((1,)), d((2, v)), d((2,))], DTOP,
                struct.pack("<ff", 1.0, 0.0))
