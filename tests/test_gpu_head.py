"""distill_topk and sample_row on the GPU against their definitions in 64 bits."""
from __future__ import annotations

import math
import struct

import pytest
import torch

import head_ref as ref

pytestmark = pytest.mark.gpu
DTOP = int.from_bytes(b"DTOP", "little")
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def rows_apart(t, dev, pad, off=0):
    """t on the device with rows pad elements apart, NaN between them."""
    r, c = t.shape
    buf = torch.full((r * (c + pad) + off,), math.nan if t.is_floating_point() else -7, dtype=t.dtype, device=dev)
    v = buf[off:].view(r, c + pad)[:, :c]
    v.copy_(t)
    return v


# ------------------------------------------------------------------ distill
def student(r, v, k, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn((r, v), generator=g) * 3
    ids = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(r)]).to(torch.int32)
    t = torch.randn((r, k), generator=g).sort(-1, descending=True).values * 2 + 5
    return z.to(DT[dtype]), t.to(DT[dtype]), ids, g


def distill(C, dev, z, t, ids, tau, alpha, labels=None, w=None, scratch=0, pad=0, in_place=False, loss_only=False,
            stream=0):
    zd, td, idd = rows_apart(z, dev, pad, pad), rows_apart(t, dev, pad), rows_apart(ids, dev, pad)
    r, v = z.shape
    dz = zd if in_place else rows_apart(torch.full_like(z, math.nan), dev, pad)
    loss, rl = torch.full((1,), math.nan, device=dev), torch.full((r,), math.nan, device=dev)
    ins = [zd, td, idd] + ([labels.to(dev)] if labels is not None else []) + ([w.to(dev)] if w is not None else [])
    outs = [loss] + ([] if loss_only else [dz]) + [rl]
    if scratch:
        outs.append(torch.full((r, scratch, 4), math.nan, device=dev))
    C.op_call(C.OpKind.DistillTopk, ins, outs, DTOP, struct.pack("<ff", tau, alpha), stream)
    return loss.cpu(), dz.cpu(), rl.cpu()


def check(got, z, t, ids, tau, alpha, labels=None, w=None, loss_only=False):
    tau, alpha = (struct.unpack("<f", struct.pack("<f", x))[0] for x in (tau, alpha))
    loss, dz, rl, bz, bl = ref.distill(z, t, ids, tau, alpha, labels, w)
    assert ((got[2].double() - rl).abs() <= bl).all(), ((got[2].double() - rl).abs() / bl).max()
    wr = w.double() if w is not None else torch.full_like(rl, 1.0 / len(rl))
    assert abs(float(got[0]) - loss) <= (wr.abs() * bl).sum() + 4 * ref.U * loss.abs()
    if not loss_only:
        far = (got[1].double() - dz).abs()
        assert (far <= bz).all(), (far / bz).max()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("r,v,k", [(1, 1, 1), (2, 5, 3), (3, 64, 64), (4, 1000, 20), (2, 8192, 64), (3, 8193, 7),
                                   (2, 20011, 256), (1, 70001, 1024)])
@pytest.mark.parametrize("tau,alpha", [(1.0, 0.0), (2.0, 0.25)])
def test_distill(C, dev, r, v, k, dtype, tau, alpha):
    z, t, ids, g = student(r, v, k, dtype, v + k)
    labels = torch.randint(0, v, (r,), generator=g, dtype=torch.int32) if alpha else None
    for scratch in (0, 64):
        got = distill(C, dev, z, t, ids, tau, alpha, labels, scratch=scratch, pad=v % 2)
        check(got, z, t, ids, tau, alpha, labels)


def test_distill_masks_and_repeats(C, dev):
    """Rows without a teacher, without a label, with neither; the same class
    twice, with a label among the teacher's; classes out of range; -inf
    logits; rows of weight 0, whose logits may be anything."""
    for v, dtype in ((300, "f32"), (9001, "bf16"), (50001, "bf16")):
        r, k = 8, 6
        z, t, ids, g = student(r, v, k, dtype, 11)
        labels = torch.tensor([0, 5, -1, v, v - 1, 3, 2, 1], dtype=torch.int32)
        ids[0] = -1
        ids[2, 1:] = v
        ids[3] = -1  # (its label is out of range too)
        ids[4] = 9
        ids[5, :3], ids[5, 3:] = 3, 7
        z[6, ids[6, 0] + 1 if ids[6, 0] + 1 < v and not (ids[6] == ids[6, 0] + 1).any() else v // 2] = -math.inf
        z[6, ids[6].long()] = 1.0
        t[1, 2] = -math.inf
        w = torch.tensor([0.5, 1.0, 0.25, 2.0, 1.0, 1.0, 1.0, 0.0])
        zz = z.clone()
        zz[7] = math.nan
        for tau, alpha in ((1.0, 0.0), (1.0, 0.5), (3.0, 0.5), (0.5, 1.0)):
            for scratch in (0, 16):
                got = distill(C, dev, zz, t, ids, tau, alpha, labels, w, scratch=scratch, pad=3)
                check(got, z, t, ids, tau, alpha, labels, w)
                assert (got[1][7] == 0).all() and got[2][7] == 0


def test_distill_row_of_nothing_is_nan(C, dev):
    for v in (500, 50000):
        z, t, ids, _ = student(3, v, 4, "f32", 2)
        z[1] = -math.inf
        for scratch in (0, 8):
            loss, dz, rl = distill(C, dev, z, t, ids, 1.0, 0.0, scratch=scratch)
            assert dz[1].isnan().all() and rl[1].isnan() and not dz[[0, 2]].isnan().any()


@pytest.mark.parametrize("v", [77, 4096, 12289, 50003])
def test_distill_in_place_loss_alone_and_repeated(C, dev, v):
    z, t, ids, g = student(5, v, 33, "bf16", v)
    labels = torch.randint(0, v, (5,), generator=g, dtype=torch.int32)
    for scratch in (0, 32):
        one = distill(C, dev, z, t, ids, 2.0, 0.3, labels, scratch=scratch)
        two = distill(C, dev, z, t, ids, 2.0, 0.3, labels, scratch=scratch, in_place=True)
        three = distill(C, dev, z, t, ids, 2.0, 0.3, labels, scratch=scratch, loss_only=True)
        for a, b in zip(one, two):
            assert torch.equal(a, b)
        assert torch.equal(one[0], three[0]) and torch.equal(one[2], three[2])
        check(one, z, t, ids, 2.0, 0.3, labels)


def test_distill_gradient_against_differences(C, dev):
    """dz against the loss itself, by central differences along random
    directions: the loss in f32 is off by at most bl a row, the third
    derivative's share by h^2 |d|^3 / 6 (softmax and its derivatives are at
    most 1 in the 1-norm, times tau^2 tau^-3 <= 1)."""
    z, t, ids, g = student(4, 600, 16, "f32", 9)
    labels = torch.randint(0, 600, (4,), generator=g, dtype=torch.int32)
    w = torch.tensor([1.0, 0.5, 0.25, 1.0])
    tau, alpha, h = 2.0, 0.25, 2.0 ** -5
    _, dz, _ = distill(C, dev, z, t, ids, tau, alpha, labels, w)
    _, _, _, bz, bl = ref.distill(z, t, ids, tau, alpha, labels, w)
    for _ in range(4):
        d = torch.sign(torch.randn((4, 600), generator=g))
        zp, zm = z + h * d, z - h * d
        up = distill(C, dev, zp, t, ids, tau, alpha, labels, w)[0]
        down = distill(C, dev, zm, t, ids, tau, alpha, labels, w)[0]
        slope = (float(up) - float(down)) / (2 * h)
        # zp and zm are rounded: 2^-24 |z| a coordinate; loss errors 2 sum(w bl) / (2 h)
        tol = (w * bl).sum() * 2 / h + 2 * h * h * w.sum() + (bz.sum()) + float((dz.abs() * z.abs()).sum()) * ref.U / h
        assert abs(slope - float((dz.double() * d).sum())) <= tol


def test_distill_captured(C, dev):
    v = 50009
    z, t, ids, g = student(6, v, 20, "f32", 4)
    zd, td, idd = z.to(dev), t.to(dev), ids.to(dev)
    loss, dz, rl, sc = (torch.empty(s, device=dev) for s in ((1,), (6, v), (6,), (6, 16, 4)))

    def call(stream=0):
        C.op_call(C.OpKind.DistillTopk, [zd, td, idd], [loss, dz, rl, sc], DTOP, struct.pack("<ff", 1.0, 0.0), stream)

    h = C.graph_create()
    call(C.graph_begin_h(h))
    C.graph_end_h(h)
    for i in range(4):
        zd.copy_(torch.randn((6, v), generator=g) * 2)
        C.graph_launch_h(h)
        got = [x.clone() for x in (loss, dz, rl)]
        torch.cuda.synchronize()
        for x in (loss, dz, rl):
            x.fill_(math.nan)
        call()
        assert all(torch.equal(a, b) for a, b in zip(got, (loss, dz, rl)))
    C.graph_destroy(h)


# ------------------------------------------------------------------- sample
def sample(C, dev, z, u, temp, k, p, m, scratch=False, pad=0, off=0):
    r = z.shape[0]
    f = lambda x, dt=torch.float32: torch.as_tensor(x, dtype=dt).expand(r).contiguous().to(dev)  # noqa: E731
    zd = rows_apart(z, dev, pad, off)
    tok, lp = torch.full((r,), -9, device=dev, dtype=torch.int32), torch.full((r,), math.nan, device=dev)
    outs = [tok, lp] + ([torch.full((r, 8192), -1, device=dev, dtype=torch.int32)] if scratch else [])
    C.op_call(C.OpKind.SampleRow, [zd, f(u), f(temp), f(k, torch.int32), f(p), f(m)], outs)
    return tok.cpu(), lp.cpu()


def check_sample(C, dev, z, u, temp, k, p, m, pad=0, off=0):
    r = z.shape[0]
    f = lambda x, dt=torch.float32: torch.as_tensor(x, dtype=dt).expand(r).contiguous()  # noqa: E731
    args = [f(u), f(temp), f(k, torch.int32), f(p), f(m)]
    for scratch in (False, True):
        tok, lp = sample(C, dev, z, *args, scratch=scratch, pad=pad, off=off)
        for i in range(r):
            wt, wl = ref.sample(z[i], *[x[i].item() for x in args])
            assert int(tok[i]) == wt, (i, int(tok[i]), wt, [x[i].item() for x in args], scratch)
            # a weight is off by 2^-38 of the largest or less, the logarithm is rounded once
            assert lp[i].item() == wl or abs(lp[i].item() - wl) <= 2 * ref.U * abs(wl) + 1e-7, (i, lp[i], wl)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 40, 0.8, 0.0), (1.0, 0, 1.0, 0.05),
            (0.9, 100, 0.95, 0.02), (0.0, 0, 1.0, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (5.0, 7, 0.5, 0.3)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("v", [1, 2, 7, 63, 1000, 2049, 8191, 8193, 33000, 66001, 140001])
def test_sample(C, dev, v, dtype):
    g = torch.Generator().manual_seed(v)
    r = len(SETTINGS) * (3 if v < 20000 else 1)
    z = (torch.randn((r, v), generator=g) * 3).to(DT[dtype])
    s = [SETTINGS[i % len(SETTINGS)] for i in range(r)]
    check_sample(C, dev, z, torch.rand(r, generator=g), [x[0] for x in s], [x[1] for x in s], [x[2] for x in s],
                 [x[3] for x in s], pad=v % 3, off=v % 2)


@pytest.mark.parametrize("v", [100, 5000, 20000, 70000])
def test_sample_ties_and_flat_rows(C, dev, v):
    """Rows of few different values, or of one: cuts inside a tie go by the
    class; cuts that leave thousands of classes."""
    g = torch.Generator().manual_seed(v)
    flat = torch.zeros(v)
    two = torch.randint(0, 2, (v,), generator=g).float()
    few = torch.randint(-3, 3, (v,), generator=g).float() * 0.5
    near = torch.randn(v, generator=g) * 1e-3
    zeros = torch.where(torch.rand(v, generator=g) < 0.5, -0.0, 0.0)
    z = torch.stack([flat, two, few, near, zeros])
    for temp, k, p, m in ((1.0, 0, 1.0, 0.0), (1.0, v // 3, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (2.0, v // 2, 0.7, 0.0),
                          (0.5, 3, 1.0, 0.0), (1.0, v - 1, 0.999, 0.4), (1.0, 0, 1e-6, 0.0), (100.0, 0, 0.9, 0.5)):
        check_sample(C, dev, z, torch.rand(5, generator=g), temp, k, p, m)


def test_sample_not_finite_and_edges(C, dev):
    inf, nan = math.inf, math.nan
    for v in (6, 10007, 40009):
        base = torch.full((9, v), -inf)
        base[1, 3] = -50.0
        base[2, :] = nan
        base[3, 2], base[3, 4] = inf, inf
        base[3, 5] = 3.0
        base[4, :6] = torch.tensor([1.0, nan, 1.0, -inf, nan, 0.5])
        base[5, v - 1] = 2.0
        base[5, 0] = 2.0
        base[6, :] = 1.0
        base[7, :6] = torch.tensor([3e38, -3e38, 3e38, 0.0, 1.0, -3e38])
        base[8, :6] = torch.tensor([-0.0, 0.0, -0.0, 0.0, -1e-45, 1e-45])
        for u in (0.0, 1.0 - 2.0 ** -24, 0.5, 1.5, -1.0, nan):
            for temp, k, p, m in ((1.0, 0, 1.0, 0.0), (1.0, 2, 1.0, 0.0), (1.0, 0, 0.6, 0.0), (inf, 0, 1.0, 0.0),
                                  (1e-3, 0, 0.99, 0.0), (nan, 0, 1.0, 0.0), (-1.0, 0, 1.0, 0.0), (1.0, -5, nan, nan),
                                  (1.0, 2 ** 31 - 1, 2.0, 7.0), (1e-38, 3, 0.9, 0.1)):
                check_sample(C, dev, base, u, temp, k, p, m)


def test_sample_draws_every_class_at_its_share(C, dev):
    """u on a grid of n: each class is drawn as often as its share of n, +- 1."""
    n, v = 4096, 37
    z = torch.randn((1, v), generator=torch.Generator().manual_seed(1)).expand(n, v).contiguous()
    u = (torch.arange(n) + 0.5) / n
    tok, _ = sample(C, dev, z, u, 1.0, 0, 1.0, 0.0)
    share = torch.softmax(z[0].double(), 0) * n
    assert ((torch.bincount(tok, minlength=v) - share).abs() <= 1).all()
    assert (tok.diff() >= 0).all()


def test_sample_captured_and_without_log_probability(C, dev):
    g = torch.Generator().manual_seed(6)
    r, v = 4, 34000
    z = torch.empty((r, v), device=dev)
    u, temp, p, m = (torch.empty(r, device=dev) for _ in range(4))
    k = torch.full((r,), 20, device=dev, dtype=torch.int32)
    for x, y in ((temp, 1.0), (p, 0.9), (m, 0.0)):
        x.fill_(y)
    tok, lp = torch.empty(r, device=dev, dtype=torch.int32), torch.empty(r, device=dev)
    sc = torch.empty((r, 8192), device=dev, dtype=torch.int32)
    for outs in ([tok], [tok, lp], [tok, lp, sc]):
        h = C.graph_create()
        C.op_call(C.OpKind.SampleRow, [z, u, temp, k, p, m], outs, stream=C.graph_begin_h(h))
        C.graph_end_h(h)
        for i in range(4):
            z.copy_(torch.randn((r, v), generator=g) * 2)
            u.copy_(torch.rand(r, generator=g))
            tok.fill_(-9)
            C.graph_launch_h(h)
            got = tok.cpu()
            want = [ref.sample(z[j].cpu(), u[j].item(), 1.0, 20, p[j].item(), 0.0)[0] for j in range(r)]
            assert got.tolist() == want
        C.graph_destroy(h)


def test_on_policy_distillation_step(C, dev):
    """The ops as they are used together: hidden rows and head weights in 8
    bits, logits, a token drawn a row, the teacher's top logits there, loss
    and gradient, and the gradient's products in 8 bits."""
    from test_gpu_fp8 import QFP8, strided

    g = torch.Generator(device=dev).manual_seed(8)
    R, H, V, K = 48, 256, 1000, 16
    rnd = lambda *s: torch.randn(s, device=dev, generator=g)  # noqa: E731
    h, w = rnd(R, H).to(torch.bfloat16), (rnd(V, H) / 4).to(torch.bfloat16)

    def both(x, by, fp8=torch.float8_e4m3fn):
        r, c = x.shape
        f = lambda n: n if by == "rows" else ref.blocks(n)  # noqa: E731
        outs = [strided(r, c, fp8, dev, -c % 16)[0], torch.empty((f(r), ref.blocks(c)), device=dev),
                strided(c, r, fp8, dev, -r % 16)[0], torch.empty((f(c), ref.blocks(r)), device=dev)]
        C.op_call(C.OpKind.QuantFp8, [x], outs, QFP8, struct.pack("<i", 1))
        return outs

    hq, hs, hqt, hst = both(h, "rows")
    wq, ws, wqt, wst = both(w, "blocks")
    z = torch.empty((R, V), device=dev, dtype=torch.bfloat16)
    C.op_call(C.OpKind.GemmFp8, [hq, hs, wq, ws], [z])
    full = lambda x, dt=torch.float32: torch.full((R,), x, device=dev, dtype=dt)  # noqa: E731
    tok, lp = full(0, torch.int32), full(0.0)
    u = torch.rand(R, device=dev, generator=g)
    C.op_call(C.OpKind.SampleRow, [z, u, full(0.8), full(20, torch.int32), full(0.9), full(0.0)], [tok, lp])
    assert tok.tolist() == [ref.sample(z[i].cpu(), u[i].item(), full(0.8)[0].item(), 20, full(0.9)[0].item(), 0.0)[0]
                            for i in range(R)]
    t, ids = (z.float() + rnd(R, V)).topk(K, -1)
    ids = ids.to(torch.int32)
    loss, rl, dz = torch.empty(1, device=dev), full(0.0), torch.empty_like(z)
    C.op_call(C.OpKind.DistillTopk, [z, t, ids, tok], [loss, dz, rl], DTOP, struct.pack("<ff", 1.0, 0.5))
    want = ref.distill(z.cpu(), t.cpu(), ids.cpu(), 1.0, 0.5, tok.cpu())
    assert ((dz.cpu().double() - want[1]).abs() <= want[3]).all()
    dq, ds, dqt, dst = both(dz, "rows", torch.float8_e5m2)
    dh, dw = torch.empty((R, H), device=dev), torch.empty((V, H), device=dev)
    C.op_call(C.OpKind.GemmFp8, [dq, ds, wqt, wst], [dh])
    C.op_call(C.OpKind.GemmFp8, [dqt, dst, hqt, hst], [dw])
    # e5m2 codes of dz (half a step 2^-3) times e4m3 codes (2^-4), errors of either sign
    for got, exact in ((dh, want[1] @ w.cpu().double()), (dw, want[1].t() @ h.cpu().double())):
        assert (got.cpu().double() - exact).norm() <= (2.0 ** -3 + 2.0 ** -4) * exact.norm()
