"""linear_xent's products at many classes and rows, block by block: W's rows of 32
neighbouring classes have one element other than zero, all in the same column, and
so have X's rows of 32 neighbouring rows.  An element of dX is then a sum over the
classes of a few such blocks alone, one of dW over the rows of a few, and a block
that is left out of a product or counted twice shows in its size, where it is lost
in the bound of a sum over all classes.  (Zeros add nothing and cost no rounding.)"""
from __future__ import annotations

import random

import pytest
import torch

from head_ref import HALF_STEP, TINY, U
from test_gpu_linear_xent import DT, call

BLOCK = 32
CASES = [(600, 25000, 200, 0), (600, 25000, 200, 12544), (1025, 13001, 264, 6656), (4096, 4096, 136, 0),
         (4096, 4096, 136, 1024), (129, 70000, 280, 0), (129, 70000, 280, 35072), (2500, 3001, 512, 1536),
         (64, 28436, 128, 28416), (128, 5889, 512, 5376), (40, 50257, 256, 4864), (1, 10270, 512, 5376),
         (300, 9001, 72, 2304)]


def columns(n, d):
    return torch.arange(n) // BLOCK % d


def problem(r, v, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x, w = torch.zeros(r, d), torch.zeros(v, d)
    x[torch.arange(r), columns(r, d)] = 0.5 + 0.5 * torch.rand(r, generator=g)
    w[torch.arange(v), columns(v, d)] = 0.5 + 0.5 * torch.rand(v, generator=g)
    labels = torch.randint(0, v, (r,), generator=g, dtype=torch.int32)
    labels[3::7] = -1
    return x.to(DT[dtype]), w.to(DT[dtype]), labels, 0.5 + torch.rand(r, generator=g)


def wanted(x, w, labels, rw):
    """(dX, its bound), (dW, its bound) before the rounding to their type, and G."""
    h, (r, d), v = HALF_STEP[x.dtype], x.shape, w.shape[0]
    dev, f16 = x.device, x.dtype == torch.float16
    x, w = x.double(), w.double()
    wr = torch.where(labels >= 0, rw.double(), 0.0)[:, None]
    z = x @ w.t().contiguous()
    p = torch.softmax(z, 1)
    g = p.clone()
    at = torch.arange(r, device=dev)
    g[at, labels.long().clamp(min=0)] -= 1.0
    g = g * wr
    # A logit is one product of at most 1 (or zero), off by a rounding; a probability by those of its logit and of the
    # sum's, by the additions of the sum (256 classes a tile, lanes and waves, the tiles), the exponents' arguments
    # (at most 1) and two exponentials.
    rel = 4 * U + (256 + v / 128 + 32) * 2 * U + 24 * U
    # The numerator is rounded, then G (to the operands' type); an f16 below the normal numbers by 2^-25 of 2^14 or 2^13.
    ge = wr * p * rel + h * wr * p * (1 + rel) + h * (g.abs() + wr * p * rel) + 4 * U * wr * (p + 1)
    if f16:
        ge = ge + 2.0 ** -36 * wr.max()
    if h != HALF_STEP[torch.float32]:
        ge = ge + 2.0 ** -39 * wr
    # additions that are not of zeros: the classes (rows) of a column's blocks, and at most 64 shares and 256 parts
    nx, nw = ((-(-n // (BLOCK * d)) * BLOCK + 320) * 2 * U for n in (v, r))
    ga = g.abs() + ge
    gt, gat = ge.t().contiguous(), ga.t().contiguous()
    return (g @ w, ge @ w + nx * (ga @ w)), (g.t().contiguous() @ x, gt @ x + nw * (gat @ x)), g


def kept(got, want, bound, dt):
    return (got.double() - want).abs() <= bound + HALF_STEP[dt] * (want.abs() + bound) + TINY[dt]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("r,v,d,piece", CASES)
def test_blocks(C, dev, r, v, d, piece, dtype):
    x, w, labels, rw = problem(r, v, d, dtype, r + v + piece)
    (dx, bx), (dw, bw), _ = wanted(*(t.to(dev) for t in (x, w, labels, rw)))
    for outs in ("all", "dx"):
        got = call(C, dev, x, w, labels, rw, outs, piece)
        assert kept(got[1], dx.cpu(), bx.cpu(), x.dtype).all()
        if outs == "all":
            assert kept(got[2], dw.cpu(), bw.cpu(), x.dtype).all()
    if dtype != "f32":
        got = call(C, dev, x, w, labels, rw, "all", piece, dw_type=torch.float32)
        assert kept(got[2], dw.cpu(), bw.cpu(), torch.float32).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("r,v,d", [(129, 70000, 280), (600, 25000, 200), (64, 28436, 128), (40, 50257, 256),
                                   (300, 9001, 72), (2500, 3001, 512)])
def test_the_bound_shows_a_block(r, v, d, dtype):
    """The definition itself keeps the bound; with 32 classes (64 in 16 bits: a K-step) left out of dX or counted
    twice, or 32 rows out of dW, it does not."""
    x, w, labels, rw = problem(r, v, d, dtype, r)
    (dx, bx), (dw, bw), g = wanted(x, w, labels, rw)
    assert kept(dx.to(x.dtype), dx, bx, x.dtype).all() and kept(dw.to(x.dtype), dw, bw, x.dtype).all()
    rng = random.Random(r)
    step = BLOCK if dtype == "f32" else 2 * BLOCK
    for k in {0, (v - 1) // step, *(rng.randrange((v - 1) // step) for _ in range(4))}:
        part = slice(k * step, (k + 1) * step)
        off = g[:, part] @ w.double()[part]
        for sign in (-1, 1):
            assert not kept((dx + sign * off).to(x.dtype), dx, bx, x.dtype).all(), (k, sign)
    if r > step:
        for k in {0, *(rng.randrange(r // step) for _ in range(4))}:
            part = slice(k * step, (k + 1) * step)
            off = g[part].t().contiguous() @ x.double()[part]
            for sign in (-1, 1):
                assert not kept((dw + sign * off).to(x.dtype), dw, bw, x.dtype).all(), (k, sign)
