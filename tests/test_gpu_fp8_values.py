"""gemm_fp8 on the values that normally distributed codes do not have: outlier
channels, heavy tails, products that cancel, scales far from 1; and rows that
do not depend on one another."""
from __future__ import annotations

import math
import struct

import pytest
import torch

import head_ref as ref
from test_gpu_fp8 import DT, QFP8, codes, strided

pytestmark = pytest.mark.gpu


def quantised(C, x, by, fp8, dev, pad):
    """The op's codes and scales of x, rows on 16-byte steps and pad more bytes."""
    r, c = x.shape
    q, _ = strided(r, c, ref.FP8[fp8], dev, -c % 16 + pad)
    s = torch.empty((r if by == "rows" else ref.blocks(r), ref.blocks(c)), device=dev)
    C.op_call(C.OpKind.QuantFp8, [x.to(dev)], [q, s], QFP8, struct.pack("<i", 0))
    return q, s


@pytest.mark.parametrize("a8", ["e4m3", "e5m2"])
@pytest.mark.parametrize("kind", ["channels x 30", "channels x 1000", "lognormal", "positive", "cancelling"])
@pytest.mark.parametrize("m,n,k", [(20, 90, 512), (150, 130, 784)])
def test_outliers_and_cancelling_products(C, dev, m, n, k, kind, a8):
    """Every output within the bound of what its type's products keep: f32 sums, or 13 bits below each group's
    largest product (f32 sums for few rows); straight into LDS and from any alignment."""
    g = torch.Generator().manual_seed(m + len(kind))
    x, w = torch.randn((m, k), generator=g), torch.randn((n, k), generator=g)
    if kind.startswith("channels"):
        x *= torch.where(torch.rand((1, k), generator=g) < 0.02, float(kind.split()[-1]), 1.0)
    elif kind == "lognormal":
        x *= torch.exp(2 * torch.randn((m, k), generator=g))
    elif kind == "positive":
        x = x.abs()
    else:
        x[:, 1::2] = -x[:, ::2]
        w[:, 1::2] = w[:, ::2] * (1 + torch.randn((n, k // 2), generator=g) / 16)
    for pad in (0, 1):
        (a, sa), (b, sb) = quantised(C, x, "rows", a8, dev, pad), quantised(C, w, "blocks", "e4m3", dev, pad)
        ah, sah, bh, sbh = (t.cpu() for t in (a, sa, b, sb))
        want, mag = ref.gemm(ah, sah, bh, sbh)
        groups = ref.group_max(ah, sah, bh, sbh)
        for out in ("f32", "bf16", "f16"):
            if out == "f16":  # within f16's range
                shrink = 2.0 ** -max(0, math.frexp(float(want.abs().max()))[1] - 14)
            else:
                shrink = 1.0
            c = torch.empty((m, n), dtype=DT[out], device=dev)
            C.op_call(C.OpKind.GemmFp8, [a, sa * shrink, b, sb], [c])
            bound = ref.gemm_bound(want * shrink, mag * shrink, k, DT[out], None if out == "f32" else groups * shrink)
            far = (c.cpu().double() - want * shrink).abs()
            assert (far <= bound).all(), (out, pad, (far / bound).max())


@pytest.mark.parametrize("ea,eb", [(100, -100), (-70, -50), (60, 40), (-126, 20)])
def test_scales_far_from_one(C, dev, ea, eb):
    """Each pair's product is a normal f32."""
    g = torch.Generator().manual_seed(3)
    for m, n, k in ((4, 40, 300), (70, 60, 300), (70, 60, 512)):
        a, sa, ad, _ = codes(m, k, "e4m3", "rows", g, dev, -k % 16)
        b, sb, bd, _ = codes(n, k, "e4m3", "rows", g, dev, -k % 16)
        sa, sb = (1 + sa / 2) * 2.0 ** ea, (1 + sb / 2) * 2.0 ** eb
        want, mag = ref.gemm(a, sa, b, sb)
        for out in ("f32", "bf16"):
            c = torch.empty((m, n), dtype=DT[out], device=dev)
            C.op_call(C.OpKind.GemmFp8, [ad, sa.to(dev), bd, sb.to(dev)], [c])
            bound = ref.gemm_bound(want, mag, k, DT[out], None if out == "f32" else ref.group_max(a, sa, b, sb))
            assert ((c.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k,pad", [(20, 64, 300, 0), (20, 9001, 256, 0), (200, 300, 513, 0), (200, 300, 512, 0),
                                       (300, 4100, 272, 0), (600, 700, 400, 1)])
def test_a_row_does_not_depend_on_the_others(C, dev, m, n, k, pad, out):
    """The same bits of some rows beside other rows, NaN and the largest codes among them; likewise of columns."""
    g = torch.Generator().manual_seed(m + n)
    _, _, a, sa = codes(m, k, "e4m3", "rows", g, dev, -k % 16 + pad)
    _, _, b, sb = codes(n, k, "e4m3", "rows", g, dev, -k % 16 + pad)
    one = torch.empty((m, n), dtype=DT[out], device=dev)
    two = torch.empty_like(one)
    C.op_call(C.OpKind.GemmFp8, [a, sa, b, sb], [one])
    keep_m, keep_n = torch.tensor([0, m // 2, m - 1], device=dev), torch.tensor([1, n // 3, n - 1], device=dev)
    for x, s, keep in ((a, sa, keep_m), (b, sb, keep_n)):
        rest = torch.ones(x.shape[0], dtype=torch.bool, device=dev)
        rest[keep] = False
        raw = x.view(torch.uint8)
        raw[rest] = torch.randint(0, 256, (int(rest.sum()), k), device=dev, dtype=torch.uint8)
        s[rest] = 1e3
    C.op_call(C.OpKind.GemmFp8, [a, sa, b, sb], [two])
    pick = lambda c: c[keep_m][:, keep_n]  # noqa: E731
    assert torch.equal(pick(one), pick(two)) and not pick(one).isnan().any()
    assert two.isnan().any()
