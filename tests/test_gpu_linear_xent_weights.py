"""linear_xent with row weights far apart in one call.  G of 16-bit operands has
one scale for all rows: in f16 its steps are 2^-37 of the largest weight at least,
which the bound allows, and no more."""
from __future__ import annotations

import pytest
import torch

import tail_ref as ref
from test_gpu_linear_xent import call, problem

pytestmark = pytest.mark.gpu


def kept(got, want, bound, dt):
    """Within the bound of the value rounded to dt.  What may lie behind dt's largest, want + b or want - b, may be
    infinite of that sign, and what surely does is not finite: a weight of 2^40 makes most of a gradient's elements
    such in f16, whose largest is 65504, and the bound of those next to zero is wide enough for either sign."""
    got, b, big = got.double(), ref.rounded(bound, want, dt), torch.finfo(dt).max
    inf = ((got == torch.inf) & (want + b >= big)) | ((got == -torch.inf) & (want - b <= -big))
    return (inf | ((got - want).abs() <= b)).all() and not (got.isfinite() & (want.abs() - b > big)).any()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("r,v,d,piece", [(40, 1003, 64, 0), (40, 1003, 64, 512), (150, 5001, 128, 0), (300, 2000, 72, 768)])
@pytest.mark.parametrize("least", [-12, -30])
def test_weights_far_apart(C, dev, least, r, v, d, piece, dtype):
    x, w, labels, g = problem(r, v, d, dtype, r + v)
    for top in (0, 40, -40):
        rw = torch.exp2(least * torch.rand(r, generator=g) + top) * torch.sign(torch.randn(r, generator=g))
        rw[0] = 2.0 ** top
        for outs in ("all", "dx"):
            got = call(C, dev, x, w, labels, rw, outs, piece)
            loss, dx, dw, rl, bt, bx, bw, bl = ref.linear_xent(x, w, labels, rw)
            assert ((got[3].double() - rl).abs() <= bl).all() and abs(float(got[0]) - float(loss)) <= bt
            assert kept(got[1], dx, bx, x.dtype)
            if outs == "all":
                assert kept(got[2], dw, bw, x.dtype)
