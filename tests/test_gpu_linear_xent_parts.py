"""linear_xent with scratch for a part of the classes, at sizes where the part
that scratch holds has fewer classes than its room and every other part has fewer
still: dX joins the sums of the shares that some part wrote, and no others."""
from __future__ import annotations

import pytest
import torch

import tail_ref as ref
from test_gpu_linear_xent import call, problem

pytestmark = pytest.mark.gpu


def compare(C, dev, x, w, labels, rw, outs, piece):
    """Scratch is filled with NaN: a sum that nothing wrote shows."""
    want = [t.cpu() if isinstance(t, torch.Tensor) else t
            for t in ref.linear_xent(x.to(dev), w.to(dev), labels.to(dev), None if rw is None else rw.to(dev))]
    loss, dx, dw, rl, bt, bx, bw, bl = want
    got = call(C, dev, x, w, labels, rw, outs, piece)
    assert ((got[3].double() - rl).abs() <= bl).all() and abs(float(got[0]) - float(loss)) <= bt
    assert ((got[1].double() - dx).abs() <= ref.rounded(bx, dx, x.dtype)).all()
    if outs == "all":
        assert ((got[2].double() - dw).abs() <= ref.rounded(bw, dw, x.dtype)).all()


@pytest.mark.parametrize("outs", ["dx", "all"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("r,v,d,piece", [(128, 5889, 512, 5376), (16, 12344, 128, 6400), (1, 10270, 512, 5376),
                                         (64, 28436, 128, 28416), (40, 5121, 72, 5120)])
def test_parts_shorter_than_a_piece(C, dev, r, v, d, piece, dtype, outs):
    x, w, labels, g = problem(r, v, d, dtype, r + piece)
    rw = torch.rand(r, generator=g) + 0.1
    labels[0] = v - 1
    compare(C, dev, x, w, labels, rw, outs, piece)


@pytest.mark.parametrize("outs", ["dx", "all"])
@pytest.mark.parametrize("labelled", [64, 128, 129, 512])
def test_shares_by_the_rows_that_count(C, dev, labelled, outs):
    """The device chooses dX's shares by how many rows have a label."""
    r, v, d, piece = 512, 50257, 768, 49408
    x, w, labels, _ = problem(r, v, d, "bf16", labelled)
    labels[torch.arange(r) * labelled // r == torch.arange(-1, r - 1) * labelled // r] = -1
    assert int((labels >= 0).sum()) == labelled
    compare(C, dev, x, w, labels, None, outs, piece)
