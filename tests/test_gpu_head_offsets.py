"""distill_topk on logits far from zero, by the workgroup a row and by rows that
workgroups share, against the definition in 64 bits: a softmax does not change
when all its logits move together, so neither does the bound."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_head import DT, check, distill, student

pytestmark = pytest.mark.gpu
# the temperature at which exp(z / tau) is 2^z: no reference point is rounded
LOG2E = 1.4426950408889634


def moved(r, v, k, dtype, shift, seed):
    """Logits whose largest lie near shift, and labels."""
    z, t, ids, g = student(r, v, k, "f32", seed)
    labels = torch.randint(0, v, (r,), generator=g, dtype=torch.int32)
    return (z + shift).to(DT[dtype]), t, ids, labels


@pytest.mark.parametrize("r,p,v", [(1, 64, 131072), (2, 8, 50021), (9, 64, 131072)])
@pytest.mark.parametrize("shift", [-140.0, -1000.0, -1e4])
def test_far_below_zero(C, dev, r, p, v, shift):
    """Fewer parts than a wave has lanes, and as many."""
    z, t, ids, labels = moved(r, v, 5, "f32", shift, v + r)
    for alpha in (0.0, 0.5) if shift == -140.0 else (0.0,):
        lab = labels if alpha else None
        for scratch in (0, p):
            check(distill(C, dev, z, t, ids, LOG2E, alpha, lab, scratch=scratch), z, t, ids, LOG2E, alpha, lab)


@pytest.mark.parametrize("v", [131072, 50021])
def test_parts_without_a_class(C, dev, v):
    """All classes but a few, or but one part's, are masked; the rest lie far below zero."""
    z, t, ids, _ = moved(3, v, 4, "f32", -150.0, v)
    few = z[0, [5, v - 1]].clone()
    z[0] = -math.inf
    z[0, [5, v - 1]] = few
    ids[0] = torch.tensor([5, v - 1, -1, v])
    z[1, 2048:] = -math.inf
    ids[1] = torch.tensor([0, 2047, 7, 100])
    for scratch in (0, 64):
        check(distill(C, dev, z, t, ids, LOG2E, 0.0, scratch=scratch), z, t, ids, LOG2E, 0.0)
