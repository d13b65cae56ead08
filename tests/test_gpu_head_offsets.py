"""distill_topk on logits far from zero, by the workgroup a row and by rows that
workgroups share, against the definition in 64 bits: a softmax does not change
when all its logits move together, so neither does the bound."""
from __future__ import annotations

import math

import pytest
import torch

import head_ref as ref
from test_gpu_head import DT, check, distill, student

pytestmark = pytest.mark.gpu
# the temperature at which exp(z / tau) is 2^z: no reference point is rounded
LOG2E = 1.4426950408889634


@pytest.fixture
def below_normal(monkeypatch):
    """Small temperatures bring exponentials below the smallest normal f32,
    2^-126; the exponential instruction gives 0 there.  An element of the gradient
    is then off by at most 2^-126 w ((1 - a) tau / S + a / S1) <= 2^-126: w <= 1/2, tau <= 2, and the sums S
    and S1 are 1 or more."""
    for t in ref.TINY:
        monkeypatch.setitem(ref.TINY, t, ref.TINY[t] + 2.0 ** -126)


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


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shift,tau,alpha", [(-1000.0, 1.0, 0.0), (1000.0, 1.0, 0.5), (-1e4, 2.0, 0.5),
                                             (-20.0, 0.05, 0.0), (-20.0, 0.05, 0.5), (3e4, 0.7, 0.25)])
def test_moved_together(C, dev, below_normal, shift, tau, alpha, dtype):
    """The bounds of logits around zero, whatever was added to all of them."""
    for r, p, v in ((3, 64, 700), (2, 8, 50021), (2, 64, 131072)):
        z, t, ids, labels = moved(r, v, 6, dtype, shift, v)
        lab = labels if alpha else None
        for scratch in (0, p):
            check(distill(C, dev, z, t, ids, tau, alpha, lab, scratch=scratch), z, t, ids, tau, alpha, lab)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("v", [500, 9001, 50021, 140001])
def test_masks_of_the_lowest_value(C, dev, v, dtype):
    """Rows masked with the type's lowest finite value: whole (all classes are
    then equally likely), but for a few classes, but for one part; a row of the highest."""
    z, t, ids, labels = moved(4, v, 5, dtype, 0.0, v)
    low = torch.finfo(z.dtype).min
    few = z[1, ids[1].long()].clone()
    z[0], z[1], z[3] = low, low, -low
    z[1, ids[1].long()] = few
    z[2, 300:] = low
    ids[2] = torch.arange(5) * 50
    labels[1], labels[2] = ids[1, 0], 7
    for tau, alpha in ((1.0, 0.0), (0.5, 0.0), (2.0, 0.5)):
        lab = labels if alpha else None
        for scratch in (0, 8):
            check(distill(C, dev, z, t, ids, tau, alpha, lab, scratch=scratch), z, t, ids, tau, alpha, lab)


@pytest.mark.parametrize("v", [500, 50021])
def test_teachers_far_from_zero(C, dev, below_normal, v):
    """The teacher's logits moved together, alike, or masked with the lowest value."""
    z, t, ids, _ = moved(5, v, 6, "f32", 0.0, v)
    t[0] += 1000.0
    t[1] -= 1e4
    t[2] = -3.0e38
    t[3, 2:] = torch.finfo(torch.float32).min
    t[4] = 3.0e38
    for tau in (1.0, 0.3, 2.0):
        for scratch in (0, 8):
            check(distill(C, dev, z, t, ids, tau, 0.0, scratch=scratch), z, t, ids, tau, 0.0)


@pytest.mark.parametrize("v", [300, 9001, 50021])
def test_a_term_of_weight_0_is_left_out(C, dev, v):
    """The labels' loss alone where the teacher's term is infinite or no number,
    and the teacher's alone where the label's is."""
    z, t, ids, labels = moved(4, v, 6, "f32", 0.0, v)
    z[0, ids[0, 1].long()] = -math.inf
    labels[0] = ids[0, 0]
    zl, labels[1:] = z.clone(), ids[1:, 5] + 1
    labels[labels == v] = 0
    tn = t.clone()
    tn[1, 2], tn[2] = math.nan, math.inf
    zl[3, labels[3].long()] = -math.inf
    ids[3, 5] = -1
    ids[3][ids[3] == labels[3]] = -1
    none = torch.full_like(ids, -1)  # (the definition without the teacher's term)
    for scratch in (0, 8):
        for tau in (1.0, 2.0):
            check(distill(C, dev, z, tn, ids, tau, 1.0, labels, scratch=scratch), z, t, none, tau, 1.0, labels)
            rest = slice(1, 4)
            check(distill(C, dev, zl[rest], t[rest], ids[rest], tau, 0.0, labels[rest], scratch=scratch), zl[rest],
                  t[rest], ids[rest], tau, 0.0)


@pytest.mark.parametrize("tau", [2.0 ** -60, 2.0 ** -30, 2.0 ** 30, 2.0 ** 60])
def test_temperatures_of_the_whole_range(C, dev, below_normal, tau):
    """(the smallest ones: exponentials below 2^-126 again, times tau < 1; the largest ones have none)"""
    for v in (500, 50021):
        z, t, ids, labels = moved(2, v, 6, "f32", 0.0, v)
        for scratch in (0, 8):
            check(distill(C, dev, z, t, ids, tau, 0.5, labels, scratch=scratch), z, t, ids, tau, 0.5, labels)
