"""grad_norm and AdamW with the clip factor on the GPU against their definitions
in 64 bits."""
from __future__ import annotations

import math
import struct

import pytest
import torch

import tail_ref as ref
from head_ref import HALF_STEP, TINY

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GNRM, ADAM = (int.from_bytes(t, "little") for t in (b"GNRM", b"ADAM"))


def norm_of(C, dev, gs, max_norm, outs=(), stream=0, scratch=None):
    norm = torch.full((2,), math.nan, device=dev)
    if scratch is None:
        scratch = torch.full((2048 * -(-len(gs) // 96),), math.nan, device=dev)
    C.op_call(C.OpKind.GradNorm, list(gs), [norm, scratch] + list(outs), GNRM, struct.pack("<f", max_norm), stream)
    return norm


def check_norm(norm, gs, max_norm):
    max_norm = struct.unpack("<f", struct.pack("<f", max_norm))[0]
    want = ref.grad_norm([g.cpu() for g in gs], max_norm)
    # squares and sums in f64 (2^-53 each of up to 2^27 additions), one rounding to f32
    for got, w in zip(norm.tolist(), want):
        if w > torch.finfo(torch.float32).max * (1 + 2.0 ** -24):  # no f32 holds it: rounded to nearest it is infinite
            assert got == math.inf
            continue
        assert abs(got - w) <= w * (2.0 ** -24 + 2.0 ** -26) + 2.0 ** -149, (norm, want)


def tensors(dev, shapes, types, seed, scale=1e-2):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale).to(DT[t]).to(dev) for s, t in zip(shapes, types)]


SETS = [([(1,)], ["f32"]), ([(7,), (3, 5)], ["bf16", "f32"]), ([(4096,), (4097,), (4095,), (8192,)], ["f16"] * 4),
        ([(1000, 1111), (13,), (), (2, 3, 4, 5)], ["bf16", "f32", "f16", "f32"]), ([(0,), (5,), (3, 0)], ["f32"] * 3),
        ([(0,)], ["bf16"]), ([(17 + i,) for i in range(300)], (["f32", "bf16", "f16"] * 100)),
        ([(1 << 23,), (12345,)], ["f32", "bf16"])]


@pytest.mark.parametrize("k", range(len(SETS)))
def test_norm_and_clip(C, dev, k):
    shapes, types = SETS[k]
    gs = tensors(dev, shapes, types, k)
    total = ref.grad_norm([g.cpu() for g in gs], 1.0)[0]
    for share in (0.25, 4.0):
        max_norm = max(total * share, 1e-6)
        norm = norm_of(C, dev, gs, max_norm)
        check_norm(norm, gs, max_norm)
        outs = [torch.full_like(g, math.nan) for g in gs]
        again = norm_of(C, dev, gs, max_norm, outs)
        assert torch.equal(norm, again)
        f = norm[1].item()
        for g, o in zip(gs, outs):  # one rounding of the product of two f32
            want = g.double() * f
            assert ((o.double() - want).abs() <= HALF_STEP[g.dtype] * want.abs() * (1 + 2.0 ** -20)
                    + (2.0 ** -24 * want.abs() if g.dtype != torch.float32 else 0) + TINY[g.dtype]).all()
        mine = [g.clone() for g in gs]
        norm_of(C, dev, mine, max_norm, mine)  # in place
        for a, b in zip(mine, outs):
            assert torch.equal(a, b)
        if share > 1:
            assert f == 1.0 and all(torch.equal(a, b) for a, b in zip(outs, gs))


def test_views_at_any_element(C, dev):
    """Tensors at odd elements of one buffer; what lies between them stays."""
    for t in ("f32", "bf16", "f16"):
        base = torch.randn(50000, generator=torch.Generator().manual_seed(3)).to(DT[t]).to(dev)
        sizes, at, gs, rest = [1, 777, 4099, 8200, 3, 16384 + 5], 1, [], torch.ones(50000, dtype=torch.bool)
        for n in sizes:
            gs.append(base[at:at + n])
            rest[at:at + n] = False
            at += n + 1
        before = base.clone()
        check_norm(norm_of(C, dev, gs, 1.0), gs, 1.0)
        norm = norm_of(C, dev, gs, 1.0, gs)
        assert torch.equal(base[rest.to(dev)], before[rest.to(dev)])
        moved = ~rest.to(dev)
        want = (before.double() * norm[1].double())[moved]
        assert ((base.double()[moved] - want).abs() <= 2 * HALF_STEP[DT[t]] * want.abs() + TINY[DT[t]]).all()


def test_scales_and_values_that_are_not_finite(C, dev):
    """Squares beyond f32's range; infinities and NaN."""
    for scale in (1e-30, 1e25, 1e37):
        gs = tensors(dev, [(3000,), (70, 90)], ["f32", "bf16"], 1, scale)
        check_norm(norm_of(C, dev, gs, 1.0), gs, 1.0)
    gs = tensors(dev, [(300,), (500,)], ["f32", "f32"], 2)
    gs[0][7] = math.inf
    norm = norm_of(C, dev, gs, 1.0, gs)
    assert norm.tolist() == [math.inf, 0.0] and gs[0][7].isnan() and (gs[1] == 0).all() and (gs[0][:7] == 0).all()
    gs = tensors(dev, [(300,), (500,)], ["f32", "bf16"], 2)
    gs[1][499] = math.nan
    norm = norm_of(C, dev, gs, 1.0, gs)
    assert norm.isnan().all() and all(g.isnan().all() for g in gs)
    gs = tensors(dev, [(300,)], ["f32"], 2)
    check_norm(norm_of(C, dev, gs, math.inf), gs, math.inf)
    assert norm_of(C, dev, gs, 0.0, gs)[1] == 0 and (gs[0] == 0).all()
    gs = [torch.zeros(100, device=dev)]
    assert norm_of(C, dev, gs, 1.0, gs).tolist() == [0.0, 1.0]


def test_captured_and_on_another_stream(C, dev):
    gs = tensors(dev, [(300, 700), (999,), (4096, 33)], ["f32", "bf16", "f16"], 5)
    norm, sc = torch.empty(2, device=dev), torch.empty(2048, device=dev)
    h = C.graph_create()
    C.op_call(C.OpKind.GradNorm, gs, [norm, sc] + gs, GNRM, struct.pack("<f", 0.5), C.graph_begin_h(h))
    C.graph_end_h(h)
    for i in range(4):
        new = tensors(dev, [(300, 700), (999,), (4096, 33)], ["f32", "bf16", "f16"], 10 + i, 10.0 ** -i)
        for a, b in zip(gs, new):
            a.copy_(b)
        sc.fill_(math.nan)
        C.graph_launch_h(h)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            want = norm_of(C, dev, new, 0.5, new)
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(gs, new))
    C.graph_destroy(h)


# ------------------------------------------------------------------ AdamW
def adamw(C, dev, p, g, m, v, step, norm, outs, hp):
    ins = [p, g, m, v, torch.tensor(step, dtype=torch.int32, device=dev)] + ([norm] if norm is not None else [])
    C.op_call(C.OpKind.AdamStep, ins, outs, ADAM, struct.pack("<fffff", *hp))
    return outs


@pytest.mark.parametrize("gt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,off", [(1, 0), (3, 0), (1023, 0), (4096, 0), (70001, 0), (5000, 1), (8, 3)])
def test_adamw_with_the_factor(C, dev, n, off, gt):
    """The bits of clipping the gradient first (in f32), then AdamW; with and
    without a bf16 copy, in place and apart, at any element."""
    gen = torch.Generator().manual_seed(n)
    new = lambda scale, dt=torch.float32: (torch.randn(n + off, generator=gen) * scale).to(dt).to(dev)[off:]  # noqa: E731
    p, g, m, v = new(0.1), new(1e-2, DT[gt]), new(1e-3), new(1e-2).square_()
    hp = (1e-2, 0.9, 0.99, 1e-8, 0.1)
    for f in (0.3, 1.0, 0.0):
        norm = torch.tensor([5.0, f], device=dev)
        like = lambda: torch.empty(n + off, device=dev)[off:]  # noqa: E731
        want = [like() for _ in range(3)] + [torch.empty(n + off, device=dev, dtype=torch.bfloat16)[off:]]
        adamw(C, dev, p, (g.float() * norm[1]), m, v, 3, None, want, hp)
        got = [like() for _ in range(3)] + [torch.empty(n + off, device=dev, dtype=torch.bfloat16)[off:]]
        adamw(C, dev, p, g, m, v, 3, norm, got, hp)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        own = [t.clone() for t in (p, m, v)]
        adamw(C, dev, own[0], g, own[1], own[2], 3, norm, own, hp)
        for a, b in zip(own, want):
            assert torch.equal(a, b)


def test_adamw_against_the_formula(C, dev):
    n, hp = 3001, (1e-2, 0.9, 0.999, 1e-8, 0.01)
    lr, b1, b2, eps, wd = (struct.unpack("<f", struct.pack("<f", x))[0] for x in hp)
    g = torch.Generator().manual_seed(1)
    p, gr, m, v = (torch.randn(n, generator=g) * s for s in (0.1, 1e-2, 1e-3, 1e-2))
    v = v * v
    norm = torch.tensor([4.0, 0.25])
    outs = [torch.empty(n, device=dev) for _ in range(3)]
    adamw(C, dev, *(t.to(dev) for t in (p, gr, m, v)), 7, norm.to(dev), outs, hp)
    d = [t.double() for t in (p, gr, m, v)]
    gg = d[1] * 0.25
    mm, vv = b1 * d[2] + (1 - b1) * gg, b2 * d[3] + (1 - b2) * gg * gg
    step = lr * (mm / (1 - b1 ** 7)) / ((vv / (1 - b2 ** 7)).sqrt() + eps)
    pp = d[0] * (1 - lr * wd) - step
    u = 2.0 ** -24  # a handful of roundings in each
    mag = (b1 * d[2]).abs() + ((1 - b1) * gg).abs()
    assert ((outs[1].cpu().double() - mm).abs() <= 6 * u * mag).all()
    assert ((outs[2].cpu().double() - vv).abs() <= 8 * u * vv).all()
    off = 16 * u * step.abs() + lr * 6 * u * mag / (1 - b1 ** 7) / ((vv / (1 - b2 ** 7)).sqrt() + eps)
    assert ((outs[0].cpu().double() - pp).abs() <= off + 4 * u * (d[0].abs() + step.abs())).all()


def test_norm_then_adamw_is_clip_then_adamw(C, dev):
    """As they are used together: many tensors, their norm, and the update with
    the factor, against gradients clipped in place and the update without."""
    shapes = [(300, 257), (300,), (129, 300), (129,)]
    gs = tensors(dev, shapes, ["f32"] * 4, 8, 0.1)
    ps = tensors(dev, shapes, ["f32"] * 4, 9, 0.1)
    hp = (1e-3, 0.9, 0.999, 1e-8, 0.0)
    state = lambda: ([p.clone() for p in ps], [torch.zeros_like(p) for p in ps], [torch.zeros_like(p) for p in ps])  # noqa: E731
    a, b = state(), state()
    norm = norm_of(C, dev, gs, 1.0)
    assert norm[1] < 1
    for i in range(4):
        o = [x[i] for x in a]
        adamw(C, dev, o[0], gs[i], o[1], o[2], 1, norm, o, hp)
    norm_of(C, dev, gs, 1.0, gs)
    for i in range(4):
        o = [x[i] for x in b]
        adamw(C, dev, o[0], gs[i], o[1], o[2], 1, None, o, hp)
    for x, y in zip(a, b):
        assert all(torch.equal(s, t) for s, t in zip(x, y))
