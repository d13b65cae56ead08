"""Plain definitions, in 64 bits, of the ops of a training step's tail
(linear_xent, grad_norm, AdamW with the clip factor), and the bounds that their
outputs have to keep.  U is half a step of f32, relative."""
from __future__ import annotations

import math

import torch

from head_ref import HALF_STEP, TINY, U


def linear_xent(x, w, labels, rw=None, piece=None):
    """loss, dX, dW, row loss in 64 bits and a bound for each but the first."""
    dt = x.dtype
    r, d = x.shape
    v = w.shape[0]
    x, w = x.double(), w.double()
    ok = (labels >= 0) & (labels < v)
    wr = torch.where(ok, rw.double() if rw is not None else 1.0 / max(int(ok.sum()), 1), 0.0)
    counts = ok & (wr != 0)
    i = counts.nonzero()[:, 0]
    xi, wi, lab, at = x[i], wr[i][:, None], labels[i].long(), torch.arange(len(i), device=x.device)
    z = xi @ w.t()
    lse = torch.logsumexp(z, 1, keepdim=True)
    zl = z[at, lab][:, None]
    rl, dx = torch.zeros(r, dtype=torch.float64, device=x.device), torch.zeros_like(x)
    rl[i] = (lse - zl)[:, 0]
    p = (z - lse).exp()
    g = p.clone()
    g[at, lab] -= 1.0
    g = g * wi
    dx[i] = g @ w
    dw = g.t() @ xi
    # A logit: d products (and the padding to a K-step) in f32, each addition off by at most a whole step.
    far = (d + 64) * 2 * U * (xi.abs() @ w.abs().t())
    top = z.amax(1, keepdim=True)
    m = torch.where(z == -math.inf, 0.0, top - z)
    # A probability, relative: its logit's and the sum's logits' errors, the additions of the sum (256 classes a
    # tile, its lanes and waves, then the tiles), the exponents' arguments (3 roundings) and two exponentials.
    rel_sum = (256 + v / 128 + 32) * 2 * U
    most = far.amax(1, keepdim=True)
    rel = (2 * (far + most)).expm1() + rel_sum + 6 * U * (m + 1) + 12 * U
    pe = torch.where(z == -math.inf, 0.0, p * rel)
    bl = torch.zeros_like(rl)
    bl[i] = (2 * most + rel_sum + 8 * U * (lse.abs() + zl.abs() + (top - zl).abs() + 4))[:, 0]
    # G in the operands' type: the numerator is rounded, then G itself; one more rounding each of the products
    # in f32.  Numerators of 16-bit operands are kept in f16, scaled to at most 2^14: half steps of 2^-25 below the
    # normal numbers, 2^-39 of their tile's largest, which is at most the row's.  f16: G too, scaled to 2^13.
    h = HALF_STEP[dt]
    ge = wi.abs() * pe + h * (wi.abs() * (p + pe)) + h * (g.abs() + wi.abs() * pe) + 4 * U * wi.abs() * (p + 1)
    if dt == torch.float16:
        big = wr.abs().max() if len(i) else 0.0
        ge = ge + 2.0 ** -36 * big
    if dt != torch.float32:
        ge = ge + 2.0 ** -39 * wi.abs()
    e = wi.abs() * 2.0 ** -120  # (exponentials below the normal numbers are zero)
    ge = ge + e
    bx = torch.zeros_like(x)
    bx[i] = ge @ w.abs() + (v + 256) * 2 * U * ((g.abs() + ge) @ w.abs())
    bw = ge.t() @ xi.abs() + (r + 256) * 2 * U * ((g.abs() + ge).t() @ xi.abs())
    loss = (wr[i] * rl[i]).sum()
    bt = (wr[i].abs() * bl[i]).sum() + 4 * U * (wr[i].abs() * rl[i].abs()).sum()
    return loss, dx, dw, rl, bt, bx, bw, bl


def rounded(bound, value, dt):
    """The bound after one rounding to the type."""
    return bound + HALF_STEP[dt] * (value.abs() + bound) + TINY[dt]


def grad_norm(gs, max_norm):
    norm = math.sqrt(math.fsum(float(g.double().square().sum()) for g in gs))
    f = max_norm / (norm + 1e-6)
    return norm, min(f, 1.0)
