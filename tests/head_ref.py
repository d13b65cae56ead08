"""Plain definitions, in 64 bits on the CPU, of the 8-bit and vocabulary-head
ops (quant_fp8, gemm_fp8, distill_topk, sample_row), and the bounds that
their outputs have to keep.  U is half a step of f32, relative."""
from __future__ import annotations

import math

import torch

U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half a subnormal step
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
FMAX = {"e4m3": 448.0, "e5m2": 57344.0}


def blocks(n):
    return -(-n // 128)


def spread(s, rows, cols):
    """The scale of each element, for scales by rows or by blocks."""
    s = s.repeat_interleave(128, 1)[:, :cols]
    return s if s.shape[0] == rows else s.repeat_interleave(128, 0)[:rows]


def quant(x, fp8, by, pow2):
    """Codes and scales with the op's own f32 steps, so both are bit for bit."""
    x = x.float()
    r, c = x.shape
    pad = torch.nn.functional.pad(x.abs(), (0, -c % 128, 0, -r % 128 if by == "blocks" else 0))
    amax = pad.view(r, -1, 128).amax(2) if by == "rows" else pad.view(blocks(r), 128, -1, 128).amax(3).amax(1)
    s = (amax / FMAX[fp8]).clamp_min(2.0 ** -126)
    if pow2:
        up = ((s.view(torch.int32).long() + 0x7FFFFF) & 0x7F800000).to(torch.int32).view(torch.float32)
        s = torch.where(s.isnan(), s, up)
    q = (x * spread(1.0 / s, r, c)).to(FP8[fp8])
    return q, s


def gemm(a, sa, b, sb, bias=None):
    """The product in 64 bits, and the sum of the terms' magnitudes."""
    x = a.float().double() * spread(sa.double(), *a.shape)
    y = b.float().double() * spread(sb.double(), *b.shape)
    c, mag = x @ y.t(), x.abs() @ y.abs().t()
    if bias is not None:
        c, mag = c + bias.double(), mag + bias.double().abs()
    return c, mag


def group_max(a, sa, b, sb):
    """Over the groups of 8 consecutive K: the sum of each group's largest product's magnitude."""
    x = (a.float().double() * spread(sa.double(), *a.shape)).abs()
    y = (b.float().double() * spread(sb.double(), *b.shape)).abs()
    total = torch.zeros((x.shape[0], y.shape[0]), dtype=torch.float64)
    for k in range(0, x.shape[1], 8):
        top = torch.zeros_like(total)
        for e in range(k, min(k + 8, x.shape[1])):
            top = torch.maximum(top, x[:, e, None] * y[None, :, e])
        total += top
    return total


def gemm_bound(c, mag, k, out, groups=None):
    """128 products and the blocks' sums in f32, each step off by at most a
    whole step (the matrix cores may truncate), two more for the scales and
    one for the bias; then one rounding to the output's type.  Outputs of 16
    bits (`groups`: group_max) come from the 8-bit matrix instructions: in a
    group of 8 products the 7 smaller ones are cut to multiples of 2^-13 of
    the largest one's power of two, so each is off by less than 2^-13 of the
    largest."""
    f32 = (128 + blocks(k) + 4) * 2 * U * mag
    if out != torch.float32:
        f32 = f32 + 7 * 2.0 ** -13 * groups
    return f32 + HALF_STEP[out] * (c.abs() + f32) + TINY[out]


def distill(z, t, ids, tau, alpha, labels=None, w=None):
    """loss, dz, row_loss in 64 bits, and bounds for dz and row_loss."""
    dt = z.dtype
    z, t = z.double(), t.double()
    r, v = z.shape
    wr = w.double() if w is not None else torch.full((r,), 1.0 / r, dtype=torch.float64)
    dz, rl = torch.zeros_like(z), torch.zeros(r, dtype=torch.float64)
    bz, bl = torch.zeros_like(z), torch.zeros(r, dtype=torch.float64)
    # of a probability's relative error: the sum over a lane's elements and the tree (v / 2048 + 20 steps
    # cover every division of a row), 2 steps of an exponential's result
    rel_sum = (v / 2048 + 24) * 2 * U
    for i in range(r):
        if wr[i] == 0:
            continue
        m = z[i].max()
        lq = torch.log_softmax(z[i] / tau, 0)
        # an exponential's argument is off by 3 roundings of itself
        rel = rel_sum + 3 * U * torch.where(z[i] == -math.inf, 0.0, (m - z[i]) / tau) + 4 * U
        given = [(int(c), float(x)) for c, x in zip(ids[i], t[i]) if 0 <= c < v]
        soft, part, g, mag = 0.0, 0.0, torch.zeros(v, dtype=torch.float64), torch.zeros(v, dtype=torch.float64)
        if given:
            lt = torch.log_softmax(torch.tensor([x for _, x in given], dtype=torch.float64) / tau, 0)
            tmax = max(x for _, x in given)
            g, mag = lq.exp(), lq.exp() * rel
            for (c, x), lp in zip(given, lt):
                p = lp.exp()
                if p > 0:
                    soft += p * (lp - lq[c])
                    # the terms' parts, 8 roundings each; the sums' logarithms by rel_sum
                    part += p * (8 * U * (lp.abs() + lq[c].abs() + (m - z[i, c]).abs() / tau + (tmax - x) / tau + 8)
                                 + 2 * rel_sum)
                    part += p * rel_sum * (lp - lq[c]).abs()
                    g[c] -= p
                    mag[c] += p * (rel_sum + 3 * U * (tmax - x) / tau + 6 * U)
        g, mag = g * (1 - alpha) * tau, mag * (1 - alpha) * tau
        rl[i], bl[i] = (1 - alpha) * tau * tau * soft, (1 - alpha) * tau * tau * part
        if alpha and labels is not None and 0 <= labels[i] < v:
            lq1 = torch.log_softmax(z[i], 0)
            rel1 = rel_sum + 3 * U * torch.where(z[i] == -math.inf, 0.0, m - z[i]) + 4 * U
            g, mag = g + alpha * lq1.exp(), mag + alpha * lq1.exp() * rel1
            g[labels[i]] -= alpha
            mag[labels[i]] += alpha * 4 * U
            rl[i] -= alpha * lq1[labels[i]]
            bl[i] += alpha * (8 * U * (lq1[labels[i]].abs() + (m - z[i, labels[i]]).abs() + 8) + 2 * rel_sum)
        dz[i] = wr[i] * g
        # the weighted parts once more, and one rounding to the type
        bz[i] = wr[i] * (mag + 6 * U * g.abs())
    bz = bz + HALF_STEP[dt] * (dz.abs() + bz) + TINY[dt]
    bl = bl + 4 * U * rl.abs()
    return (wr * rl).sum(), dz, rl, bz, bl


def sample(z, u, temperature, top_k, top_p, min_p):
    """(token, log-probability) of one row, in 64 bits."""
    z = torch.where(z.isnan(), -math.inf, z.double())
    u = min(u, 1 - 2.0 ** -24) if u > 0 else 0.0
    top = z.max()
    if top == -math.inf:
        return -1, -math.inf
    order = torch.sort(z, descending=True, stable=True).indices
    if not temperature > 0:
        return int(order[0]), 0.0
    w = torch.where(z == top, 1.0, torch.exp(-((top - z) / temperature).nan_to_num(nan=math.inf, posinf=math.inf)))
    w = torch.where(z == -math.inf, 0.0, w)
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        mass = w[order]
        before = torch.cat([torch.zeros(1, dtype=torch.float64), mass.cumsum(0)[:-1]])
        keep = before < top_p * mass.sum()
        keep[0] = True
        order = order[keep]
    if min_p > 0:
        order = order[w[order] >= min(min_p, 1.0)]
    order = order[w[order] > 0].sort().values
    cum = w[order].cumsum(0)
    at = min(int((cum <= u * cum[-1]).sum()), len(order) - 1)
    return int(order[at]), math.log(float(w[order[at]] / cum[-1]))
