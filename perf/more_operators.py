"""The tail of a language model's training step, through the framework's public
entry points (`_C.op_call`): what it costs on one GPU.

  linear_xent  softmax cross-entropy of a vocabulary head from the hidden rows
               and the head's weights, the logits not kept: the loss alone, or
               the loss with the gradients of both
  grad_norm    the norm of a model's gradients over all tensors and the clip
               factor; and the clipped gradients
  adamw        AdamW on gradients that are scaled by the clip factor as they
               are read
A program makes the eager calls below; the outputs and scratch are allocated
once, as a program's would be.  `run` computes either those calls (`own`) or
the same operators from elementary operations.
"""
import math
import os
import struct
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
GNRM = int.from_bytes(b"GNRM", "little")
ADAM = int.from_bytes(b"ADAM", "little")
LR, EPS, DECAY = 1e-3, 1e-8, 0.01
BETA1, BETA2 = struct.unpack("<ff", struct.pack("<ff", 0.9, 0.999))  # as the call's attributes hold them
STEP = 5  # the step that the AdamW cases take


# ---------------------------------------------------------------- the cases
def _xent(rows, classes, dim, dtype, grad, counted, weights):
    return {"kind": "xent", "rows": rows, "classes": classes, "dim": dim, "dtype": dtype, "grad": grad,
            "counted": counted, "weights": weights}


def _grads(kind, layers, dim, hidden, dtype, max_norm):
    return {"kind": kind, "layers": layers, "dim": dim, "hidden": hidden, "dtype": dtype, "max_norm": max_norm}


def _adamw(rows, cols, g, shadow):
    return {"kind": "adamw", "rows": rows, "cols": cols, "g": g, "shadow": shadow}


def listed():
    return [
        # an answer of a few tokens being scored: the weights' bytes count
        dict(_xent(16, 32000, 4096, "bf16", False, 1.0, False), name="score_16x32000x4096_bf16"),
        # a validation batch, a quarter of it prompt without labels; an odd vocabulary
        dict(_xent(4096, 50021, 1024, "f16", False, 0.75, False), name="loss_4096x50021x1024_f16"),
        # few rows that train: one short answer
        dict(_xent(64, 32003, 2048, "f16", True, 1.0, True), name="grad_64x32003x2048_f16"),
        # a training batch's tokens, a quarter of them without labels
        dict(_xent(4096, 32000, 4096, "bf16", True, 0.75, False), name="grad_4096x32000x4096_bf16"),
        # fp32 on image rows' width (784), odd numbers of rows and classes, each row with a weight of its own
        dict(_xent(1023, 10007, 784, "f32", True, 0.9, True), name="grad_1023x10007x784_f32"),
        # the largest: a batch of 8192 rows of the benchmark's width at a large vocabulary
        dict(_xent(8192, 131072, 4096, "bf16", True, 1.0, False), name="grad_8192x131072x4096_bf16"),
        # the gradients of a small MLP (784 to 256): latency
        dict(_grads("norm", 1, 784, 256, "f32", 1.0), name="norm_784x256_f32"),
        # the gradients of the benchmark's four layers of 4096 x 4096
        dict(_grads("norm", 2, 4096, 4096, "f32", 1.0), name="norm_4x4096x4096_f32"),
        # many tensors of odd sizes, matrices in bf16 and vectors in fp32, clipped
        dict(_grads("clip", 40, 1000, 1111, "mixed", 0.5), name="clip_240_tensors_mixed"),
        # one layer of the benchmark's width, with the bf16 copy of its weights
        dict(_adamw(4096, 4096, "f32", True), name="adamw_4096x4096_f32_shadow"),
        # an odd layer whose gradient is kept in 16 bits
        dict(_adamw(1003, 777, "bf16", False), name="adamw_1003x777_bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size of lo..hi, even over the logarithm: any, or a multiple of 8 or of 64."""
    n = _log(rng, lo, hi)
    step = rng.choice((1, 8, 64, 64))
    return min(max(-(-n // step) * step, lo), hi)


def draw(rng):
    kind = rng.choice(("xent", "xent", "xent", "norm", "clip", "adamw"))
    if kind == "xent":
        dtype, dim, classes = rng.choice(("bf16", "bf16", "f16", "f32")), _size(rng, 64, 4096), _size(rng, 1000, 131072)
        most = min(8192, (1 << (34 if dtype == "f32" else 37)) // (classes * dim) * 4)
        return _xent(_log(rng, 1, max(most, 8)), classes, dim, dtype, rng.random() < 0.6,
                     rng.choice((1.0, 0.9, 0.5)), rng.random() < 0.5)
    if kind == "adamw":
        return _adamw(_size(rng, 1, 8192), _size(rng, 16, 8192), rng.choice(("f32", "f32", "bf16", "f16")),
                      rng.random() < 0.5)
    return _grads(kind, _log(rng, 1, 60), _size(rng, 16, 2048), _size(rng, 16, 4096),
                  rng.choice(("f32", "bf16", "mixed", "f16")), rng.choice((0.5, 0.5, 2.0)))


# ---------------------------------------------------------------- inputs
def _scratch_bytes(case):
    """Room for the rows, their sums and up to 1 GiB of a piece of the classes."""
    es = SIZE[case["dtype"]]
    rows, dim = -(-case["rows"] // 256) * 256, -(-case["dim"] // 64) * 64
    classes = -(-case["classes"] // 256) * 256
    piece = min(1 << 30, (rows + dim) * classes * es)
    return (1 << 26) + rows * dim * (es + 4) + rows * classes // 8 + 4096 * dim * 4 + piece


def _shapes(case):
    """(shape, type) of the gradients of a model's layers: two matrices and four vectors each."""
    d, h, dtype = case["dim"], case["hidden"], case["dtype"]
    mat, vec = ("bf16", "f32") if dtype == "mixed" else (dtype, dtype)
    return case["layers"] * [((h, d), mat), ((h,), vec), ((d, h), mat), ((d,), vec), ((d,), vec), ((d,), vec)]


def _max_norm(case):
    """As a program sets it: a share of what its gradients' norm is around (the values' mean square is about 1.9e-5)."""
    return case["max_norm"] * math.sqrt(1.9e-5 * sum(math.prod(s) for s, _ in _shapes(case)))


def prepare(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    st = {"case": dict(case)}
    rnd = lambda *s: torch.randn(s, device=dev, generator=gen)  # noqa: E731
    uni = lambda *s: torch.rand(s, device=dev, generator=gen)  # noqa: E731
    if case["kind"] == "xent":
        r, v, d, dt = case["rows"], case["classes"], case["dim"], DTYPES[case["dtype"]]
        w = rnd(v, d).mul_(1.28 / math.sqrt(d))
        labels = torch.randint(0, v, (r,), device=dev, generator=gen)
        # rows whose label is anything from as likely as the others to almost certain
        x = rnd(r, d) + 6.0 * uni(r, 1) * w[labels]
        labels[uni(r) >= case["counted"]] = -1
        labels[0] = v - 1
        st["x"], st["w"], st["labels"] = x.to(dt), w.to(dt), labels.to(torch.int32)
        if case["weights"]:
            rw = 0.5 + uni(r)
            st["row_weights"] = rw / rw.sum()
        st["loss"], st["row_loss"] = torch.empty(1, device=dev), torch.empty(r, device=dev)
        if case["grad"]:
            st["dx"], st["dw"] = torch.empty((r, d), device=dev, dtype=dt), torch.empty((v, d), device=dev, dtype=dt)
        st["scratch"] = torch.empty(_scratch_bytes(case) // 4, device=dev)
    elif case["kind"] == "adamw":
        s = (case["rows"], case["cols"])
        st["p"], st["g"] = rnd(*s).mul_(0.02), rnd(*s).mul_(1e-3).to(DTYPES[case["g"]])
        st["m"], st["v"] = rnd(*s).mul_(1e-4), uni(*s).mul_(1e-6)
        st["step"] = torch.tensor(STEP, device=dev, dtype=torch.int32)
        norm = 1.0 + 3.0 * uni(1)
        st["norm"] = torch.cat([norm, 1.0 / (norm + 1e-6)])
        st["outs"] = [torch.empty(s, device=dev) for _ in range(3)]
        if case["shadow"]:
            st["outs"].append(torch.empty(s, device=dev, dtype=torch.bfloat16))
    else:
        shapes = _shapes(case)
        scale = torch.rand(len(shapes), generator=torch.Generator().manual_seed(int(seed))).mul_(4.0).sub_(10.0).exp2_()
        st["g"] = [rnd(*s).mul_(float(c)).to(DTYPES[t]) for (s, t), c in zip(shapes, scale)]
        st["norm"], st["scratch"] = torch.empty(2, device=dev), torch.empty(2048 * (1 + len(shapes) // 64), device=dev)
        if case["kind"] == "clip":
            # the clipped gradients one behind the other, in a buffer for each type
            st["flat"] = {t: torch.empty(sum(g.numel() for g in st["g"] if g.dtype == t), device=dev, dtype=t)
                          for t in sorted({g.dtype for g in st["g"]}, key=str)}
            at = dict.fromkeys(st["flat"], 0)
            st["outs"] = []
            for g in st["g"]:
                st["outs"].append(st["flat"][g.dtype][at[g.dtype]:at[g.dtype] + g.numel()].view_as(g))
                at[g.dtype] += g.numel()
    return st


# ---------------------------------------------------------------- the framework's calls
def _ops():
    p = os.path.abspath(os.path.join("ai-compiler-framework_amd", "python"))
    if p not in sys.path:
        sys.path.insert(0, p)
    from aicf_cuda import _C

    return _C


def _run_own(st):
    case, C = st["case"], _ops()
    if case["kind"] == "xent":
        ins = [st[n] for n in ("x", "w", "labels", "row_weights") if n in st]
        outs = [st[n] for n in ("loss", "dx", "dw", "row_loss") if n in st]
        C.op_call(C.OpKind.LinearXent, ins, outs + [st["scratch"]])
        return outs
    if case["kind"] == "adamw":
        C.op_call(C.OpKind.AdamStep, [st[n] for n in ("p", "g", "m", "v", "step", "norm")], st["outs"], ADAM,
                  struct.pack("<fffff", LR, BETA1, BETA2, EPS, DECAY))
        return st["outs"]
    outs = st.get("outs", [])
    C.op_call(C.OpKind.GradNorm, st["g"], [st["norm"], st["scratch"]] + outs, GNRM, struct.pack("<f", _max_norm(case)))
    return [st["norm"]] + list(st.get("flat", {}).values())


# ---------------------------------------------------------------- the plain forms
def _xent_plain(st):
    x, w, v = st["x"].float(), st["w"].float(), st["w"].shape[0]
    labels = st["labels"].long()
    known = (labels >= 0) & (labels < v)
    at = labels.clamp(0, v - 1)[:, None]
    rw = st["row_weights"] if "row_weights" in st else known.float() / known.sum().clamp(min=1)
    rw = torch.where(known, rw, 0.0)
    z = x @ w.t()
    top = z.amax(1, keepdim=True)
    e = (z - top).exp_()
    s = e.sum(1, keepdim=True)
    row_loss = torch.where(rw != 0, (s.log() + top - z.gather(1, at))[:, 0], 0.0)
    loss = (rw.double() * row_loss.double()).sum().float().reshape(1)
    if not st["case"]["grad"]:
        return [loss, row_loss]
    g = e.mul_(rw[:, None] / s)
    g.scatter_add_(1, at, -rw[:, None])
    return [loss, (g @ w).to(st["x"].dtype), (g.t() @ x).to(st["w"].dtype), row_loss]


def _norm_plain(st):
    max_norm = _max_norm(st["case"])
    norm = torch.stack([g.float().square().sum() for g in st["g"]]).sum().sqrt()
    factor = (max_norm / (norm + 1e-6)).clamp(max=1.0)
    outs = [torch.cat([(g.float() * factor).to(t).view(-1) for g in st["g"] if g.dtype == t]) for t in st.get("flat", {})]
    return [torch.stack([norm, factor])] + outs


def _adamw_plain(st):
    g = st["g"].float() * st["norm"][1]
    m = BETA1 * st["m"] + (1.0 - BETA1) * g
    v = BETA2 * st["v"] + (1.0 - BETA2) * g * g
    t = st["step"].double()
    c1, c2 = 1.0 - BETA1 ** t, 1.0 - BETA2 ** t
    p = st["p"] * (1.0 - LR * DECAY) - (LR / c1).float() * m / ((v / c2.float()).sqrt() + EPS)
    return [p, m, v] + ([p.to(torch.bfloat16)] if st["case"]["shadow"] else [])


def _run_plain(st):
    return {"xent": _xent_plain, "adamw": _adamw_plain, "norm": _norm_plain, "clip": _norm_plain}[st["case"]["kind"]](st)


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ---------------------------------------------------------------- the least work
def work(case):
    if case["kind"] == "xent":
        r, v, d, es = case["rows"], case["classes"], case["dim"], SIZE[case["dtype"]]
        n = max(1, round(r * case["counted"]))  # the rows that count; the others' gradient is written
        size = (n + v) * d * es + 8 * r + (4 * r if case["weights"] else 0)
        if case["grad"]:
            size += (r + v) * d * es
        return {"bytes": size, "flops": (6 if case["grad"] else 2) * n * v * d}
    if case["kind"] == "adamw":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (24 + SIZE[case["g"]] + (2 if case["shadow"] else 0)), "flops": 14 * n}
    n = sum(math.prod(s) for s, _ in _shapes(case))
    size = sum(math.prod(s) * SIZE[t] for s, t in _shapes(case))
    return {"bytes": size * (1 if case["kind"] == "norm" else 2), "flops": n * (2 if case["kind"] == "norm" else 3)}


# ---------------------------------------------------------------- the definitions in 64 bits
def _xent_exact(st):
    r, (v, d) = st["x"].shape[0], st["w"].shape
    dev, f64 = st["x"].device, torch.float64
    w = st["w"].to(f64)
    wt = w.t().contiguous()
    labels = st["labels"].long()
    ok = (labels >= 0) & (labels < v)
    if "row_weights" in st:
        rw = st["row_weights"].to(f64) * ok
    else:
        rw = ok.to(f64) / max(1, int(ok.sum()))
    row_loss = torch.zeros(r, device=dev, dtype=f64)
    dx = torch.zeros((r, d), device=dev, dtype=f64)
    dw = torch.zeros((v, d), device=dev, dtype=f64) if st["case"]["grad"] else None
    rows = (rw != 0).nonzero()[:, 0]
    for i in rows.split(max(1, (1 << 28) // v)):
        x = st["x"][i].to(f64)
        z = torch.mm(x, wt)
        at = torch.arange(len(i), device=dev)
        lse = torch.logsumexp(z, 1)
        row_loss[i] = lse - z[at, labels[i]]
        if dw is not None:
            z = torch.softmax(z, 1)
            z[at, labels[i]] -= 1.0
            z *= rw[i][:, None]
            dx[i] = torch.mm(z, w)
            dw += torch.mm(z.t().contiguous(), x)
    loss = torch.dot(rw, row_loss).reshape(1)
    return [loss, row_loss] if dw is None else [loss, dx, dw, row_loss]


def exact(case, seed):
    st = prepare(case, seed)
    f64 = torch.float64
    if case["kind"] == "xent":
        return _xent_exact(st)
    if case["kind"] == "adamw":
        g = st["g"].to(f64) * st["norm"][1].to(f64)
        m = torch.lerp(g, st["m"].to(f64), BETA1)
        v = torch.lerp(g ** 2, st["v"].to(f64), BETA2)
        hat = (m / (1 - BETA1 ** STEP)) / ((v / (1 - BETA2 ** STEP)).sqrt() + EPS)
        p = st["p"].to(f64) * (1 - LR * DECAY) - LR * hat
        return [p, m, v] + ([p] if case["shadow"] else [])
    total = math.fsum(float(torch.linalg.vector_norm(g.to(f64)) ** 2) for g in st["g"])
    norm = math.sqrt(total)
    factor = min(1.0, _max_norm(case) / (norm + 1e-6))
    outs = [torch.cat([g.flatten().to(f64) for g in st["g"] if g.dtype == t]) * factor for t in st.get("flat", {})]
    return [torch.tensor([norm, factor], dtype=f64, device="cuda:0")] + outs
