"""The distillation step of the plan runtime: Linear layers in 8 bits lowered
to quantisations and products, a token drawn a row, the loss from a teacher's
top logits, gradients and AdamW; its lowering, and on the device every value of
a step against the 64-bit formulas, eager and replayed."""
from __future__ import annotations

import pytest
import torch

import head_ref as ref
from aicf_hip import lowered_to_text
from aicf_hip.ir import IRGraph
from aicf_hip.lower import compile_lowered
from aicf_hip.mlp import build_mlp_distill, init_mlp_distill, make_executor

SIZES = dict(B=48, din=200, dh=256, V=1003, K=16)


def test_lowering():
    ir, low, plan = build_mlp_distill(**SIZES, tau=2.0, label_weight=0.25, pow2=True)
    lin = ["quant_fp8", "quant_fp8", "gemm_fp8"]
    assert [o["op"] for o in low] == (lin + ["gelu"] + lin + ["sample_row", "distill_topk", "quant_fp8", "gemm_fp8",
                                      "gemm_fp8", "reduce_sum", "gelu_bwd", "quant_fp8", "gemm_fp8", "reduce_sum",
                                      "step_inc"] + ["adamw_step"] * 4)
    assert all(o["kernel_id"] for o in low)
    name = lambda v: ir.values[v].name  # noqa: E731
    by = {name(o["outputs"][0]): [name(v) for v in o["inputs"]] for o in low if o["op"] == "gemm_fp8"}
    assert by == {"z1": ["x.q", "x.s", "1.W8.q", "1.W8.s", "1.b"], "logits": ["h1.q", "h1.s", "2.W8.q", "2.W8.s", "2.b"],
                  "d_h1": ["dY.q", "dY.s", "2.W8.qT", "2.W8.sT"], "d_2.W": ["dY.qT", "dY.sT", "h1.qT", "h1.sT"],
                  "d_1.W": ["d_z1.qT", "d_z1.sT", "x.qT", "x.sT"]}
    assert {plan.specs[v].name for v in plan.params} == {"1.W", "1.b", "2.W", "2.b"}
    assert "gemm_fp8_mfma_v0" in lowered_to_text(low, "distill")


def test_weights_quantised_once_and_refusals():
    """quant_w=False leaves the weight's codes as they are; wrong numbers of values are refused."""
    ir = IRGraph()
    nv = lambda n, s, dt="torch.float32": ir.new_value(name=n, shape=s, dtype=dt)  # noqa: E731
    x, w, y = nv("x", (4, 128)), nv("0.W", (8, 128)), nv("y", (4, 8))
    q = [nv("xq", (4, 128), "torch.float8_e4m3fn"), nv("xs", (4, 1)), nv("wq", (8, 128), "torch.float8_e4m3fn"),
         nv("ws", (1, 1))]
    ir.emit(op="LinearFp8", inputs=[x, w], outputs=[y] + q, attrs={"quant_w": False})
    assert [o["op"] for o in compile_lowered(ir)] == ["quant_fp8", "gemm_fp8"]
    for node in (dict(op="LinearFp8", inputs=[x, w], outputs=[y] + q[:2]),
                 dict(op="LinearFp8", inputs=[x, w], outputs=[y] + q, attrs={"bias": True}),
                 dict(op="LinearFp8Bwd", inputs=[y, q[0], q[1]], outputs=[w] + q, attrs={"need_dx": True})):
        bad = IRGraph(values=ir.values)
        bad.emit(**node)
        with pytest.raises(RuntimeError, match="linear_fp8"):
            compile_lowered(bad)


def gelu_grad(z):
    z = z.clone().requires_grad_()
    torch.nn.functional.gelu(z, approximate="tanh").sum().backward()
    return z.grad


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [SIZES, dict(B=50, din=128, dh=96, V=300, K=4),
                                   dict(B=5, din=64, dh=130, V=50021, K=33)])
def test_step_eager_and_replayed(sizes):
    ir, low, plan = build_mlp_distill(**sizes, tau=2.0, label_weight=0.25)
    B = sizes["B"]
    outs = ("token", "logprob", "loss", "row_loss", "dY", "d_1.W", "d_2.W", "d_1.b", "d_2.b")

    def states(replayed):
        """The values of three steps and the parameters after them."""
        ins, params = init_mlp_distill(**sizes)
        first = {k: v.clone() for k, v in params.items()}
        ex = make_executor(ir, low, plan, own_graph=True)
        if replayed:
            ex.capture(inputs=ins, params=params)
        seen = []
        for _ in range(3):
            ex.replay() if replayed else ex.run(inputs=ins, params=params)
            torch.cuda.synchronize()
            seen.append({n: ex.value(n).cpu() for n in outs})
        if not replayed:
            check(ex, ins)
        assert all(not torch.equal(first[k], params[k]) for k in params)
        end = {k: v.cpu() for k, v in params.items()}
        ex.close()
        return seen + [end]

    def check(ex, ins):
        """The last step's values, each from the stored values before it."""
        val = lambda n: ex.value(n).cpu()  # noqa: E731
        z = val("logits")
        c = {k: v.cpu() for k, v in ins.items()}
        loss, grad, _, bound = ref.distill(z, c["teacher"], c["teacher.ids"], 2.0, 0.25, c["t"])[:4]
        assert ((val("dY").double() - grad).abs() <= bound).all()
        for i in range(B):
            assert val("token")[i] == ref.sample(z[i], *(c[k][i].item() for k in
                                                 ("u", "temperature", "top_k", "top_p", "min_p")))[0]
        # gradients from the stored dY, d_h1, h1 and x: e5m2 codes (half a step 2^-3) times e4m3 codes (2^-4), and
        # the rounding of d_z1 to bf16, errors of either sign
        rel = 2.0 ** -3 + 2.0 ** -4 + 2.0 ** -8
        dy = val("dY").double()
        dz = val("d_h1").double() * gelu_grad(val("z1").double())
        for got, want in (("d_2.W", dy.t() @ val("h1").double()), ("d_1.W", dz.t() @ c["x"].double()),
                          ("d_2.b", dy.sum(0)), ("d_1.b", dz.sum(0))):
            assert (val(got).double() - want).norm() <= rel * want.norm(), got

    eager, replayed = states(False), states(True)
    for a, b in zip(eager, replayed):
        assert all(torch.equal(a[n], b[n]) for n in a)
    assert eager[0]["loss"].item() != eager[1]["loss"].item()
