"""The language-model step of the plan runtime: linear cross-entropy, gradient
norm, AdamW with the clip factor; its lowering, and on the device every value of
a step against the 64-bit formulas, eager and replayed."""
from __future__ import annotations

import pytest
import torch

import tail_ref as ref
from aicf_hip.mlp import build_mlp_lm, init_mlp_lm, make_executor

SIZES = dict(B=48, din=200, dh=256, V=1003)


def test_lowering():
    ir, low, plan = build_mlp_lm(**SIZES)
    assert [o["op"] for o in low] == ["gemm_epilogue", "linear_xent", "gelu_bwd", "gemm", "reduce_sum", "grad_norm",
                                      "step_inc"] + ["adamw_step"] * 3
    assert [o["kernel_id"] for o in low][-3:] == ["adamw_step_clip_v0"] * 3
    assert {plan.specs[v].name for v in plan.params} == {"1.W", "1.b", "2.W", "1.Wb", "2.Wb"}
    ir, low, _ = build_mlp_lm(**SIZES, clip_in_place=True)
    assert [o["kernel_id"] for o in low][-3:] == ["adamw_step_f32_v1"] * 3
    norm = next(o for o in low if o["op"] == "grad_norm")
    assert norm["outputs"][2:] == norm["inputs"]


def test_updates_stay_behind_the_norm():
    """StageF leaves AdamW its own launches where a norm of all gradients comes first."""
    _, low, _ = build_mlp_lm(**SIZES, clip_in_place=True, fuse_small=True)
    ops = [o["op"] for o in low]
    assert "grad_group_adamw" not in ops
    assert ops.index("grad_norm") < min(i for i, o in enumerate(ops) if o.startswith("adamw"))


def gelu_grad(z):
    z = z.clone().requires_grad_()
    torch.nn.functional.gelu(z, approximate="tanh").sum().backward()
    return z.grad


@pytest.mark.gpu
@pytest.mark.parametrize("sizes,piece", [(SIZES, 0), (dict(B=300, din=128, dh=128, V=2000), 512),
                                         (dict(B=5, din=64, dh=130, V=5021), 0)])
def test_step_eager_and_replayed(sizes, piece):
    B = sizes["B"]
    outs = ("loss", "row_loss", "d_h1", "d_1.W", "d_2.W", "d_1.b", "norm")
    built = {c: build_mlp_lm(**sizes, max_norm=0.05, piece=piece, clip_in_place=c) for c in (False, True)}

    def states(replayed, clip_in_place=False):
        """The values of three steps and the parameters after them."""
        ins, params = init_mlp_lm(**sizes)
        first = {k: v.clone() for k, v in params.items()}
        ex = make_executor(*built[clip_in_place], own_graph=True)
        if replayed:
            ex.capture(inputs=ins, params=params)
        seen = []
        for _ in range(3):
            before = {k: v.cpu() for k, v in params.items()}
            ex.replay() if replayed else ex.run(inputs=ins, params=params)
            torch.cuda.synchronize()
            seen.append({n: ex.value(n).cpu() for n in outs})
        if not replayed and not clip_in_place:
            check(ex, ins, before)
        assert all(not torch.equal(first[k], params[k]) for k in params)
        assert all(torch.equal(params[f"{k}.Wb"], params[f"{k}.W"].to(torch.bfloat16)) for k in "12")
        end = {k: v.cpu() for k, v in params.items()}
        ex.close()
        return seen + [end]

    def check(ex, ins, before):
        """The last step's values, each from the stored values before it."""
        val = lambda n: ex.value(n).cpu()  # noqa: E731
        loss, dx, dw, rl, bt, bx, bw, bl = ref.linear_xent(val("h1"), before["2.Wb"], ins["t"].cpu())
        assert abs(float(val("loss")) - float(loss)) <= bt and ((val("row_loss").double() - rl).abs() <= bl).all()
        assert ((val("d_h1").double() - dx).abs() <= ref.rounded(bx, dx, torch.bfloat16)).all()
        assert ((val("d_2.W").double() - dw).abs() <= ref.rounded(bw, dw, torch.float32)).all()
        # d_z1 in bf16 (half a step 2^-8), then a product and a sum of it
        dz = val("d_h1").double() * gelu_grad(val("z1").double())
        for n, want in (("d_1.W", dz.t() @ ins["x"].cpu().double()), ("d_1.b", dz.sum(0))):
            assert (val(n).double() - want).norm() <= 2.0 ** -8 * want.norm(), n
        want = ref.grad_norm([val(n) for n in ("d_1.W", "d_1.b", "d_2.W")], 0.05)
        assert all(abs(a - b) <= 2.0 ** -22 * b for a, b in zip(val("norm").tolist(), want)) and want[1] < 1

    eager, replayed, in_place = states(False), states(True), states(False, True)
    for a, b in zip(eager, replayed):
        assert all(torch.equal(a[n], b[n]) for n in a)
    assert all(torch.equal(eager[-1][k], in_place[-1][k]) for k in eager[-1])  # the same bits either way
    assert eager[0]["loss"].item() != eager[1]["loss"].item()
    assert (eager[0]["row_loss"][3::4] == 0).all() and eager[0]["loss"].item() == pytest.approx(
        eager[0]["row_loss"].double().sum().item() / (B - B // 4), rel=1e-6)
