"""Lowering of AdamW steps whose clip factor comes from outside the graph: the
norm is a plan's input (of gradients on several ranks, say), no grad_norm makes it."""
from __future__ import annotations

import pytest

from aicf_hip.lower import compile_lowered
from aicf_hip.mlp import build_mlp_mse

FUSIONS = [dict(fuse_optimizer=True), dict(fuse_tail=True, fuse_colsum=True), dict(fuse_small=True),
           dict(fuse_optimizer=True, fuse_colsum=True, fuse_tail=True, fuse_small=True)]


@pytest.mark.parametrize("fusions", FUSIONS, ids=lambda f: "+".join(f))
def test_flat_step_with_a_norm_from_outside(fusions):
    """The flat update of the benchmark's step, with the norm as its sixth input, keeps its own launch."""
    ir, _, _ = build_mlp_mse(1024, 512, 3, device="cpu")
    plain = compile_lowered(ir, fuse_bias=True)
    norm = ir.new_value(name="norm", shape=(2,), dtype="torch.float32", device="cpu")
    step = next(n for n in ir.nodes if n.op == "AdamWStep")
    step.inputs.append(norm.id)
    low = compile_lowered(ir, fuse_bias=True, **fusions)
    adam = [it for it in low if it["op"] == "adamw_step"]
    assert len(adam) == 1 and adam[0]["kernel_id"] == "adamw_step_clip_v0"
    assert list(adam[0]["inputs"]) == list(step.inputs) and list(adam[0]["outputs"]) == list(step.outputs)
    ops = [it["op"] for it in low]
    assert not {"gemm_adamw", "colsum_adamw", "mse_colsum", "adamw_multi", "grad_group_adamw"} & set(ops)
    assert ops[-2:] == ["step_inc", "adamw_step"]
    made = lambda items: {int(o) for it in items for o in it["outputs"]}  # noqa: E731
    assert made(plain) <= made(low)  # every gradient is still written


def test_the_same_step_without_the_norm_is_fused():
    ir, _, _ = build_mlp_mse(1024, 512, 3, device="cpu")
    ops = [it["op"] for it in compile_lowered(ir, fuse_bias=True, fuse_optimizer=True)]
    assert ops.count("gemm_adamw") == 3
    ops = [it["op"] for it in compile_lowered(ir, fuse_bias=True, fuse_optimizer=True, fuse_colsum=True, fuse_tail=True)]
    assert "colsum_adamw" in ops
