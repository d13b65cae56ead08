"""Calls of the vocabulary-head ops at the borders of what they take, on the
host before any launch (the addresses are never touched)."""
from __future__ import annotations

import ctypes
import struct

import pytest

from aicf_cuda import abi
from test_head_ops import DISTILL, DTOP, F32, I32, At, refused


@pytest.mark.parametrize("tau,taken", [(2.0 ** -60, True), (2.0 ** 60, True), (1.0, True), (2.0 ** -61, False),
                                       (2.0 ** 61, False), (1e-39, False), (3e38, False)])
def test_distill_temperature(tau, taken):
    """Where log2(e) / tau or tau^2 would leave f32's range the call is refused."""
    lib, d = abi.load(), At()
    ins, outs = [d((2, 50)), d((2, 3)), d((2, 3), I32)], [d((1,)), d((2, 50)), d((2,))]
    if not taken:
        return refused(lib, DISTILL, ins, outs, DTOP, struct.pack("<ff", tau, 0.0))
    # taken: the launch itself turns down an output without memory
    outs[2] = abi.make_desc(None, F32, (2,))
    blob, keep = abi.make_blob(DTOP, struct.pack("<ff", tau, 0.0))
    st = lib.aicf_dispatch_v0(DISTILL, abi.desc_array(ins), 3, abi.desc_array(outs), 3, ctypes.byref(blob), None)
    assert st == abi.STATUS_INVALID_ARGUMENT
