"""The scratch that linear_xent asks for over a given W: exactly that much is
taken, wherever W's rows lie.  On the host (the addresses are never touched)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from aicf_cuda import _C, abi
from test_head_ops import BF16, F16, F32, I32, At
from test_tail_ops import XENT, refused, scratch, taken

SIZE = {F32: 4, F16: 2, BF16: 2}


@pytest.fixture(scope="module")
def lib():
    return abi.load()


def wanted(lib, rows, w, grad=1, piece=0):
    return lib.aicf_linear_xent_scratch_for(rows, ctypes.byref(w), grad, piece)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("r,v,dim,ld,off", [(64, 1000, 128, 128, 0), (64, 1000, 128, 128, 1), (5, 1000, 128, 129, 0),
                                            (300, 2049, 64, 72, 0), (40, 200, 100, 100, 3), (1, 1, 8, 8, 1),
                                            (7, 600, 33, 40, 0)])
def test_exactly_what_is_asked_for_is_taken(lib, r, v, dim, ld, off, dt):
    d = At()
    x, lab, loss, rl = d((r, dim), dt), d((r,), I32), d((1,)), d((r,))
    w = d((v, dim), dt, (ld, 1), (97 << 40) + off * SIZE[dt])
    dx, dw = d((r, dim), dt), d((v, dim), dt)
    missing = abi.make_desc(None, F32, (r,))
    for grad, piece in ((0, 0), (0, 256), (1, 0), (1, 256), (1, 512)):
        n = wanted(lib, r, w, grad, piece)
        assert n > 0 and n % 256 == 0
        least = wanted(lib, r, w, grad, 256)
        outs = lambda k, row_loss: [loss] + ([dx, dw] if grad else []) + [row_loss, d((k // 4,))]  # noqa: E731
        taken(lib, XENT, [x, w, lab], outs(n, missing))
        refused(lib, XENT, [x, w, lab], outs(least - 256, rl))


def test_a_copy_is_counted(lib):
    d = At()
    for dt in (F32, BF16):
        es = SIZE[dt]
        whole = scratch(lib, 64, 1000, 128, dt, 0)
        assert wanted(lib, 64, d((1000, 128), dt), 0) == whole  # contiguous, on 16 bytes
        assert wanted(lib, 64, d((1000, 128), dt, (160, 1)), 0) == whole  # rows apart by whole 16-byte steps
        for w in (d((1000, 128), dt, None, (97 << 40) + es), d((1000, 128), dt, (129, 1)), d((1000, 128), dt, (0, 1))):
            assert wanted(lib, 64, w, 0) - whole == 1024 * 128 * es
            assert wanted(lib, 64, w, 0, 256) - whole == 256 * 128 * es
        assert wanted(lib, 64, d((1000, 100), dt)) == scratch(lib, 64, 1000, 100, dt)
        assert wanted(lib, 64, d((1000, 99), dt)) == scratch(lib, 64, 1000, 99, dt)


def test_refuses(lib):
    d = At()
    assert lib.aicf_linear_xent_scratch_for(64, None, 1, 0) == -1
    for w in (d((1000, 128), I32), d((1000,)), d((10, 10, 10)), d((0, 128)), d((1000, 0)), d((1000, 128), F32, (1, 1000)),
              d((2 ** 28 + 1, 64)), d((10, 2 ** 23))):
        assert wanted(lib, 64, w) == -1
    assert wanted(lib, -1, d((1000, 128))) == -1 and wanted(lib, 2 ** 31, d((1000, 128))) == -1


def test_from_python():
    base = torch.empty(1000 * 136 + 8, dtype=torch.bfloat16)
    assert base.data_ptr() % 16 == 0
    even, odd = base[:128000].view(1000, 128), base[1:128001].view(1000, 128)
    apart = base[:136000].view(1000, 136)[:, :128]
    whole = _C.linear_xent_scratch(64, 1000, 128, torch.bfloat16, False)
    assert _C.linear_xent_scratch(64, even, False) == _C.linear_xent_scratch(64, apart, False) == whole
    assert _C.linear_xent_scratch(64, odd, False) == whole + 1024 * 128 * 2
    assert _C.linear_xent_scratch(rows=64, w=odd, gradients=False, piece=256) == whole + 256 * 128 * 2
    assert _C.linear_xent_scratch(64, even) == _C.linear_xent_scratch(64, 1000, 128, torch.bfloat16)
    for bad in (base, base[:1000].view(10, 10, 10), even.t(), even[:0]):
        with pytest.raises(RuntimeError):
            _C.linear_xent_scratch(64, bad)
