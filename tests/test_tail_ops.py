"""Refusals of linear_xent, grad_norm and AdamW with the clip factor, on the host
before any launch (the addresses are never touched), their names, and the
scratch that linear_xent asks for."""
from __future__ import annotations

import ctypes
import struct

import pytest

from aicf_cuda import abi
from aicf_hip.executor import OPNAME_TO_KIND, pack_attrs
from test_head_ops import BF16, F16, F32, I32, At

INV, NOTIMPL = abi.STATUS_INVALID_ARGUMENT, abi.STATUS_NOT_IMPLEMENTED
ADAM_STEP, XENT, NORM = 10, 34, 35
IDS = {ADAM_STEP: "adamw_step_clip_v0", XENT: "linear_xent_v0", NORM: "grad_norm_v0"}
GNRM, ADAM = (int.from_bytes(t, "little") for t in (b"GNRM", b"ADAM"))


@pytest.fixture(scope="module")
def lib():
    return abi.load()


def refused(lib, kind, ins, outs, schema=0, payload=b""):
    ia, oa = abi.desc_array(ins), abi.desc_array(outs)
    blob, keep = abi.make_blob(schema, payload)
    bp = ctypes.byref(blob) if schema or payload else None
    st = lib.aicf_dispatch_v0(kind, ia, len(ins), oa, len(outs), bp, None)
    by_id = lib.aicf_dispatch_by_id_v0(kind, IDS[kind].encode(), ia, len(ins), oa, len(outs), bp, None)
    assert by_id == INV and st == NOTIMPL, (st, by_id)


def taken(lib, kind, ins, outs, schema=0, payload=b""):
    """The call is supported: with an output without memory it is the launch that turns it down, before any HIP call."""
    ia, oa = abi.desc_array(ins), abi.desc_array(outs)
    blob, keep = abi.make_blob(schema, payload)
    st = lib.aicf_dispatch_v0(kind, ia, len(ins), oa, len(outs), ctypes.byref(blob), None)
    assert st == INV, st


def test_names(lib):
    assert lib.aicf_opkind_name(XENT) == b"linear_xent" and lib.aicf_opkind_name(NORM) == b"grad_norm"
    for kind, name in IDS.items():
        assert lib.aicf_registry_has(kind, name.encode()) == 1
    assert [OPNAME_TO_KIND[n] for n in ("linear_xent", "grad_norm")] == [XENT, NORM]
    assert pack_attrs("grad_norm", {"max_norm": 0.5}) == (GNRM, struct.pack("<f", 0.5))


def scratch(lib, r, v, d, dt=BF16, grad=1, piece=0):
    return lib.aicf_linear_xent_scratch(r, v, d, dt, grad, piece)


def test_scratch(lib):
    whole = scratch(lib, 512, 32000, 1024)
    assert whole >= 512 * 32000 * 2
    half = scratch(lib, 512, 32000, 1024, piece=16000)
    assert half < whole and scratch(lib, 512, 32000, 1024, piece=15873) == half  # rounded up to 256 classes
    assert whole - scratch(lib, 512, 32000, 1024, piece=256) == 512 * (32000 - 256) * 2
    assert scratch(lib, 512, 32000, 1024, grad=0) < scratch(lib, 512, 32000, 1024, piece=256)
    assert scratch(lib, 512, 32000, 1024, piece=10 ** 9) == whole
    # rows of W that tiles cannot read in place are copied, a piece at a time
    assert scratch(lib, 512, 32000, 1001, grad=0, piece=256) - scratch(lib, 512, 32000, 1024, grad=0) == 256 * 1024 * 2
    assert scratch(lib, 512, 32000, 1000, grad=0, piece=256) == scratch(lib, 512, 32000, 1024, grad=0)  # (1000: in place)
    for bad in ((-1, 10, 10), (1, 0, 10), (1, 10, 0), (1, 2 ** 28 + 1, 64), (2 ** 31, 10, 10), (1, 10, 2 ** 23),
                (2 ** 20, 1000, 1024)):
        assert scratch(lib, *bad) == -1
    assert scratch(lib, 2 ** 20, 1000, 1024, grad=0) > 0  # (without gradients: no limit of 2^31 bytes)
    assert scratch(lib, 10, 10, 10, I32) == -1 and scratch(lib, 10, 10, 10, 99) == -1


def test_linear_xent_refuses(lib):
    d = At()
    r, v, dim = 64, 1000, 128
    x, w, lab, rw = d((r, dim), BF16), d((v, dim), BF16), d((r,), I32), d((r,))
    loss, dx, dw, rl = d((1,)), d((r, dim), BF16), d((v, dim), BF16), d((r,))
    sc = d((scratch(lib, r, v, dim) // 4,))
    no = lambda i, o: refused(lib, XENT, i, o)  # noqa: E731
    missing = abi.make_desc(None, F32, (r,))
    for ins in ([x, w, lab], [x, w, lab, rw]):
        for outs in ([loss, missing, sc], [loss, dx, missing, sc], [loss, dx, dw, missing, sc]):
            taken(lib, XENT, ins, outs)
    taken(lib, XENT, [x, w, lab], [loss, dx, d((v, dim), F32), missing, sc])
    no([x, w], [loss, rl, sc])
    no([x, w, lab, rw, rw], [loss, rl, sc])
    no([x, w, lab], [loss, rl])
    no([x, w, lab], [loss, dx, dw, dw, rl, sc])
    no([x, d((v, dim), F16), lab], [loss, rl, sc])
    no([d((r, dim), I32), d((v, dim), I32), lab], [loss, rl, sc])
    no([x, d((v, dim + 1), BF16), lab], [loss, rl, sc])
    no([x, d((0, dim), BF16), lab], [loss, rl, sc])
    no([d((r, 0), BF16), d((v, 0), BF16), lab], [loss, rl, sc])
    no([d((r, dim, 1), BF16), w, lab], [loss, rl, sc])
    no([d((r, dim), BF16, (1, r)), w, lab], [loss, rl, sc])
    no([x, w, d((r,), F32)], [loss, rl, sc])
    no([x, w, d((r - 1,), I32)], [loss, rl, sc])
    no([x, w, d((r,), I32, (2,))], [loss, rl, sc])
    no([x, w, lab, d((r,), BF16)], [loss, rl, sc])
    no([x, w, lab, d((r + 1,))], [loss, rl, sc])
    no([x, w, lab], [d((2,)), rl, sc])
    no([x, w, lab], [d((1,), BF16), rl, sc])
    no([x, w, lab], [loss, d((r, 1)), sc])
    no([x, w, lab], [loss, d((r, dim), F32), rl, sc])       # dX in another type
    no([x, w, lab], [loss, d((r, dim + 1), BF16), rl, sc])
    no([x, w, lab], [loss, dx, d((v, dim), F16), rl, sc])
    no([x, w, lab], [loss, dx, d((v, dim), BF16, (dim - 1, 1)), rl, sc])  # rows that meet
    no([x, w, lab], [loss, d((r, dim), BF16, (0, 1)), rl, sc])
    no([x, w, lab], [loss, rl, d((10,))])                   # scratch too small
    no([x, w, lab], [loss, dx, rl, d((scratch(lib, r, v, dim, piece=256) // 4 - 64,))])
    no([x, w, lab], [loss, rl, d((1 << 24,), BF16)])
    no([x, w, lab], [loss, rl, d((1 << 12, 1 << 12))])
    no([x, w, lab], [loss, rl, d((1 << 24,), F32, (2,))])
    no([x, w, lab], [loss, d((r, dim), BF16, None, x.data), rl, sc])      # over an input
    no([x, w, lab], [loss, dx, d((v, dim), BF16, None, w.data), rl, sc])
    no([x, w, lab], [loss, dx, rl, d((1 << 24,), F32, None, dx.data + 64)])
    no([x, w, lab], [loss, d((r,), F32, None, loss.data), sc])
    # W at a byte that no 16-byte load takes: a copy of a piece's rows has to fit too
    odd = d((v, dim), BF16, None, (99 << 40) + 2)
    no([x, odd, lab], [loss, rl, d((scratch(lib, r, v, dim, grad=0) // 4,))])
    taken(lib, XENT, [x, odd, lab], [loss, missing, d((scratch(lib, r, v, dim, grad=0) // 4 + 256 * dim // 2 + 64,))])
    # more rows than 31 bits count bytes of, with gradients
    big = 1 << 20
    bx, bl, brw = d((big, 1024), BF16), d((big,), I32), d((big,))
    no([bx, d((v, 1024), BF16), bl], [loss, d((big, 1024), BF16), brw, d((1 << 36,))])


def test_grad_norm_refuses(lib):
    d = At()
    g, h = d((100, 7)), d((5,), BF16)
    norm, sc = d((2,)), d((2048,))
    pay = struct.pack("<f", 1.0)
    no = lambda i, o, schema=GNRM, payload=pay: refused(lib, NORM, i, o, schema, payload)  # noqa: E731
    missing = abi.make_desc(None, F32, (2,))
    taken(lib, NORM, [g, h], [missing, sc], GNRM, pay)
    taken(lib, NORM, [g, h], [missing, sc, g, d((5,), BF16)], GNRM, pay)
    taken(lib, NORM, [g, g], [missing, sc], GNRM, pay)  # twice the same: counted twice
    no([], [norm, sc])
    no([g], [norm])
    no([g, h], [norm, sc, g])
    no([g], [norm, sc, g, h])
    no([g], [norm, sc], GNRM, struct.pack("<f", -1.0))
    no([g], [norm, sc], GNRM, struct.pack("<f", float("nan")))
    no([g], [norm, sc], GNRM, b"")
    no([g], [norm, sc], GNRM, pay + pay)
    no([g], [norm, sc], ADAM, pay)
    no([d((4,), I32)], [norm, sc])
    no([d((4, 4), F32, (8, 1))], [norm, sc])
    no([d((4, 4), F32, (1, 4))], [norm, sc])
    no([g], [d((1,)), sc])
    no([g], [d((2,), BF16), sc])
    no([g], [norm, d((2047,))])
    no([g] * 97, [norm, d((4095,))])
    no([g], [norm, d((4096,), F32, (2,))])
    no([g], [norm, d((2048,), F32, None, (98 << 40) + 4)])
    no([g], [norm, d((2048,), BF16)])
    no([g], [norm, sc, d((100, 7), BF16)])
    no([g], [norm, sc, d((7, 100))])
    no([g], [norm, sc, d((100, 7), F32, None, g.data + 4)])   # over itself, but not the same
    no([g, g], [norm, sc, g, g])                              # clipped twice
    no([g, h], [norm, sc, g, d((5,), BF16, None, g.data)])
    no([g], [d((2,), F32, None, g.data), sc])
    no([g], [norm, d((2048,), F32, None, g.data)])
    no([g], [norm, sc, d((100, 7), F32, None, sc.data)])
    no([d((1 << 30, 1 << 30))], [norm, sc])
    no([d((1 << 62, 1 << 62))], [norm, sc])
    no([d((1 << 41,)), d((1 << 41,)), d((1,))], [norm, sc])


def test_adamw_with_the_factor_refuses(lib):
    d = At()
    s = (64, 33)
    p, g, m, v, step, norm = d(s), d(s, BF16), d(s), d(s), d((), I32), d((2,))
    outs = [p, m, v]
    pay = struct.pack("<fffff", 1e-3, 0.9, 0.999, 1e-8, 0.0)
    no = lambda i, o: refused(lib, ADAM_STEP, i, o, ADAM, pay)  # noqa: E731
    missing = abi.make_desc(None, F32, s)
    taken(lib, ADAM_STEP, [p, g, m, v, step, norm], [missing, m, v], ADAM, pay)
    taken(lib, ADAM_STEP, [p, d(s), m, v, step, norm], [missing, d(s), d(s), d(s, BF16)], ADAM, pay)
    no([p, g, m, v, step], outs)                       # the variant without the factor takes f32 gradients only
    no([p, g, m, v, step, d((1,))], outs)
    no([p, g, m, v, step, d((2,), BF16)], outs)
    no([p, g, m, v, step, norm, norm], outs)
    no([p, g, m, v, d((2,), I32), norm], outs)
    no([p, d(s, I32), m, v, step, norm], outs)
    no([p, d((33, 64), BF16), m, v, step, norm], outs)
    no([p, d(s, BF16, (1, 64)), m, v, step, norm], outs)
    no([d(s, BF16), g, m, v, step, norm], outs)
    no([p, g, m, d(s, BF16), step, norm], outs)
    no([p, g, m, v, step, norm], [p, m])
    no([p, g, m, v, step, norm], [p, v, m])            # exchanged
    no([p, g, m, v, step, norm], [p, m, m])
    no([p, g, m, v, step, norm], [p, m, v, d(s)])
    no([p, g, m, v, step, norm], [p, m, v, d(s, BF16, None, g.data)])
    no([p, g, m, v, step, norm], [d(s, F32, None, p.data + 4), m, v])
    no([p, g, m, v, step, d((2,), F32, None, p.data)], outs)
