"""Refusals of quant_fp8, gemm_fp8, distill_topk and sample_row, on the host
before any launch (the addresses are never touched), and their names."""
from __future__ import annotations

import ctypes
import struct

import pytest

from aicf_cuda import abi

OK, INV, NOTIMPL = abi.STATUS_OK, abi.STATUS_INVALID_ARGUMENT, abi.STATUS_NOT_IMPLEMENTED
F32, F16, BF16, I32, E4, E5 = (abi.DTYPE_F32, abi.DTYPE_F16, abi.DTYPE_BF16, abi.DTYPE_I32, abi.DTYPE_F8E4M3,
                               abi.DTYPE_F8E5M2)
QUANT, GEMM, DISTILL, SAMPLE = 30, 31, 32, 33
IDS = {QUANT: "quant_fp8_v0", GEMM: "gemm_fp8_mfma_v0", DISTILL: "distill_topk_v0", SAMPLE: "sample_row_v0"}
QFP8, DTOP = (int.from_bytes(t, "little") for t in (b"QFP8", b"DTOP"))


@pytest.fixture(scope="module")
def lib():
    return abi.load()


class At:
    """Descriptors at addresses of their own, 2^40 apart."""

    def __init__(self):
        self.n = 0

    def __call__(self, shape, dtype=F32, stride=None, ptr=None):
        self.n += 1
        return abi.make_desc(self.n << 40 if ptr is None else ptr, dtype, shape, stride)


def refused(lib, kind, ins, outs, schema=0, payload=b""):
    ia, oa = abi.desc_array(ins), abi.desc_array(outs)
    blob, keep = abi.make_blob(schema, payload)
    bp = ctypes.byref(blob) if schema or payload else None
    st = lib.aicf_dispatch_v0(kind, ia, len(ins), oa, len(outs), bp, None)
    by_id = lib.aicf_dispatch_by_id_v0(kind, IDS[kind].encode(), ia, len(ins), oa, len(outs), bp, None)
    assert by_id == INV and st == NOTIMPL, (st, by_id)


def test_names_and_registration(lib):
    for kind, name in ((QUANT, b"quant_fp8"), (GEMM, b"gemm_fp8"), (DISTILL, b"distill_topk"), (SAMPLE, b"sample_row")):
        assert lib.aicf_opkind_name(kind) == name
        assert lib.aicf_registry_count(kind) == 1
        assert lib.aicf_registry_has(kind, IDS[kind].encode()) == 1


def test_quant_refuses(lib):
    d = At()
    x, q, s = d((256, 384), BF16), d((256, 384), E4), d((256, 3))
    qt, st = d((384, 256), E4), d((384, 2))
    r = lambda i, o, **kw: refused(lib, QUANT, i, o, **kw)  # noqa: E731
    r([x], [q])
    r([x, x], [q, s])
    r([x], [q, s, qt])
    r([d((256, 384), I32)], [q, s])
    r([d((256, 384), E4)], [q, s])
    r([x], [d((256, 384), BF16), s])
    r([x], [d((256, 383), E4), s])
    r([x], [q, d((256, 4))])
    r([x], [q, d((255, 3))])
    r([x], [q, d((256, 3), F16)])
    r([x], [q, s, d((384, 256), E5), st])                      # two 8-bit types
    r([x], [q, s, qt, d((3, 2))])                              # by rows and by blocks
    r([x], [q, s, qt, d((384, 3))])
    r([d((256, 384), BF16, (1, 256))], [q, s])                 # columns apart
    r([x], [d((256, 384), E4, (100, 1)), s])                   # rows that meet
    r([x], [q, d((256, 3), F32, (2, 1))])
    r([x], [q, s], schema=QFP8, payload=struct.pack("<i", 2))  # an unknown flag
    r([x], [q, s], schema=QFP8, payload=b"")
    r([d((256, 0), BF16)], [d((256, 0), E4), d((256, 0))])
    r([x], [d((256, 384), E4, None, x.data + 100), s])         # over the input
    r([x], [q, d((256, 3), F32, None, q.data)])
    r([d((4, 4, 4), BF16)], [q, s])


def test_gemm_refuses(lib):
    d = At()
    a, sa, b, sb, bias, c = (d((64, 300), E4), d((64, 3)), d((200, 300), E5), d((2, 3)), d((200,)), d((64, 200), BF16))
    r = lambda i, o: refused(lib, GEMM, i, o)  # noqa: E731
    r([a, sa, b], [c])
    r([a, sa, b, sb, bias, bias], [c])
    r([a, sa, b, sb], [c, c])
    r([d((64, 300), BF16), sa, b, sb], [c])
    r([a, sa, d((200, 299), E5), sb], [c])
    r([a, d((63, 3)), b, sb], [c])
    r([a, d((64, 2)), b, sb], [c])
    r([a, sa, b, d((3, 3))], [c])
    r([a, sa, b, d((2, 3), BF16)], [c])
    r([a, sa, b, sb, d((199,))], [c])
    r([a, sa, b, sb, d((200,), BF16)], [c])
    r([a, sa, b, sb, d((200,), F32, (2,))], [c])
    r([a, sa, b, sb], [d((64, 201), BF16)])
    r([a, sa, b, sb], [d((64, 200), E4)])
    r([a, sa, b, sb], [d((64, 200), BF16, (1, 64))])
    r([d((64, 300), E4, (1, 64)), sa, b, sb], [c])
    r([a, sa, b, sb], [d((64, 200), BF16, None, a.data)])
    r([d((64, 0), E4), d((64, 0)), d((200, 0), E4), d((2, 0))], [c])


def test_distill_refuses(lib):
    d = At()
    z, t, ids, lab, w = d((8, 1000), BF16), d((8, 20)), d((8, 20), I32), d((8,), I32), d((8,))
    loss, dz, rl, sc = d((1,)), d((8, 1000), BF16), d((8,)), d((8, 16, 4))
    pay = struct.pack("<ff", 1.0, 0.0)

    def r(i, o, p=pay):
        refused(lib, DISTILL, i, o, DTOP, p)

    r([z, t], [loss, dz, rl])
    r([z, t, ids], [loss])
    r([z, t, ids, w, lab], [loss, dz, rl])
    r([z, t, ids, lab, w, w], [loss, dz, rl])
    r([z, t, ids], [loss, dz, rl, sc, sc])
    r([z, t, ids], [loss, d((8, 1000)), rl])
    r([z, t, ids], [loss, d((8, 999), BF16), rl])
    r([z, t, ids], [loss, dz, d((7,))])
    r([z, t, ids], [d((2,)), dz, rl])
    r([z, t, ids], [loss, dz, rl, d((8, 1, 4))])
    r([z, t, ids], [loss, dz, rl, d((8, 16, 3))])
    r([z, t, d((8, 20))], [loss, dz, rl])
    r([z, t, d((8, 19), I32)], [loss, dz, rl])
    r([z, d((7, 20)), d((7, 20), I32)], [loss, dz, rl])
    r([z, d((8, 1025)), d((8, 1025), I32)], [loss, dz, rl])
    r([z, d((8, 0)), d((8, 0), I32)], [loss, dz, rl])
    r([z, t, ids, d((7,), I32)], [loss, dz, rl])
    r([d((8, 1000), I32), t, ids], [loss, dz, rl])
    r([d((0, 1000), BF16), d((0, 20)), d((0, 20), I32)], [loss, d((0, 1000), BF16), d((0,))])
    r([z, t, ids], [loss, d((8, 1000), BF16, None, z.data + 2), rl])   # over the logits, but not on them
    r([z, t, ids], [loss, d((8, 1000), BF16, (1008, 1), z.data), rl])
    r([z, t, ids, w], [loss, dz, d((8,), F32, None, w.data)])
    for p in (struct.pack("<ff", 0.0, 0.0), struct.pack("<ff", -1.0, 0.0), struct.pack("<ff", float("nan"), 0.0),
              struct.pack("<ff", float("inf"), 0.0), struct.pack("<ff", 1.0, 1.5), struct.pack("<ff", 1.0, -0.1),
              struct.pack("<ff", 1.0, float("nan")), struct.pack("<f", 1.0)):
        r([z, t, ids], [loss, dz, rl], p)


def test_sample_refuses(lib):
    d = At()
    z, u, temp, k, p, m = d((8, 1000), F16), d((8,)), d((8,)), d((8,), I32), d((8,)), d((8,))
    tok, lp, sc = d((8,), I32), d((8,)), d((8, 8192), I32)
    r = lambda i, o: refused(lib, SAMPLE, i, o)  # noqa: E731
    good = [z, u, temp, k, p, m]
    r(good[:5], [tok])
    r(good, [])
    r(good, [tok, lp, sc, sc])
    r(good, [d((8,))])
    r(good, [d((7,), I32)])
    r(good, [tok, d((8,), I32)])
    r(good, [tok, lp, d((8, 8191), I32)])
    r(good, [tok, lp, d((8, 8192))])
    r([d((8, 1000), I32)] + good[1:], [tok])
    r([d((8, 1000), E4)] + good[1:], [tok])
    r([d((8, 0), F16)] + good[1:], [tok])
    r([d((8, (1 << 24) + 1), F16)] + good[1:], [tok])
    r([z, d((9,))] + good[2:], [tok])
    r([z, u, temp, d((8,)), p, m], [tok])
    r([z, u, temp, k, p, d((8,), F32, (2,))], [tok])
    r([d((8, 1000), F16, (1, 8))] + good[1:], [tok])
    r(good, [tok, d((8,), F32, None, u.data)])


def test_calls_without_memory_and_empty_calls(lib):
    """A descriptor without memory is refused at the launch, in the library;
    a call that has nothing to do is done."""
    d = At()

    def call(kind, ins, outs, schema=0, payload=b""):
        ia, oa = abi.desc_array(ins), abi.desc_array(outs)
        blob, keep = abi.make_blob(schema, payload)
        return lib.aicf_dispatch_v0(kind, ia, len(ins), oa, len(outs), ctypes.byref(blob), None)

    none = lambda shape, dt=F32: abi.make_desc(None, dt, shape)  # noqa: E731
    assert call(QUANT, [none((4, 128), F32)], [d((4, 128), E4), d((4, 1))]) == INV
    assert call(GEMM, [d((4, 128), E4), d((4, 1)), d((8, 128), E4), d((8, 1))], [none((4, 8))]) == INV
    assert call(DISTILL, [d((4, 100)), d((4, 5)), none((4, 5), I32)], [d((1,)), d((4, 100)), d((4,))], DTOP,
                struct.pack("<ff", 1.0, 0.0)) == INV
    assert call(SAMPLE, [d((4, 100)), d((4,)), d((4,)), d((4,), I32), d((4,)), none((4,))], [d((4,), I32)]) == INV
    assert call(QUANT, [none((0, 128))], [none((0, 128), E4), none((0, 1))]) == OK
    assert call(GEMM, [none((0, 128), E4), none((0, 1)), d((8, 128), E4), d((8, 1))], [none((0, 8))]) == OK
    assert call(SAMPLE, [none((0, 100)), none((0,)), none((0,)), none((0,), I32), none((0,)), none((0,))],
                [none((0,), I32)]) == OK


def test_executor_knows_the_ops():
    from aicf_hip.executor import OPNAME_TO_KIND, pack_attrs

    assert [OPNAME_TO_KIND[n] for n in ("quant_fp8", "gemm_fp8", "distill_topk", "sample_row")] == [30, 31, 32, 33]
    assert pack_attrs("quant_fp8", {"pow2": True}) == (QFP8, struct.pack("<i", 1))
    assert pack_attrs("distill_topk", {"temperature": 2.0, "label_weight": 0.5}) == (DTOP, struct.pack("<ff", 2.0, 0.5))
    assert pack_attrs("gemm_fp8", {}) == (0, b"") and pack_attrs("sample_row", {}) == (0, b"")
