"""AdamW with the clip factor over more elements than one launch has work-items:
at an odd element (a lane each), in place."""
from __future__ import annotations

import struct

import pytest
import torch

pytestmark = pytest.mark.gpu
ADAM = int.from_bytes(b"ADAM", "little")
HP = struct.pack("<fffff", 1e-2, 0.9, 0.999, 1e-8, 0.1)


def test_more_than_32_bits_of_elements(C, dev):
    n = 2 ** 32 + 2 ** 20 + 5
    if torch.cuda.mem_get_info()[0] < 80 * 2 ** 30:
        pytest.skip("needs 80 GiB")
    gen = torch.Generator(device=dev).manual_seed(1)
    # a pattern of 1021 values that repeats (n is far from a multiple of it)
    pat = [torch.rand(1021, device=dev, generator=gen) + 0.5 for _ in range(4)]
    g_pat = pat[3].to(torch.bfloat16)
    reps = -(-n // 1021)

    def fill(p):
        t = torch.empty(1 + reps * 1021, device=dev, dtype=p.dtype)
        t[1:].view(reps, 1021)[:] = p
        return t[1:1 + n]

    p, m, v = (fill(t) for t in pat[:3])
    g = fill(g_pat)
    step, norm = torch.tensor(3, device=dev, dtype=torch.int32), torch.tensor([4.0, 0.25], device=dev)
    assert p.data_ptr() % 16 == 4
    C.op_call(C.OpKind.AdamStep, [p, g, m, v, step, norm], [p, m, v], ADAM, HP)
    own = [t.clone() for t in pat[:3]]
    C.op_call(C.OpKind.AdamStep, [own[0], g_pat, own[1], own[2], step, norm], own, ADAM, HP)
    for got, want, old in zip((p, m, v), own, pat):
        assert not torch.equal(want, old)
        rows = got[:n // 1021 * 1021].view(-1, 1021)
        assert all(bool((part == want).all()) for part in rows.split(1 << 19))
        assert torch.equal(got[n // 1021 * 1021:], want[:n % 1021])
