"""The 8-bit GEMM's inline-asm loads straight into LDS, of 16 and of 4 bytes a
lane: 5 wait states after every VALU write of a scalar that one reads (CPU only:
hipcc cross-compiles gfx950 assembly here)."""
from __future__ import annotations

import re

from test_fp8_codegen import asm_loads, bodies  # noqa: F401  (the compiled kernels, once)
from test_gemm_codegen import asm_load_sgpr_hazards


def test_loads_wait_for_scalars_that_the_valu_wrote(bodies):  # noqa: F811
    wide = narrow = 0
    for name, body in bodies.items():
        hazards = asm_load_sgpr_hazards(body)
        assert not hazards, (name, hazards[:4])
        starts = sum("ASMSTART" in ln and re.search(r"buffer_load_dword.*\blds\b", "".join(body[i + 1:i + 4])) is not None
                     for i, ln in enumerate(body))
        loads = asm_loads(body)
        assert starts == len(loads) > 0, name  # each of them is seen by the check
        narrow += sum("buffer_load_dword " in body[i].replace("\t", " ") for i, _ in loads)
        wide += sum("buffer_load_dwordx4 " in body[i].replace("\t", " ") for i, _ in loads)
    assert wide > 500 and narrow > 100, (wide, narrow)


def test_the_check_sees_a_planted_write_before_a_load_of_4_bytes(bodies):  # noqa: F811
    name, body = next(iter(bodies.items()))
    at = next(i for i, _ in asm_loads(body) if "buffer_load_dword " in body[i].replace("\t", " "))
    start = max(i for i in range(at) if "ASMSTART" in body[i])
    soff = body[at].split(";")[0].split(",")[2].split()[0]
    bad = body[:start] + [f"\tv_readfirstlane_b32 {soff}, v0"] + body[start:]
    pad = any("s_nop 4" in ln for ln in body[start:at])
    assert pad or asm_load_sgpr_hazards(bad), name
    loop = body[start:at + 2]
    loop = [ln.replace("s_nop 4", "s_nop 0") for ln in loop]
    assert asm_load_sgpr_hazards([f"\tv_readfirstlane_b32 {soff}, v0"] + loop)
