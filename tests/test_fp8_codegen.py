"""Code-generation guard for the 8-bit GEMM whose tiles go straight into LDS
(CPU only: hipcc cross-compiles gfx950 assembly here).  Its loads are inline asm
that the compiler does not count: an offset register must stay as it is until
its load is done, nothing may spill, and the K loop waits once a block."""
from __future__ import annotations

import re
import shutil
import subprocess
from pathlib import Path

import pytest

from test_gemm_codegen import REPO, _vgprs, _written_vgprs, kernel_body

SRC = REPO / "ai-compiler-framework_amd" / "csrc" / "kernels" / "gemm_fp8.hip"


@pytest.fixture(scope="module")
def bodies(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(hipcc).exists():
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("fp8_asm") / "gemm_fp8.s"
    cmd = [hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
           "-packed-fp32-ops", f"-I{REPO / 'include'}", "--cuda-device-only", "-S", str(SRC), "-o", str(out)]
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=900)
    assert r.returncode == 0, r.stdout[-4000:]
    asm = out.read_text()
    names = re.findall(r"^(_Z\S*gemm_fp8_lds_kernel\S*):", asm, re.M)
    return {n: kernel_body(asm, n[n.index("gemm_fp8_lds_kernel"):]) for n in names}


def loop_lines(body):
    """The lines between each backward branch and its target."""
    at = {ln.split(":")[0]: i for i, ln in enumerate(body) if ln.startswith(".LBB")}
    for i, ln in enumerate(body):
        m = re.search(r"s_cbranch_\w+\s+(\.LBB\w+)", ln.split(";")[0])
        if m and at.get(m.group(1), i) < i:
            yield body[at[m.group(1)]:i + 1]


def asm_loads(body):
    """(line, offset VGPR) of the direct-to-LDS loads."""
    out = []
    for i, ln in enumerate(body):
        m = re.search(r"buffer_load_dword(?:x4)?\s+v(\d+),.*\boffen\b.*\blds\b", ln)
        if m:
            out.append((i, int(m.group(1))))
    return out


def test_every_form_is_there(bodies):
    # 4 pairs of types, scales of B by rows or blocks; f32 outputs 3 tiles, 16-bit ones 4
    assert len(bodies) == 4 * 2 * 7


def test_no_spills(bodies):
    for name, body in bodies.items():
        assert not [ln for ln in body if "scratch_" in ln], name


def test_k_loop_waits_once_and_keeps_its_offsets(bodies):
    for name, body in bodies.items():
        loops = [lp for lp in loop_lines(body) if asm_loads(lp) and any("v_mfma" in ln for ln in lp)]
        assert loops, name
        for lp in loops:
            waits = [ln for ln in lp if "s_waitcnt" in ln.split(";")[0] and "vmcnt" in ln]
            assert len(waits) == sum("s_barrier" in ln for ln in lp) > 0, (name, waits)
            regs = {r for _, r in asm_loads(lp)}
            written = set().union(*(_written_vgprs(ln) for ln in lp if "offen" not in ln))
            assert not regs & written, (name, regs & written)


def first_write(body, start, reg):
    """The first line from start on that writes reg before a full wait; backward
    branches are left to the test of the loops."""
    for ln in body[start:]:
        s = ln.split(";")[0]
        if "s_waitcnt" in s and "vmcnt(0)" in s:
            return None
        if "offen" not in s and reg in _written_vgprs(ln):
            return ln
    return None


def test_offsets_are_kept_until_the_loads_are_done(bodies):
    checked = 0
    for name, body in bodies.items():
        for i, reg in asm_loads(body):
            hit = first_write(body, i + 1, reg)
            assert hit is None, f"{name}: v{reg} is written at '{hit.strip()}' before a vmcnt(0) wait"
            checked += 1
    assert checked > 100, checked


def test_the_guard_sees_a_planted_write(bodies):
    name, body = next(iter(bodies.items()))
    i, reg = asm_loads(body)[0]
    assert _vgprs(f"v{reg}") == {reg}
    bad = body[:i + 1] + [f"\tv_mov_b32_e32 v{reg}, 0"] + body[i + 1:]
    assert first_write(bad, i + 1, reg) is not None
