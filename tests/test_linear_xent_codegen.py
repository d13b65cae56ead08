"""Code generation of the linear cross-entropy's products (CPU only: hipcc
cross-compiles gfx950 assembly here): they are the tiled GEMM with epilogues of
their own, and keep what its tests ask of it."""
from __future__ import annotations

import re
import shutil
import subprocess

import pytest

from test_gemm_codegen import (REPO, _first_write_before_drain, asm_lds_loads, asm_load_sgpr_hazards, k_loop,
                               kernel_body)

SRC = REPO / "ai-compiler-framework_amd" / "csrc" / "kernels" / "linear_xent.hip"


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    out = tmp_path_factory.mktemp("lx_asm") / "linear_xent.s"
    cmd = [hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
           "-packed-fp32-ops", f"-I{REPO / 'include'}", "--cuda-device-only", "-S", str(SRC), "-o", str(out)]
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=600)
    assert r.returncode == 0, r.stdout[-4000:]
    return out.read_text()


def test_no_scratch_memory(asm):
    found = 0
    for m in re.finditer(r"\.amdhsa_kernel (\S+)\n(.*?)\.end_amdhsa_kernel", asm, re.S):
        found += "gemm_nt_kernel" in m.group(1)
        seg = re.search(r"\.amdhsa_private_segment_fixed_size\s+(\d+)", m.group(2))
        assert seg and int(seg.group(1)) == 0, (m.group(1), seg and seg.group(1))
    assert found > 30, found


def test_large_tiles_wait_for_their_loads_once_per_k_step(asm):
    names = re.findall(r"^_Z\S*(gemm_nt_kernelILi[12]ELi\dELi\dELi256ELi256E\S*):", asm, re.M)
    assert len(names) >= 10, names
    for name in names:
        loop = k_loop(kernel_body(asm, name))
        waits = [ln.strip() for ln in loop if "s_waitcnt" in ln and "vmcnt" in ln]
        assert len(waits) == 1, (name, waits)


def test_asm_loads(asm):
    """Offsets unwritten until the loads are done; 5 wait states after a scalar that the VALU wrote."""
    checked = 0
    for name in re.findall(r"^(_Z\S*gemm_nt_kernel\S*):", asm, re.M):
        body = kernel_body(asm, name[name.index("gemm_nt_kernel"):])
        labels = {ln.split(":")[0]: i for i, ln in enumerate(body) if ln.startswith(".LBB")}
        for start, reg in asm_lds_loads(body):
            assert _first_write_before_drain(body, start, reg, labels) is None, name
            checked += 1
        assert not asm_load_sgpr_hazards(body), name
    assert checked > 100, checked
