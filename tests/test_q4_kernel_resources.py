"""Register and LDS guards of the 4-bit decode and the accounts (CPU only: compiles, runs nothing).

A scratch reload in a tile loop waits for every copy in flight, so no basic block that issues MFMAs may touch scratch;
one workgroup fills a CU, so its LDS must fit."""
import os
import re
import subprocess

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "ds-flashdmla-moe_amd", "csrc")
HIPCC = "/opt/rocm/bin/hipcc"
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-I" + os.path.join(ROOT, "include"),
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-Wno-unused-function", "--cuda-device-only", "-S"]
VGPR_FORM = ["-mllvm", "-amdgpu-mfma-vgpr-form"]   # as in the Makefile: not for the decodes


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc is needed")
@pytest.mark.parametrize("source,flags,kernels", [("dmla_q4_decode.hip", [], 1), ("dmla_q4_wide.hip", [], 1),
                                                  ("dmla_mass.hip", VGPR_FORM, 3)])
def test_tile_loops_are_spill_free_and_fit_a_cu(tmp_path, source, flags, kernels):
    out = tmp_path / "k.s"
    run = subprocess.run([HIPCC] + FLAGS + flags + [os.path.join(CSRC, source), "-o", str(out)], capture_output=True,
                         text=True, timeout=600)
    assert run.returncode == 0, run.stderr[-2000:]
    asm = out.read_text()
    starts = [m.end() for m in re.finditer(r"^_ZN4dmla\S*_kernel\S*:", asm, re.M)]
    assert len(starts) == kernels
    for start in starts:
        body = asm[start:asm.index(".Lfunc_end", start)]
        tiles = 0
        for block in re.split(r"^(?=\.LBB\d+_\d+:|; %bb\.\d+:)", body, flags=re.M):
            if len(re.findall(r"^\s+v_mfma", block, re.M)) >= 15:
                tiles += 1
                assert not re.search(r"^\s+scratch_", block, re.M), "scratch access in a tile iteration"
        assert tiles >= 1
    lds = [int(x) for x in re.findall(r"; LDSByteSize: (\d+)", asm)]
    assert len(lds) == kernels and max(lds) <= 160 * 1024
