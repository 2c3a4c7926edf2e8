"""Register and LDS guards of the chunk attention and the page scores (CPU only: compiles, runs nothing).

A scratch reload in a tile loop waits for every copy in flight, so no basic block of a tile's MFMAs may touch scratch; an
access through a pointer of no known address space (flat) waits for LDS and memory both, so there is none; one
workgroup fills a CU, so its LDS must fit."""
import os
import re
import subprocess

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "ds-flashdmla-moe_amd", "csrc")
HIPCC = "/opt/rocm/bin/hipcc"
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-I" + os.path.join(ROOT, "include"),
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-Wno-unused-function", "--cuda-device-only", "-S"]
VGPR_FORM = ["-mllvm", "-amdgpu-mfma-vgpr-form"]   # as in the Makefile: not for the chunk attention


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc is needed")
@pytest.mark.parametrize("source,flags,kernels,with_tiles", [("dmla_chunk.hip", [], 2, 1), ("dmla_select.hip", VGPR_FORM, 11, 4),
                                                             ("dmla_pages.hip", VGPR_FORM, None, 0)])
def test_tile_loops_are_spill_free_and_fit_a_cu(tmp_path, source, flags, kernels, with_tiles):
    out = tmp_path / "k.s"
    run = subprocess.run([HIPCC] + FLAGS + flags + [os.path.join(CSRC, source), "-o", str(out)], capture_output=True,
                         text=True, timeout=600)
    assert run.returncode == 0, run.stderr[-2000:]
    asm = out.read_text()
    starts = [m.end() for m in re.finditer(r"^_ZN4dmla\S*_kernel\S*:", asm, re.M)]
    assert kernels is None or len(starts) == kernels
    loops = 0
    for start in starts:
        body = asm[start:asm.index(".Lfunc_end", start)]
        assert not re.search(r"^\s+flat_", body, re.M), "flat access"
        tiles = 0
        for block in re.split(r"^(?=\.LBB\d+_\d+:|; %bb\.\d+:)", body, flags=re.M):
            if len(re.findall(r"^\s+v_mfma", block, re.M)) >= 8:   # (few rows: 8 or 9 for each barrier)
                tiles += 1
                assert not re.search(r"^\s+scratch_", block, re.M), "scratch access in a tile iteration"
        loops += tiles > 0
    assert loops == with_tiles
    lds = [int(x) for x in re.findall(r"; LDSByteSize: (\d+)", asm)]
    assert len(lds) >= len(starts) and max(lds) <= 160 * 1024
