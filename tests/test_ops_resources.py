"""Build-time guard (no GPU): the product kernels of the gated block and the distillation kernels need no scratch memory.  Their tiles
and rows live in registers; a spilled one is written to memory and read back in the middle of the loop that the registers are for."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "graphslim_amd", "csrc")


@pytest.mark.parametrize("src,must,least", [
    ("gs_gated.hip", r"gs_gated_(gemm|pair|rows)_kernel", 20),
    ("gs_distill.hip", r"gs_distill_(regs|row)_kernel", 30),
    ("gs_embedding.hip", r"gs_embedding_", 30)])
def test_no_scratch(src, must, least, tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    out = subprocess.run([hipcc, "-O3", "-fPIC", "--offload-arch=gfx950", "-std=c++17", "-Wno-unused-function", "-Xclang", "-target-feature",
                          "-Xclang", "-packed-fp32-ops", "--cuda-device-only", "-c", os.path.join(CSRC, src), "-o", str(tmp_path / "o.o"),
                          "-Rpass-analysis=kernel-resource-usage"], capture_output=True, text=True, cwd=CSRC)
    assert out.returncode == 0, out.stderr[-2000:]
    names = re.findall(r"Function Name: (\S+)", out.stderr)
    scratch = [int(v) for v in re.findall(r"ScratchSize \[bytes/lane\]: (\d+)", out.stderr)]
    assert len(names) == len(scratch)
    seen = [(n, sc) for n, sc in zip(names, scratch) if re.search(must, n)]
    assert len(seen) >= least, (len(seen), names)
    for n, sc in seen:
        assert sc == 0, f"{n} needs {sc} bytes of scratch per lane"
