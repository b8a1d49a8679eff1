"""What the compiler reports for the kernels of the 8-bit caches and the shared prefix (no GPU needed): registers spilled to
scratch memory cost a launch its set-up, and a loop its time."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "topk_attn_amd", "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


@pytest.mark.parametrize("source,extra", [("kv_quant.hip", []), ("kv_attend.hip", ["-mllvm", "-amdgpu-mfma-vgpr-form=1"])])
def test_scratch_memory(source, extra):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    cmd = [HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wno-unused-function", "-Xclang", "-target-feature", "-Xclang",
           "-packed-fp32-ops", "--cuda-device-only", "-Rpass-analysis=kernel-resource-usage", "-c", "-o", os.devnull, source] + extra
    done = subprocess.run(cmd, cwd=CSRC, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-2000:]
    found = re.findall(r"Function Name: (\S+).*?ScratchSize \[bytes/lane\]: (\d+)", done.stderr, flags=re.S)
    assert len(found) >= 12
    for name, scratch in found:
        assert int(scratch) == 0, (name, scratch)
