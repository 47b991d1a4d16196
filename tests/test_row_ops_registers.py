"""The row operators' kernels keep everything in registers: none spills and none has scratch
memory. The policy loss holds a row of logits in a workgroup's registers, the head norm four rows
a lane: what does not fit goes to memory, with the right results and several times the time."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = "/opt/rocm/bin/hipcc"


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
@pytest.mark.parametrize("source, kernels", [("qknorm", 60), ("router", 48), ("logprob", 55)])
def test_row_kernels_use_no_scratch(tmp_path, source, kernels):
    asm = tmp_path / "kernels.s"
    cmd = [HIPCC, "-O3", "-std=c++17", "--offload-arch=gfx950", "-fPIC", "-w", "-mllvm",
           "-pragma-unroll-threshold=1000000", "-Xclang", "-target-feature", "-Xclang",
           "-packed-fp32-ops", "-I" + os.path.join(ROOT, "include"), "--cuda-device-only", "-S",
           os.path.join(ROOT, "dtensor-muon_amd", "csrc", source + ".hip"), "-o", str(asm)]
    subprocess.run(cmd, check=True, capture_output=True, timeout=900)
    text = asm.read_text()
    found = re.findall(r"\.private_segment_fixed_size:\s+(\d+).*?\.symbol:\s+(\S+)\.kd.*?"
                       r"\.vgpr_spill_count:\s+(\d+)", text, re.S)
    assert len(found) >= kernels
    assert not [f for f in found if int(f[0]) or int(f[2])]
    assert not re.search(r"v_pk_(add|mul|fma)_f32", text)
