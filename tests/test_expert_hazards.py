"""The experts' product kernels issue matrix products and panel loads from inline asm, which the compiler's
hazard recognizer does not look into. This compiles expert_gemm.hip for gfx950 and scans every kernel
with them, whole (mfma_hazards.py for what products read and write, load_hazards.py for scalar registers
that vector instructions wrote and loads read), and looks at what the kernels keep in memory: nothing in
their loops."""
import os
import re
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
HIPCC = "/opt/rocm/bin/hipcc"
sys.path.insert(0, HERE)
import load_hazards  # noqa: E402
import mfma_hazards  # noqa: E402

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")


def compiled(tmp_path, source):
    asm = tmp_path / (source + ".s")
    cmd = [HIPCC, "-O3", "-std=c++17", "--offload-arch=gfx950", "-fPIC", "-w", "-mllvm",
           "-pragma-unroll-threshold=1000000", "-Xclang", "-target-feature", "-Xclang",
           "-packed-fp32-ops", "-I" + os.path.join(ROOT, "include"), "--cuda-device-only", "-S",
           os.path.join(ROOT, "dtensor-muon_amd", "csrc", source + ".hip"), "-o", str(asm)]
    subprocess.run(cmd, check=True, capture_output=True, timeout=900)
    return asm


def loop_of(lines, what, least):
    """The shortest loop with so many of `what`: from a label to a branch back to it."""
    labels, found = {}, []
    for at, line in enumerate(lines):
        label = re.match(r"(\.LBB\w+):", line)
        if label:
            labels[label.group(1)] = at
        back = re.search(r"s_c?branch\S*\s+(\.LBB\w+)", line)
        if back and back.group(1) in labels:
            body = lines[labels[back.group(1)]:at]
            if sum(what in x for x in body) >= least:
                found.append(body)
    return min(found, key=len)


def test_product_kernels(tmp_path, monkeypatch):
    # 8 passes, as the bf16 product of this shape
    monkeypatch.setitem(mfma_hazards.MFMA_WAIT, "v_mfma_f32_16x16x32_f16", 11)
    asm = compiled(tmp_path, "expert_gemm")
    found = [(n, lines) for n, lines in load_hazards.kernels(asm) if "expert_gemm_pipe" in n]
    assert len(found) == 6  # three forms, two types
    for name, lines in found:
        assert sum("v_mfma" in x for x in lines) >= 256 and sum(" lds" in x for x in lines) >= 64, name
        assert not mfma_hazards.scan(lines), name
        assert not load_hazards.scan(lines), name
        inner = loop_of(lines, "v_mfma", 256)
        assert sum("v_mfma" in x for x in inner) == 256, name
        assert not [x for x in inner if "scratch_" in x or "v_accvgpr" in x], name
    assert not re.search(r"v_pk_(add|mul|fma)_f32", asm.read_text())


@pytest.mark.parametrize("source, kernels", [("expert_gemm", 22), ("experts", 17), ("adamw", 22)])
def test_other_kernels_use_no_scratch(tmp_path, source, kernels):
    text = compiled(tmp_path, source).read_text()
    found = re.findall(r"\.private_segment_fixed_size:\s+(\d+).*?\.symbol:\s+(\S+)\.kd.*?"
                       r"\.vgpr_spill_count:\s+(\d+)", text, re.S)
    assert len(found) >= kernels
    assert not [f for f in found if (int(f[0]) or int(f[2])) and "expert_gemm_pipe" not in f[1]]
    assert not re.search(r"v_pk_(add|mul|fma)_f32", text)


_READ = "v_readfirstlane_b32 s8, v1"
_LOAD = "buffer_load_dwordx4 v2, s[8:11], s4 offen lds"


@pytest.mark.parametrize("name, code, hazards", [
    ("straight line", [_READ, _LOAD], 1),
    ("the offset", ["v_readlane_b32 s4, v1, 0", _LOAD], 1),
    ("enough instructions", [_READ] + ["s_mov_b32 s20, 0"] * 5 + [_LOAD], 0),
    ("one too few", [_READ] + ["s_mov_b32 s20, 0"] * 4 + [_LOAD], 1),
    ("enough wait states", [_READ, "s_nop 4", _LOAD], 0),
    ("other registers", ["v_readfirstlane_b32 s12, v1", _LOAD], 0),
    ("scalar writes", ["s_mov_b32 s8, s12", _LOAD], 0),
    ("through a label", [_READ, ".LBB0_1:", _LOAD], 1),
    ("by a branch", [_READ, "s_branch .LBB0_2", ".LBB0_1:", "s_endpgm", ".LBB0_2:", _LOAD], 1),
    ("not by falling through", [_READ, "s_branch .LBB0_2", ".LBB0_1:", _LOAD, ".LBB0_2:", "s_endpgm"], 0),
    ("around a loop", [".LBB0_1:", _LOAD] + ["s_nop 7"] + [_READ, "s_cbranch_scc1 .LBB0_1"], 1),
])
def test_scanner(name, code, hazards):
    assert len(load_hazards.scan([line + "\n" for line in code])) == hazards, name
