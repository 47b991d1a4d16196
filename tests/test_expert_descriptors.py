"""The buffer descriptors of the experts' product kernels are whole wherever a load can be reached from
(descriptor_scan.py): expert_gemm.hip is compiled for gfx950 and scanned, the scanner on small pieces."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
HIPCC = "/opt/rocm/bin/hipcc"
sys.path.insert(0, HERE)
import descriptor_scan  # noqa: E402
import load_hazards  # noqa: E402


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
def test_product_kernels_load_through_whole_descriptors(tmp_path):
    asm = tmp_path / "expert_gemm.s"
    subprocess.run([HIPCC, "-O3", "-std=c++17", "--offload-arch=gfx950", "-fPIC", "-w", "-mllvm",
                    "-pragma-unroll-threshold=1000000", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                    "-I" + os.path.join(ROOT, "include"), "--cuda-device-only", "-S",
                    os.path.join(ROOT, "dtensor-muon_amd", "csrc", "expert_gemm.hip"), "-o", str(asm)],
                   check=True, capture_output=True, timeout=900)
    found = [(n, lines) for n, lines in load_hazards.kernels(asm) if "expert_gemm_pipe" in n]
    assert len(found) == 6
    for name, lines in found:
        assert sum(" lds" in x for x in lines) >= 64, name
        assert not descriptor_scan.scan(lines), name


_SET = ["s_mov_b32 s7, 0x20000"]
_LOAD = ["buffer_load_dwordx4 v2, s[4:7], s9 offen lds"]


@pytest.mark.parametrize("name, code, bad", [
    ("set", _SET + _LOAD, 0),
    ("never set", _LOAD, 1),
    ("written over", _SET + ["s_mul_i32 s7, s1, s2"] + _LOAD, 1),
    ("copied", ["s_mov_b32 s31, 0x20000", "s_mov_b64 s[6:7], s[30:31]"] + _LOAD, 0),
    ("its neighbour copied", ["s_mov_b32 s30, 0x20000", "s_mov_b64 s[6:7], s[30:31]"] + _LOAD, 1),
    ("kept in a lane", _SET + ["v_writelane_b32 v255, s7, 3", "s_mov_b32 s7, 0", "v_readlane_b32 s7, v255, 3"] + _LOAD, 0),
    ("another lane", _SET + ["v_writelane_b32 v255, s7, 3", "v_readlane_b32 s7, v255, 4"] + _LOAD, 1),
    ("a mask", _SET + ["v_cmp_lt_i32_e64 s[6:7], s1, v2"] + _LOAD, 1),
    ("on both ways", ["s_cbranch_scc0 .LBB0_1"] + _SET + ["s_branch .LBB0_2", ".LBB0_1:"] + _SET + [".LBB0_2:"] + _LOAD, 0),
    ("on one way", ["s_cbranch_scc0 .LBB0_1"] + _SET + [".LBB0_1:"] + _LOAD, 1),
    ("around a loop", _SET + [".LBB0_1:"] + _LOAD + ["s_mov_b32 s7, s8", "s_cbranch_scc0 .LBB0_1"], 1),
    ("where nothing comes", ["s_endpgm", ".LBB0_1:"] + _LOAD, 0),
])
def test_scanner(name, code, bad):
    assert len(descriptor_scan.scan(code)) == bad
