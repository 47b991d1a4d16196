"""The row operators' libraries without a device: what their entry points refuse before a launch,
what needs which library, and what the kernels keep in registers."""

import os
import re
import subprocess
import sys

import pytest

from muonium_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = "/opt/rocm/bin/hipcc"


@pytest.mark.parametrize("call, code", [
    (lambda L: L.muon_policy_loss_rescale(1, 7, 4, 3, 4, 1, 1.0, 1, 1, 1, 1, None), 2),
    (lambda L: L.muon_policy_loss_rescale(1, 1, 4, 3, 0, 1, 1.0, 1, 1, 1, 1, None), 1),
    (lambda L: L.muon_policy_loss_rescale(1, 1, 4, 3, 4, 1, 0.0, 1, 1, 1, 1, None), 5),
    (lambda L: L.muon_policy_loss_rescale(1, 2, 4, 3, 4, 1, 1.0, 1, 1, 1, 1, None), 5),
    (lambda L: L.muon_policy_loss_rescale(1, 0, 1 << 17, 3, 1 << 17, 1, 1.0, 1, 1, 1, 1, None), 5),
    (lambda L: L.muon_policy_loss_rescale(1, 1, 4, 3, 4, 1, 1.0, None, 1, 1, 1, None), 5),
    (lambda L: L.muon_policy_loss_rescale(1, 1, 4, 3, 4, 1, 1.0, 1, None, 1, 1, None), 5),
    (lambda L: L.muon_policy_loss_rescale(1, 1, 4, 3, 4, 1, 1.0, 1, 1, None, 1, None), 5),
    (lambda L: L.muon_policy_loss_rescale(1, 1, 4, 3, 4, 1, 1.0, 1, 1, 1, None, None), 5),
])
def test_rescale_refuses_without_launching(call, code):
    assert call(_lib.load()) == code
    assert "policy_loss_rescale" in _lib.last_error()


def test_rescale_of_no_rows_returns_ok():
    assert _lib.load().muon_policy_loss_rescale(None, 1, 4, 0, 4, None, 1.0, None, None, None, None, None) == 0


@pytest.mark.parametrize("bits", [0, 8, 16, 128])
def test_positions_are_of_32_or_64_bits(bits):
    """The kernels read positions of no other width: the call would read past their end."""
    lib, s = _lib.load(), _lib.i64_array([8] * 12)
    assert lib.muon_qk_norm_rope(1, 1, s, None, None, 0, 1, 1, 9, 1, bits, 0, 1, 1, 1, 1, 1, 1, 1, 8, 8, 0,
                                 1e-6, None) == 5
    assert "positions" in _lib.last_error()
    assert lib.muon_qk_norm_rope_backward(1, 1, 1, 1, s, None, None, 0, 1, 1, 9, 1, bits, 0, 1, 1, None, None,
                                          None, 1, 1, 1, 1, 1, 8, 8, 0, 1e-6, None) == 5
    assert "positions" in _lib.last_error()


def run_python(code):
    path = os.path.join(ROOT, "dtensor-muon_amd")
    return subprocess.run([sys.executable, "-c", code, path], capture_output=True, text=True, timeout=300)


def test_gram_needs_nothing_of_the_torch_operators():
    """Its import neither loads nor misses their library; theirs says what is missing."""
    done = run_python('''
import sys
sys.path.insert(0, sys.argv[1])
import muonium_amd.kernels as kernels
from muonium_amd.kernels import gram, gram_
from muonium_amd import _lib
assert "muonium_amd._row_ops" not in sys.modules
assert "libmuon_amd_torch" not in open("/proc/self/maps").read()
assert {"gram", "route", "policy_loss", "Routing"} <= set(dir(kernels))
_lib._LIB_PATH = "/nowhere/libmuon_amd.so"
try:
    from muonium_amd.kernels import route
except ImportError as e:
    assert "libmuon_amd_torch.so is missing" in str(e), e
else:
    raise AssertionError("imported")
assert not hasattr(kernels, "other")
''')
    assert done.returncode == 0, done.stderr
    done = run_python('''
import sys
sys.path.insert(0, sys.argv[1])
from muonium_amd.kernels import *
import muonium_amd.kernels as kernels
assert kernels.route is route and "libmuon_amd_torch" in open("/proc/self/maps").read()
assert qk_norm_rope and token_logprobs and policy_loss and gram and gram_ and PolicyLoss and Routing
''')
    assert done.returncode == 0, done.stderr


def planned(tmp_path, python):
    """What make would run from nothing, with `python` as its python3."""
    (tmp_path / "python3").write_text(f"#!/bin/sh\n{python}\n")
    (tmp_path / "python3").chmod(0o755)
    env = {**os.environ, "PATH": f"{tmp_path}:{os.environ['PATH']}"}
    env.pop("TORCH_DIR", None)
    done = subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "dtensor-muon_amd", "csrc")],
                          env=env, capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stderr
    assert "-shared -fPIC -o ../muonium_amd/_lib/libmuon_amd.so.tmp" in done.stdout
    return done.stdout


@pytest.mark.parametrize("missing", ["python", "torch", "rocm"])
def test_make_builds_the_c_abi_without_torch(tmp_path, missing):
    """Without a python3, without torch, and beside a torch of another device."""
    (tmp_path / "torch").mkdir()
    (tmp_path / "torch" / "__init__.py").write_text("")
    python = {"python": "exit 127",
              "torch": f'exec {sys.executable} -I -S "$@"',
              "rocm": f'PYTHONPATH={tmp_path} exec {sys.executable} -S "$@"'}[missing]
    plan = planned(tmp_path, python)
    assert "row_ops.cpp" not in plan and "is not built" in plan


def test_make_builds_the_torch_operators_with_torch(tmp_path):
    plan = planned(tmp_path, f'exec {sys.executable} "$@"')
    assert "row_ops.cpp" in plan and "is not built" not in plan


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")
def test_rescale_kernels_use_no_scratch(tmp_path):
    asm = tmp_path / "kernels.s"
    cmd = [HIPCC, "-O3", "-std=c++17", "--offload-arch=gfx950", "-fPIC", "-w", "-mllvm",
           "-pragma-unroll-threshold=1000000", "-Xclang", "-target-feature", "-Xclang",
           "-packed-fp32-ops", "-I" + os.path.join(ROOT, "include"), "--cuda-device-only", "-S",
           os.path.join(ROOT, "dtensor-muon_amd", "csrc", "rescale.hip"), "-o", str(asm)]
    subprocess.run(cmd, check=True, capture_output=True, timeout=900)
    text = asm.read_text()
    found = re.findall(r"\.private_segment_fixed_size:\s+(\d+).*?\.vgpr_spill_count:\s+(\d+)", text, re.S)
    assert len(found) == 4 and all(f == ("0", "0") for f in found)
    assert not re.search(r"v_pk_(add|mul|fma)_f32", text)
