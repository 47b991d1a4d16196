"""The torch operators' library in a program without Python: it loads beside libtorch, and its operators are
registered there."""

import importlib.util
import os
import shutil
import subprocess

import pytest

from muonium_amd import _row_ops

PROGRAM = r'''
#include <dlfcn.h>
#include <stdio.h>
int main(int argc, char** argv) {
  void* lib = dlopen(argv[1], RTLD_NOW | RTLD_GLOBAL);
  if (!lib) {
    fprintf(stderr, "%s\n", dlerror());
    return 1;
  }
  puts("loaded");
  return 0;
}
'''


@pytest.fixture
def loader(tmp_path):
    compiler = shutil.which("gcc") or shutil.which("cc")
    if compiler is None:
        pytest.skip("needs a C compiler")
    (tmp_path / "load.c").write_text(PROGRAM)
    subprocess.run([compiler, str(tmp_path / "load.c"), "-o", str(tmp_path / "load"), "-ldl"], check=True)
    torch_lib = os.path.join(os.path.dirname(importlib.util.find_spec("torch").origin), "lib")
    env = {**os.environ, "LD_LIBRARY_PATH": ":".join([torch_lib, "/opt/rocm/lib", os.environ.get("LD_LIBRARY_PATH", "")])}
    return lambda path: subprocess.run([str(tmp_path / "load"), path], env=env, capture_output=True, text=True, timeout=300)


def test_the_operators_library_loads_without_python(loader):
    done = loader(_row_ops._TORCH_LIB_PATH)
    assert done.returncode == 0 and done.stdout == "loaded\n", done.stderr


def test_the_operators_library_asks_for_no_python():
    needed = subprocess.run(["readelf", "-d", _row_ops._TORCH_LIB_PATH], capture_output=True, text=True, check=True).stdout
    assert "libtorch_cpu" in needed and "python" not in needed


def test_the_walker_is_a_module_of_its_own():
    if not os.path.exists(_row_ops._PYTHON_LIB_PATH):
        pytest.skip("built without Python's headers")
    assert callable(_row_ops.module.adamw_step)
    with pytest.raises(TypeError, match="adamw_step|step\\("):
        _row_ops.module.adamw_step(1)
