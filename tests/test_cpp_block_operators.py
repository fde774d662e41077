"""The operators around a block's matrix products through the C++ templates of include/portdnn: they compile as plain C++17 against
the C ABI, and on a GPU tests/cpp/block_operators_test.cc passes."""
import os
import subprocess

import pytest

from test_cpp_api import CUDA, ROOT

SRC, EXE = (os.path.join(ROOT, "tests", "cpp", "block_operators_test" + e) for e in (".cc", ""))


def _build():
    from portdnn_b200 import build
    build.build()
    cmd = ["g++", "-std=c++17", "-Wall", "-I" + os.path.join(ROOT, "include"), "-I" + os.path.join(CUDA, "include"), SRC,
           "-L" + os.path.join(ROOT, "portdnn_b200"), "-lportdnn_b200", "-L" + os.path.join(CUDA, "lib64"), "-lcudart",
           "-Wl,-rpath," + os.path.join(ROOT, "portdnn_b200"), "-Wl,-rpath," + os.path.join(CUDA, "lib64"), "-o", EXE]
    res = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert res.returncode == 0, res.stdout
    return EXE


def test_headers_compile_and_link():
    assert os.path.exists(_build())


@pytest.mark.gpu
def test_program_passes():
    res = subprocess.run([_build()], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert res.returncode == 0, res.stdout
    assert "all checks passed" in res.stdout
