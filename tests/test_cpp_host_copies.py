"""The copies of the C++ host mirror (include/llmc_b200.hpp) are ordered with a context's work: tests/cpp/host_copies.cpp
runs them on the CPU over a stand-in for the CUDA runtime whose streams do not wait for one another."""

import os
import shutil
import subprocess

import pytest

from test_cpp_host import CUDA, ROOT


def test_copies_are_ordered_with_the_contexts_work(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path / "host_copies")
    cmd = [gxx, "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(CUDA, "include"),
           os.path.join(ROOT, "tests", "cpp", "host_copies.cpp"), "-o", exe]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "0 failed\n", r.stdout
