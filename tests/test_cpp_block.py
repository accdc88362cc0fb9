"""Builds and runs the C++ test of the residual feed-forward operators (tests/cpp/test_nt_block.cpp)."""
import os
import subprocess

import pytest

from conftest import ROOT

BIN = os.path.join(ROOT, "tests", "cpp", "_build", "test_nt_block")


def build_binary():
    from neurotensor_b200 import _lib
    _lib.lib()
    os.makedirs(os.path.dirname(BIN), exist_ok=True)
    pkg = os.path.join(ROOT, "neurotensor_b200")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-I", os.path.join(ROOT, "include"), "-I", pkg,
                           os.path.join(ROOT, "tests", "cpp", "test_nt_block.cpp"), "-o", BIN, "-L", pkg, "-lntb200", "-Wl,-rpath," + pkg])
    return BIN


def test_cpp_block_compiles_and_links():
    assert os.path.exists(build_binary())


@pytest.mark.gpu
def test_cpp_block_cases_pass_on_gpu():
    build_binary()   # always against the current header and library
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=300)
    print(r.stdout[-4000:], r.stderr[-2000:])
    assert r.returncode == 0 and "0 of" in r.stdout
