"""Builds and runs the C++ test of the residual feed-forward operators' edges (tests/cpp/test_nt_block_edges.cpp)."""
import os
import subprocess

import pytest

from conftest import ROOT

BIN = os.path.join(ROOT, "tests", "cpp", "_build", "test_nt_block_edges")


@pytest.fixture(scope="module")
def binary():
    from neurotensor_b200 import _lib
    _lib.lib()
    os.makedirs(os.path.dirname(BIN), exist_ok=True)
    pkg = os.path.join(ROOT, "neurotensor_b200")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-I", os.path.join(ROOT, "include"), "-I", pkg,
                           os.path.join(ROOT, "tests", "cpp", "test_nt_block_edges.cpp"), "-o", BIN, "-L", pkg, "-lntb200", "-Wl,-rpath," + pkg])
    return BIN


def run(binary, case):
    r = subprocess.run([binary, case], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]


def test_cpp_host_operands_are_refused(binary):
    run(binary, "refusals")


@pytest.mark.gpu
def test_cpp_block_in_16_bits(binary):
    run(binary, "block16")
