"""MXFP4 tensors and expert layers through the C++ host layer: its own test executable (tests/cpp/expert_tests.cpp)."""
import importlib.util
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def exe():
    spec = importlib.util.spec_from_file_location("build_expert_tests", os.path.join(ROOT, "tests", "cpp", "build_expert_tests.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod.build()


def _run(exe, mode):
    r = subprocess.run([exe, mode], capture_output=True, text=True, timeout=300)
    sys.stdout.write(r.stdout[-3000:] + r.stderr[-2000:])
    assert r.returncode == 0 and "OK (0 failures)" in r.stdout and "skipping" not in r.stdout


def test_host_experts_cpu(exe):
    _run(exe, "cpu")


@pytest.mark.gpu
def test_host_experts_gpu(exe):
    _run(exe, "gpu")
