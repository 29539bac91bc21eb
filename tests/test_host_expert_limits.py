"""What the expert ops of the C++ host layer refuse, and their largest images: tests/cpp/expert_limits_tests.cpp, a run for each of its tests."""
import importlib.util
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def exe():
    spec = importlib.util.spec_from_file_location("build_expert_limits_tests", os.path.join(ROOT, "tests", "cpp", "build_expert_limits_tests.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod.build()


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["plan", "image"])
def test_expert_limits(exe, which):
    r = subprocess.run([exe, which], capture_output=True, text=True, timeout=300)
    sys.stdout.write(r.stdout[-3000:] + r.stderr[-2000:])
    assert r.returncode == 0 and "OK (0 failures)" in r.stdout and "skipping" not in r.stdout
