"""Builds tests/cpp/expert_limits_tests (expert_limits_tests.cpp): what ops/experts.h refuses, and its largest images. Test infrastructure."""
from __future__ import annotations

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
LIBDIR = os.path.join(ROOT, "brotensor_b200", "lib")
EXE = os.path.join(HERE, "expert_limits_tests")


def build(force: bool = False) -> str:
    if ROOT not in sys.path:
        sys.path.insert(0, ROOT)
    from brotensor_b200 import build as product
    product.build_all()
    src = os.path.join(HERE, "expert_limits_tests.cpp")
    deps = [src, os.path.join(LIBDIR, "libbrotensor_b200.so")]
    if force or not os.path.exists(EXE) or any(os.path.getmtime(d) > os.path.getmtime(EXE) for d in deps):
        cmd = ["g++", "-std=c++20", "-O1", "-o", EXE, src, "-I" + os.path.join(ROOT, "include"), "-I/usr/local/cuda/include", "-L" + LIBDIR,
               "-lbrotensor_b200", "-lb200q", "-L/usr/local/cuda/lib64", "-lcudart", "-Wl,-rpath," + LIBDIR, "-lpthread"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            sys.stderr.write(" ".join(cmd) + "\n" + r.stdout + r.stderr)
            raise RuntimeError("building tests/cpp/expert_limits_tests failed")
    return EXE
