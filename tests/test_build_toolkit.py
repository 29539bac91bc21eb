"""What the sources ask of the toolkit: instructions that came late stand behind a check of its version."""
import os
import re
import shutil
import subprocess

import pytest

from brotensor_b200 import build

LATE = r"st\.global\.v8"  # PTX ISA 8.8: CUDA 12.9


def _preprocessed(source, *defines):
    if not (os.path.exists(build.NVCC) or shutil.which(build.NVCC)):
        pytest.skip("no nvcc")
    cmd = [build.NVCC] + build.ARCH + ["-std=c++17", "-E", os.path.join(build.CSRC, source)] + [f"-D{d}" for d in defines]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    return r.stdout


def test_stores_of_32_bytes_stand_in_one_place_behind_the_check():
    found = {}
    for name in sorted(os.listdir(build.CSRC)):
        with open(os.path.join(build.CSRC, name)) as f:
            n = len(re.findall(LATE, f.read()))
        if n:
            found[name] = n
    assert found == {"mx4_common.cuh": 1}


@pytest.mark.parametrize("source", ["mx4_quant.cu", "mx4_wide.cu"])
def test_without_them_an_older_toolkit_gets_two_of_16(source):
    assert re.search(LATE, _preprocessed(source, "B200Q_STORE32=1"))
    assert not re.search(LATE, _preprocessed(source, "B200Q_STORE32=0"))


@pytest.mark.parametrize("major,minor,has", [(12, 8, 0), (12, 9, 1), (13, 0, 1), (11, 9, 0)])
def test_the_check_goes_by_the_version(major, minor, has, tmp_path):
    with open(os.path.join(build.CSRC, "mx4_common.cuh")) as f:
        text = f.read()
    start = text.index("#ifndef B200Q_STORE32")
    depth, lines = 0, []
    for line in text[start:].splitlines():
        lines.append(line)
        depth += line.startswith("#if") - line.startswith("#endif")
        if depth == 0:
            break
    (tmp_path / "check.h").write_text("\n".join(lines) + "\nvalue = B200Q_STORE32\n")
    r = subprocess.run(["g++", "-E", "-P", "-x", "c++", f"-D__CUDACC_VER_MAJOR__={major}", f"-D__CUDACC_VER_MINOR__={minor}", str(tmp_path / "check.h")],
                       capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == f"value = {has}", r.stdout + r.stderr
