"""CTAs of clusters of the MXFP4 products that share an SM always find their columns of tensor memory, whatever came and went before: a cluster whose CTA waits for columns
while another holds some would otherwise wait for one that waits for it. (CTAs of no cluster come to their end by themselves.) The shared memory a CTA asks for sees to that; its rule is compiled for the host and gone through here.

Columns are given out in powers of two from 32 on, each at a multiple of its size."""
import itertools
import os
import shutil
import subprocess

import pytest

from brotensor_b200 import build

SM_BYTES, RESERVED = 228 * 1024, 1024  # of an SM, and of it for each CTA


@pytest.fixture(scope="module")
def least(tmp_path_factory):
    """columns -> least dynamic shared memory of a CTA that asks for them."""
    if not (os.path.exists(build.NVCC) or shutil.which(build.NVCC)):
        pytest.skip("no nvcc")
    d = tmp_path_factory.mktemp("least")
    (d / "least.cu").write_text('#include <cstdio>\n#include "mx4_common.cuh"\nint main() { for (unsigned c = 32; c <= 512; c *= 2) std::printf("%u %zu\\n", c, b200q::mx_smem_for_tmem(1, c, true)); }\n')
    cmd = [build.NVCC] + build.ARCH + ["-std=c++17", "-I" + build.CSRC, str(d / "least.cu"), "-o", str(d / "least")]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    out = subprocess.run([str(d / "least")], capture_output=True, text=True, check=True).stdout
    return {int(a): int(b) for a, b in (line.split() for line in out.splitlines())}


def _placements(held):
    """Every way in which the columns of `held` may lie after any history: each at some multiple of its size, none over another."""
    for at in itertools.product(*[range(0, 512, c) for c in held]):
        taken = sorted((a, a + c) for a, c in zip(at, held))
        if all(x[1] <= y[0] for x, y in zip(taken, taken[1:])):
            yield taken


def test_whoever_fits_an_sm_finds_columns(least):
    checked = 0
    for n in range(1, 9):
        for held in itertools.combinations_with_replacement(sorted(least), n):
            if sum(least[c] + RESERVED for c in held) > SM_BYTES:
                continue
            for new in least:
                if sum(least[c] + RESERVED for c in held) + least[new] + RESERVED > SM_BYTES:
                    continue
                for taken in _placements(held):
                    checked += 1
                    assert any(all(hi <= a or a + new <= lo for lo, hi in taken) for a in range(0, 512, new)), f"{new} columns beside {taken}"
    assert checked > 100
