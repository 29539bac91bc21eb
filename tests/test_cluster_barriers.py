"""MXFP4 products: barriers at which other CTAs of a cluster arrive are waited for and arrived at with the cluster's scope. (What goes wrong otherwise depends on the hardware's
timing; the sources are what can be checked.)"""
import os
import re

import pytest

from brotensor_b200 import build


def _source(name):
    with open(os.path.join(build.CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


# bar_full of a pair's leader counts its own copies, and the other CTA's through the relay; it is waited for like the copies it stands for.
@pytest.mark.parametrize("name,barriers", [("mx4_gemm.cu", {"bar_parts": "kMbarCluster"}),
                                           ("mx4_wide.cu", {"bar_full": "", "bar_empty": "kMbarOrder", "bar_accum": "kMbarOrder", "bar_free": "kMbarOrder"})])
def test_waits(name, barriers):
    text = _source(name)
    remote = set(re.findall(r"mx_map_to_rank\(smem_u32\(&(bar_\w+)", text)) | set(re.findall(r"wide_commit\(smem_u32\(&(bar_\w+)", text))
    assert remote == set(barriers)
    for b, how in barriers.items():
        waits = set(re.findall(r"mx_warp_wait(?:<(\w+)>)?\(smem_u32\(&" + b + r"\b", text))
        assert waits == {how}, b


def test_arrivals():
    for name in ("mx4_common.cuh", "mx4_gemm.cu", "mx4_wide.cu"):
        for asm in re.findall(r'"(mbarrier\.arrive[^"]*shared::cluster[^"]*)"', _source(name)):
            assert asm.startswith("mbarrier.arrive.relaxed.cluster."), (name, asm)
    text = _source("common.cuh")
    assert "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64" in text and "mbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64" in text


@pytest.mark.parametrize("name,alloc", [("mx4_gemm.cu", "tmem_alloc"), ("mx4_wide.cu", "wide_alloc")])
def test_dependents_are_let_go_behind_the_allocation(name, alloc):
    """A kernel that follows may start from then on. Had it taken the tensor memory's columns first, it would wait for this kernel's end and this kernel for the columns."""
    text = _source(name)
    body = text[text.index("__launch_bounds__"):]
    assert body.count("grid_dep_launch()") == 1
    block = re.search(r"if \(warp == 1\) \{\s*" + alloc + r"\(([^{}]*)\}", body)
    assert block and "grid_dep_launch();" in block.group(0)
