"""CPU checks of the paged cache at the edges of what its calls allow."""

import importlib
import os
import re

import pytest

from test_paged import _batch, _cache, _calls

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hunyuanocr-ncnn_b200", "csrc")


def test_waits_of_the_wide_kernel_end_alike_in_a_whole_warp():
    """What follows a wait there is of the whole warp (tensor memory, shuffles), so a wait's outcome has to be too:
    every one goes through a vote."""
    with open(os.path.join(CSRC, "hy_paged_chunk.cuh")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    waits = re.findall(r"[^\n;{]*\bmbar_(?:try_)?wait(?:_spin)?\(", text)
    assert len(waits) == 3
    assert all("__all_sync(0xffffffffu, mbar_" in w for w in waits), waits
    uses = re.findall(r"[^\n;{]*\bwarp_wait(?:_spin)?\([^;]*;", text)
    assert len(uses) > 20


@pytest.fixture(scope="module")
def paged(pkg):
    return importlib.import_module("hy_b200.paged")


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38, 0.0, -0.1])
def test_scales_whose_multiple_overflows_are_refused(paged, scale):
    """The kernels multiply scores by scale * log2(e) in 32 bits: with an infinity there a score of 0 would be NaN."""
    rc = list(_calls(paged, _cache(paged), _batch(paged), scale=scale))[2]
    assert rc == 1
    assert b"finite" in paged._library().hy_last_error()
