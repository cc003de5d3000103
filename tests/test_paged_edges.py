"""CPU checks of the paged cache at the edges of what its calls allow."""

import ctypes
import importlib
import itertools
import os
import re

import pytest

from test_paged import FAKE, _batch, _cache, _calls

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


@pytest.mark.parametrize("strides", [(0, 128), (512, 0), (64, 512), (512, 120)])
def test_outputs_that_overlap_themselves_are_refused(paged, strides):
    """Rows or heads of an output that share memory would be written by several blocks at once."""
    lib = paged._library()
    c, b = _cache(paged), _batch(paged)
    ref = [ctypes.byref(x) for x in (c, b)]
    assert lib.hy_paged_kv_read(*ref, 2, 1, FAKE, *strides, 2 * FAKE, 512, 128, None) == 1
    assert b"k rows must not overlap" in lib.hy_last_error()
    assert lib.hy_paged_kv_read(*ref, 2, 1, FAKE, 512, 128, 2 * FAKE, *strides, None) == 1
    assert b"v rows must not overlap" in lib.hy_last_error()
    assert lib.hy_paged_attention(*ref, 2, 4, 1, FAKE, 512, 128, 2 * FAKE, *strides, 0.1, 1, 0, 0, None, 0, None) == 1
    assert b"out rows must not overlap" in lib.hy_last_error()


def test_one_output_for_keys_and_values_is_refused(paged):
    lib = paged._library()
    c, b = _cache(paged), _batch(paged)
    assert lib.hy_paged_kv_read(ctypes.byref(c), ctypes.byref(b), 2, 1, FAKE, 512, 128, FAKE, 512, 128, None) == 1
    assert b"overlap" in lib.hy_last_error()


@pytest.mark.parametrize("rows_stride,cache_stride", [((1 << 31, 128), 2048), ((512, 1 << 31), 2048), ((512, 128), 1 << 31)])
def test_long_strides_are_refused_before_any_device_call(paged, rows_stride, cache_stride):
    lib = paged._library()
    calls = _calls(paged, _cache(paged, head_stride=cache_stride), _batch(paged), strides=rows_stride)
    for rc in itertools.islice(calls, 2):
        assert rc == 4
        assert b"2^31" in lib.hy_last_error()
