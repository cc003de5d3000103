"""CPU checks of the attention weights and the eviction: calls that do not hold are refused before any device work."""

import ctypes
import importlib
import os
import re

import pytest

from test_paged import FAKE, _batch, _cache


@pytest.fixture(scope="module")
def paged(pkg):
    return importlib.import_module("hy_b200.paged")


def _weights(paged, **over):
    f = dict(weights_dev=3 * FAKE, page_stride=32, head_stride=16, row_stride=1)
    f.update(over)
    return paged._Weights(**f)


def _add(paged, cache=None, batch=None, weights=None, rows=2, q_heads=4, dtype=1, q=FAKE, strides=(512, 128), lse=2 * FAKE,
         lse_strides=(4, 1), scale=0.1, causal=1, window=0, sinks=0):
    c, b, w = cache or _cache(paged), batch or _batch(paged), weights or _weights(paged)
    return paged._library().hy_paged_add_weights(ctypes.byref(c), ctypes.byref(b), rows, q_heads, dtype, q, *strides, lse,
                                                 *lse_strides, scale, causal, window, sinks, ctypes.byref(w), None)


def _evict(paged, cache=None, batch=None, weights=None, keep=8, first=1, recent=2, kv_len=FAKE, kept=4 * FAKE):
    c, b, w = cache or _cache(paged), batch or _batch(paged), weights or _weights(paged)
    return paged._library().hy_paged_evict(ctypes.byref(c), ctypes.byref(b), keep, first, recent, ctypes.byref(w), kv_len,
                                           kept, None)


def _says(paged, message):
    return message in paged._library().hy_last_error().decode()


@pytest.mark.parametrize("over,message", [
    (dict(rows=-1), "rows"), (dict(dtype=3), "F32 or BF16"), (dict(q_heads=3), "multiple"), (dict(q=None), "null"),
    (dict(q=FAKE + 4), "16 bytes"), (dict(strides=(512, 130)), "16 bytes"), (dict(lse=None), "lse is null"),
    (dict(lse=2 * FAKE + 2), "aligned"), (dict(lse_strides=(-4, 1)), "negative"), (dict(lse_strides=(0, 1)), "overlap"),
    (dict(lse_strides=(4, 0)), "overlap"), (dict(lse=3 * FAKE), "overlap"), (dict(scale=0.0), "scale"),
    (dict(scale=float("inf")), "finite"), (dict(window=-1), "negative"), (dict(sinks=-1), "negative"),
    (dict(causal=0, window=3), "causal"), (dict(rows=1 << 28, q_heads=4), "2^30"),
])
def test_add_refusals(paged, over, message):
    assert _add(paged, **over) in (1, 4, 7)
    assert _says(paged, message)


@pytest.mark.parametrize("call", [_add, _evict])
@pytest.mark.parametrize("over,message", [
    (dict(weights_dev=None), "null"), (dict(weights_dev=3 * FAKE + 2), "aligned"), (dict(page_stride=-1), "negative"),
    (dict(row_stride=0), "overlap"), (dict(head_stride=0), "overlap"), (dict(page_stride=0), "overlap"),
])
def test_weights_refusals(paged, call, over, message):
    assert call(paged, weights=_weights(paged, **over)) == 1
    assert _says(paged, message)


@pytest.mark.parametrize("over,message", [
    (dict(keep=0), "keep"), (dict(first=-1), "keep"), (dict(recent=-1), "keep"), (dict(keep=4, first=2, recent=3), "keep"),
    (dict(first=2 ** 31 - 1, recent=2 ** 31 - 1), "keep"), (dict(kept=None), "null"),
    (dict(kv_len=2 * FAKE), "own"), (dict(kept=FAKE), "overlap"),
])
def test_evict_refusals(paged, over, message):
    assert _evict(paged, **over) == 1
    assert _says(paged, message)


@pytest.mark.parametrize("over", [dict(row_stride=0), dict(head_stride=0), dict(page_stride=0)])
def test_eviction_refuses_rows_in_one_place(paged, over):
    assert _evict(paged, cache=_cache(paged, **over)) == 1
    assert _says(paged, "overlap")


def test_eviction_refuses_scales_in_one_place(paged):
    """One scale for a page is fine to read, but rows that move need theirs."""
    codes = dict(dtype=2, k_scale_dev=FAKE, v_scale_dev=FAKE, scale_page_stride=32, scale_head_stride=16)
    assert _evict(paged, cache=_cache(paged, **codes, scale_row_stride=0)) == 1
    assert _says(paged, "overlap")


def test_bad_caches_batches_and_empty_calls(paged):
    for call in (_add, _evict):
        assert call(paged, cache=_cache(paged, head_dim=96)) == 7 and _says(paged, "head_dim")
        assert call(paged, batch=_batch(paged, num_seqs=-1)) == 1 and _says(paged, "num_seqs")
        assert call(paged, batch=_batch(paged, num_seqs=0)) == 0
    assert _add(paged, rows=0, q=None, lse=None) == 0


@pytest.mark.parametrize("over,message", [
    (dict(lse=FAKE), "overlap"), (dict(lse=2 * FAKE), "overlap"), (dict(lse=3 * FAKE + 2), "aligned"),
    (dict(strides=(-1, 1)), "negative"), (dict(strides=(1, 1)), None), (dict(strides=(0, 1)), "overlap"),
])
def test_lse_refusals_of_the_attention(paged, over, message):
    lib = paged._library()
    f = dict(lse=3 * FAKE, strides=(4, 1))
    f.update(over)
    c, b = _cache(paged), _batch(paged)
    rc = lib.hy_paged_attention_lse(ctypes.byref(c), ctypes.byref(b), 2, 4, 1, FAKE, 512, 128, 2 * FAKE, 512, 128,
                                    f["lse"], *f["strides"], 0.1, 1, 0, 0, None, 0, None)
    assert rc == 1 and _says(paged, message or "workspace")


def test_waits_of_the_tensor_core_kernel_end_alike_in_a_whole_warp():
    """What follows a wait there is of the whole warp (tensor memory, shuffles, barriers that a warp arrives at once), so
    every wait is one of those that vote; and every arrival of a thread alone is the products' leader's."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hunyuanocr-ncnn_b200", "csrc",
                        "hy_paged_weigh_chunk.cuh")
    with open(path) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    assert not re.findall(r"\bmbar_(?:try_)?wait(?:_spin)?\(", text)
    assert len(re.findall(r"\bwarp_wait(?:_spin)?\(", text)) >= 10
    assert len(re.findall(r"\bmbar_arrive\(", text)) == 2   # warp_arrive's own, and the leader's
