"""CPU checks of the paged cache's C ABI: every call that does not hold is refused before any device work."""

import ctypes
import importlib

import pytest


@pytest.fixture(scope="module")
def paged(pkg):
    return importlib.import_module("hy_b200.paged")


FAKE = 1 << 20   # an aligned address that nothing reads: each call below is refused first


def _cache(paged, **over):
    f = dict(dtype=1, num_pages=4, num_kv_heads=2, page_size=16, head_dim=128, device=0, k_dev=FAKE, v_dev=FAKE,
             page_stride=4096, head_stride=2048, row_stride=128, k_scale_dev=None, v_scale_dev=None,
             scale_page_stride=0, scale_head_stride=0, scale_row_stride=0, status_dev=None)
    f.update(over)
    return paged._Cache(**f)


def _batch(paged, **over):
    f = dict(num_seqs=2, max_rows=1, table_width=4, table_stride=4, q_start_dev=FAKE, kv_len_dev=FAKE,
             block_table_dev=FAKE)
    f.update(over)
    return paged._Batch(**f)


def _calls(paged, cache, batch, rows=2, q_heads=4, dtype=1, a=FAKE, b=2 * FAKE, strides=(512, 128), scale=0.1,
           causal=1, window=0, sinks=0):
    lib = paged._library()
    c, bt = (None if x is None else ctypes.byref(x) for x in (cache, batch))
    yield lib.hy_paged_kv_write(c, bt, rows, dtype, a, *strides, b, *strides, None)
    yield lib.hy_paged_kv_read(c, bt, rows, dtype, a, *strides, b, *strides, None)
    yield lib.hy_paged_attention(c, bt, rows, q_heads, dtype, a, *strides, b, *strides, scale, causal, window, sinks,
                                 None, 0, None)


@pytest.mark.parametrize("over,message", [
    (dict(dtype=4), "dtype"), (dict(dtype=-1), "dtype"), (dict(head_dim=96), "head_dim"), (dict(num_pages=0), "positive"),
    (dict(page_size=0), "positive"), (dict(num_kv_heads=0), "positive"), (dict(k_dev=None), "null"),
    (dict(v_dev=FAKE + 8), "16 bytes"), (dict(row_stride=132), "16 bytes"), (dict(page_stride=-4096), "negative"),
    (dict(dtype=2), "scales"), (dict(dtype=3, k_scale_dev=FAKE), "scales"), (dict(k_scale_dev=FAKE), "scales"),
    (dict(device=-1), "device"), (dict(num_kv_heads=2000), "1024"),
])
def test_cache_refusals(paged, over, message):
    lib = paged._library()
    for rc in _calls(paged, _cache(paged, **over), _batch(paged)):
        assert rc in (1, 7)
        assert message in lib.hy_last_error().decode()


@pytest.mark.parametrize("over,message", [
    (dict(num_seqs=-1), "num_seqs"), (dict(num_seqs=70000), "num_seqs"), (dict(max_rows=-1), "max_rows"),
    (dict(q_start_dev=None), "null"), (dict(kv_len_dev=None), "null"), (dict(block_table_dev=None), "null"),
    (dict(table_width=-1), "negative"), (dict(table_stride=-4), "negative"), (dict(table_width=1 << 28), "2^30"),
])
def test_batch_refusals(paged, over, message):
    lib = paged._library()
    for rc in _calls(paged, _cache(paged), _batch(paged, **over)):
        assert rc in (1, 4)
        assert message in lib.hy_last_error().decode()


@pytest.mark.parametrize("over,message", [
    (dict(rows=-1), "rows"), (dict(dtype=2), "F32 or BF16"), (dict(a=None), "null"), (dict(a=FAKE + 4), "16 bytes"),
    (dict(strides=(512, 130)), "16 bytes"), (dict(strides=(-512, 128)), "negative"),
])
def test_row_refusals(paged, over, message):
    lib = paged._library()
    for rc in _calls(paged, _cache(paged), _batch(paged), **over):
        assert rc == 1
        assert message in lib.hy_last_error().decode()


@pytest.mark.parametrize("over,message", [
    (dict(q_heads=3), "multiple"), (dict(q_heads=0), "multiple"), (dict(window=-1), "negative"),
    (dict(sinks=-1), "negative"), (dict(causal=0, window=4), "causal"), (dict(scale=float("nan")), "finite"),
    (dict(scale=float("inf")), "finite"), (dict(b=FAKE), "overlap"),
])
def test_attention_refusals(paged, over, message):
    lib = paged._library()
    rc = list(_calls(paged, _cache(paged), _batch(paged), **over))[2]
    assert rc in (1, 7)
    assert message in lib.hy_last_error().decode()


def test_null_structs_and_empty_calls(paged):
    lib = paged._library()
    for rc in _calls(paged, None, _batch(paged)):
        assert rc == 1
    for rc in _calls(paged, _cache(paged), None):
        assert rc == 1
    # No rows or no sequences: nothing to do, and no device is needed to find out.
    assert all(rc == 0 for rc in _calls(paged, _cache(paged), _batch(paged), rows=0, a=None, b=None))
    assert all(rc == 0 for rc in _calls(paged, _cache(paged), _batch(paged, num_seqs=0, q_start_dev=None)))


def test_workspace_is_checked(paged):
    lib = paged._library()
    n = ctypes.c_size_t()
    c, b = _cache(paged), _batch(paged)
    assert lib.hy_paged_attention_workspace(ctypes.byref(c), ctypes.byref(b), 2, 4, 1, None) == 1
    assert lib.hy_paged_attention_workspace(ctypes.byref(c), ctypes.byref(b), 2, 3, 1, ctypes.byref(n)) == 1


def test_device_rows_need_a_context(paged):
    lib = paged._library()
    k, v, d, r, h = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_int(), ctypes.c_int64(), ctypes.c_int64()
    assert lib.hy_kv_device_rows(None, 0, ctypes.byref(k), ctypes.byref(v), ctypes.byref(d), ctypes.byref(r),
                                 ctypes.byref(h)) == 1
    assert b"null" in lib.hy_last_error()
