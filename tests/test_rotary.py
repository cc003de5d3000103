"""CPU checks of the norms with rotation: calls that do not hold are refused before any device work."""

import ctypes
import importlib

import pytest

from test_paged import FAKE, _batch, _cache


@pytest.fixture(scope="module")
def mods(pkg):
    return importlib.import_module("hy_b200.rotary"), importlib.import_module("hy_b200.paged")


def _rotation(rotary, **over):
    f = dict(q_weight_dev=FAKE, k_weight_dev=FAKE, cos_dev=FAKE, sin_dev=FAKE, table_rows=64, table_stride=128,
             positions_dev=FAKE, eps=1e-5, rotate_first=1)
    f.update(over)
    return rotary._Rotation(**f)


def _calls(mods, rotation, rows=2, q_heads=4, kv_heads=2, dim=128, dtype=1, device=0, q=FAKE, k=2 * FAKE, qo=3 * FAKE,
           ko=4 * FAKE, strides=(512, 128), out_strides=(512, 128)):
    rotary, paged = mods
    t = None if rotation is None else ctypes.byref(rotation)
    yield rotary._library().hy_norm_rotate(t, rows, q_heads, kv_heads, dim, dtype, device, q, *strides, k, *strides, qo,
                                           *out_strides, ko, *out_strides, None, None)
    c, b = _cache(paged, head_dim=dim if dim in (64, 128) else 128, num_kv_heads=kv_heads), _batch(paged)
    yield paged._library().hy_paged_kv_write_rotated(ctypes.byref(c), ctypes.byref(b), t, rows, q_heads, dtype, q,
                                                     *strides, k, *strides, 5 * FAKE, *strides, qo, *out_strides, None)


@pytest.mark.parametrize("over,message", [
    (dict(q_weight_dev=None), "null"), (dict(k_weight_dev=None), "null"), (dict(cos_dev=None), "null"),
    (dict(sin_dev=None), "null"), (dict(cos_dev=FAKE + 4), "16 bytes"), (dict(q_weight_dev=FAKE + 8), "16 bytes"),
    (dict(table_stride=130), "16 bytes"), (dict(table_rows=-1), "negative"), (dict(table_stride=-128), "negative"),
    (dict(eps=-1e-5), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
])
def test_rotation_refusals(mods, over, message):
    for rc in _calls(mods, _rotation(mods[0], **over)):
        assert rc == 1
        assert message in mods[0]._library().hy_last_error().decode()


@pytest.mark.parametrize("over,message", [
    (dict(rows=-1), "rows"), (dict(dtype=2), "F32 or BF16"), (dict(q_heads=0), "positive"), (dict(q_heads=2000), "1024"),
    (dict(q=None), "null"), (dict(q=FAKE + 2), "16 bytes"), (dict(strides=(512, 132)), "16 bytes"),
    (dict(strides=(-512, 128)), "negative"), (dict(qo=None), "null"), (dict(out_strides=(0, 128)), "overlap"),
    (dict(out_strides=(512, 64)), "overlap"), (dict(qo=FAKE, out_strides=(1024, 128)), "strides"),
    (dict(qo=2 * FAKE), "overlap"), (dict(rows=1 << 30, q_heads=4), "2^31"),
])
def test_row_refusals(mods, over, message):
    for rc in _calls(mods, _rotation(mods[0]), **over):
        assert rc in (1, 4, 7)
        assert message in mods[0]._library().hy_last_error().decode()


@pytest.mark.parametrize("over,message", [
    (dict(dim=96), "head_dim"), (dict(device=-1), "device"), (dict(kv_heads=0), "positive"), (dict(ko=3 * FAKE), "overlap"),
    (dict(ko=FAKE), "overlap"), (dict(ko=2 * FAKE, out_strides=(1024, 128)), "strides"),
])
def test_row_form_refusals(mods, over, message):
    rc = next(_calls(mods, _rotation(mods[0]), **over))
    assert rc in (1, 7)
    assert message in mods[0]._library().hy_last_error().decode()


def test_cache_form_refuses_outputs_over_its_keys_and_values(mods):
    for over in (dict(qo=5 * FAKE), dict(qo=2 * FAKE)):
        assert list(_calls(mods, _rotation(mods[0]), **over))[1] == 1
        assert b"overlap" in mods[0]._library().hy_last_error()


def test_null_rotation_and_empty_calls(mods):
    assert all(rc == 1 for rc in _calls(mods, None))
    assert all(rc == 0 for rc in _calls(mods, _rotation(mods[0]), rows=0, q=None, k=None, qo=None, ko=None))
