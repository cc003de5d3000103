"""CPU checks of the calls around the paged cache and behind the LM head: numbers past 32 bits, which a C int would wrap,
are refused before the library is called."""

import importlib

import pytest
import torch

import test_paged
import test_paged_weights
import test_rotary


@pytest.fixture(scope="module")
def paged(pkg):
    return importlib.import_module("hy_b200.paged")


class Reached(Exception):
    pass


class NoLibrary:
    """Stands for the library: a call that gets there was not refused."""

    def __getattr__(self, name):
        def call(*args):
            raise Reached(name)
        return call


def _cache(paged, dtype=torch.float32):
    """A cache of host memory without a library behind it: only the checks before a call can run."""
    c = object.__new__(paged.PagedKVCache)
    c._lib, c.k, c.device, c._index, c._heads, c._dim = NoLibrary(), torch.zeros(4, 2, 8, 64, dtype=dtype), "cpu", -1, 2, 64
    c._ref, c._workspace = None, {}
    return c


def _batch(paged):
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)   # noqa: E731
    return paged.PagedBatch(i32(0, 1), i32(20), torch.zeros(1, 3, dtype=torch.int32), 1)


@pytest.mark.parametrize("over", [
    dict(recent=2 ** 32), dict(first=2 ** 32), dict(recent=2 ** 32 + 3), dict(first=-2 ** 32), dict(recent=-1),
    dict(first=5, recent=5), dict(keep=0), dict(keep=-2 ** 32 + 8), dict(keep=2 ** 32 + 8), dict(keep=2 ** 31),
])
def test_evict_sizes(paged, pkg, over):
    c, f = _cache(paged), dict(keep=8, first=1, recent=2)
    f.update(over)
    with pytest.raises(pkg.HyError, match="keep"):
        c.evict(_batch(paged), f["keep"], torch.zeros(4, 2, 8), first=f["first"], recent=f["recent"])


@pytest.fixture
def no_stream(paged, monkeypatch):
    monkeypatch.setattr(paged, "_raw_stream", lambda index: 0)


def test_evict_sizes_that_hold_reach_the_library(paged, no_stream):
    for keep, first, recent in ((8, 0, 0), (8, 3, 5), (1, 0, 1)):
        with pytest.raises(Reached, match="hy_paged_evict"):
            _cache(paged).evict(_batch(paged), keep, torch.zeros(4, 2, 8), first=first, recent=recent)


@pytest.mark.parametrize("keep", [2 ** 30 + 1, 2 ** 31 - 512, 2 ** 31 - 1])
def test_eviction_to_more_than_positions_reach(paged, keep):
    """The list of what stays is walked in steps of a CTA's threads, by a C int that must not pass its largest."""
    assert test_paged_weights._evict(paged, keep=keep) == 1
    assert "2^30" in paged._library().hy_last_error().decode()
    assert test_paged_weights._evict(paged, keep=2 ** 30, batch=test_paged._batch(paged, num_seqs=0)) == 0


@pytest.mark.parametrize("top", [2 ** 32, 2 ** 32 + 3, -2 ** 32, -1, 65])
def test_alternatives_behind_the_lm_head(pkg, monkeypatch, top):
    """(2^32 came to the library as 0, and arrays that nobody had written came back.)"""
    monkeypatch.setattr(pkg, "_LIB", NoLibrary())
    rt = object.__new__(pkg.TextRuntime)
    rt._ctx = None
    with pytest.raises(pkg.HyError, match="top"):
        rt.lm_head_logprobs(torch.zeros(2, 1024).numpy(), top=top)
    with pytest.raises(Reached, match="hy_lm_head_logprobs"):
        rt.lm_head_logprobs(torch.zeros(2, 1024).numpy(), top=64)
    del rt._ctx


class Shape:
    """Stands for a tensor on a device: what the checks before a call read of it."""
    requires_grad = False

    def __init__(self, *shape, dtype=torch.float32):
        self.shape, self.dtype = torch.Size(shape), dtype

    def get_device(self):
        return 0

    def stride(self):
        return (self.shape[1], 1)

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 1 << 20

    def new_empty(self, shape, dtype=None):
        return Shape(*(shape if isinstance(shape, tuple) else (shape,)), dtype=dtype or self.dtype)


@pytest.mark.parametrize("rows,vocab,tokens", [
    (2 ** 32, 1, (2 ** 32,)), (2 ** 32 + 2, 5, (2 ** 32 + 2,)), (1, 2 ** 32 + 100, (1,)), (1, 9, (1, 2 ** 32)),
    (2, 9, (2, 2 ** 32 + 1)),
])
def test_log_probabilities_past_32_bits(pkg, monkeypatch, rows, vocab, tokens):
    """(A C int would wrap, and arrays that nobody had written would come back.)"""
    logprobs = importlib.import_module("hy_b200.logprobs")
    monkeypatch.setattr(logprobs, "_LIB", NoLibrary())
    monkeypatch.setattr(logprobs, "_raw_stream", lambda index: 0)
    with pytest.raises(Reached):
        logprobs.token_logprobs(Shape(2, 9), Shape(2, dtype=torch.int32))
    with pytest.raises(pkg.HyError, match="2.31"):
        logprobs.token_logprobs(Shape(rows, vocab), Shape(*tokens, dtype=torch.int32))


@pytest.mark.parametrize("per_row", [2 ** 30 + 1, 2 ** 31 - 1])
def test_more_tokens_of_a_row_than_its_threads_can_count(pkg, per_row):
    """A CTA walks a row's tokens in steps of its threads, by a C int that must not pass its largest."""
    import test_logprobs
    lib = importlib.import_module("hy_b200.logprobs")._library()
    assert test_logprobs._call(lib, rows=1, per_row=per_row, top=0) == 4
    assert "2^30" in lib.hy_last_error().decode()


def test_forward_mode_tangents(paged, pkg, no_stream):
    """The calls have no derivative of either mode: a tangent would be lost without a word."""
    import torch.autograd.forward_ad as forward_ad
    rotary = importlib.import_module("hy_b200.rotary")
    c, batch = _cache(paged), _batch(paged)
    q, k, v, lse, weights = torch.zeros(1, 4, 64), torch.zeros(1, 2, 64), torch.zeros(1, 2, 64), torch.zeros(1, 4), torch.zeros(4, 2, 8)
    norm, table, pos = torch.ones(64), torch.ones(5, 64), torch.zeros(1, dtype=torch.int32)

    def turn(*args):
        return rotary.rotation(1, 64, -1, *args, pos, 1e-5, True)

    calls = [
        (lambda q, k, v: c.write_rotated(batch, q, k, v, norm, norm, table, table, pos), (q, k, v)),
        (lambda q: c.attention(batch, q, 0.1), (q,)), (lambda out: c.attention(batch, q, 0.1, out=out), (torch.zeros(1, 4, 64),)),
        (lambda k, v: c.write(batch, k, v), (k, v)), (lambda k, v: c.read(batch, 1, out=(k, v)), (k, v)),
        (lambda q, lse, weights: c.add_weights(batch, q, lse, 0.1, weights), (q, lse, weights)),
        (lambda weights: c.evict(batch, 4, weights), (weights,)), (turn, (norm, norm, table, table)),
    ]
    for call, args in calls:
        for i in range(len(args)):
            with forward_ad.dual_level():
                dual = [forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(args)]
                with pytest.raises(pkg.HyError, match="tangent"):
                    call(*dual)
                with torch.no_grad(), pytest.raises(pkg.HyError, match="tangent"):   # (that turns off the other mode alone)
                    call(*dual)
                if call is not turn:
                    with pytest.raises(Reached):
                        call(*args)


@pytest.mark.parametrize("over", [
    dict(qo=test_paged.FAKE + 256), dict(qo=test_paged.FAKE + 1024), dict(qo=test_paged.FAKE - 768), dict(qo=test_paged.FAKE + 16),
    dict(qo=test_paged.FAKE + 1024 * 99 + 768), dict(qo=2 * test_paged.FAKE - 256), dict(qo=2 * test_paged.FAKE + 256),
    dict(rows=1, qo=test_paged.FAKE + 768, out_strides=(4096, 128)), dict(out_strides=(512, 256), qo=test_paged.FAKE + 256),
])
def test_outputs_over_other_rows_of_the_inputs(pkg, over):
    """Rows of a shared projection: an output that starts some heads or rows further in the same memory."""
    mods = importlib.import_module("hy_b200.rotary"), importlib.import_module("hy_b200.paged")
    f = dict(rows=100)
    f.update(over)
    for rc in test_rotary._calls(mods, test_rotary._rotation(mods[0], positions_dev=None, table_rows=100), **f):
        assert rc == 1
        assert b"overlap" in mods[0]._library().hy_last_error()


@pytest.mark.parametrize("ko", [test_paged.FAKE + 512, 2 * test_paged.FAKE + 256, 3 * test_paged.FAKE + 512, 2 * test_paged.FAKE - 1024 * 9])
def test_keys_over_other_rows(pkg, ko):
    mods = importlib.import_module("hy_b200.rotary"), importlib.import_module("hy_b200.paged")
    calls = test_rotary._calls(mods, test_rotary._rotation(mods[0], positions_dev=None, table_rows=100), rows=100, ko=ko)
    assert next(calls) == 1
    assert b"overlap" in mods[0]._library().hy_last_error()


def test_expanded_logarithms_are_read(paged, no_stream):
    """add_weights only reads lse: one number for all rows or heads is as good as a number for each."""
    import ctypes
    seen = []

    class Library(NoLibrary):
        def hy_paged_add_weights(self, *args):
            at, row, head = args[8:11]
            seen.append([ctypes.c_float.from_address(at + 4 * (i * row + j * head)).value for i in range(3) for j in range(4)])
            assert row > 0 and head > 0   # (the library takes no others)
            return 0

    c, q, weights = _cache(paged), torch.zeros(3, 4, 64), torch.zeros(4, 2, 8)
    c._lib = Library()
    for lse in (torch.arange(4.0).expand(3, 4), torch.arange(3.0)[:, None].expand(3, 4), torch.tensor(5.0).expand(3, 4),
                torch.arange(12.0).view(3, 4), torch.arange(12.0).view(4, 3).t()):
        c.add_weights(_batch(paged), q, lse, 0.1, weights)
        assert seen[-1] == lse.reshape(-1).tolist()


def test_calls_without_rows_and_angles(pkg):
    """No rows, and a table of angles of no rows, whose memory is null: nothing to do."""
    mods = importlib.import_module("hy_b200.rotary"), importlib.import_module("hy_b200.paged")
    turn = test_rotary._rotation(mods[0], cos_dev=None, sin_dev=None, table_rows=0, table_stride=64, positions_dev=None)
    assert list(test_rotary._calls(mods, turn, rows=0, q=None, k=None, qo=None, ko=None)) == [0, 0]
