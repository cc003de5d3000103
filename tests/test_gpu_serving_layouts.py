"""The calls around the paged cache and behind the LM head as their documentation allows them and the tests of each do not make
them: other strides in every kernel, pages that nobody may look up, two streams at once, the same thing twice."""

import importlib
import math

import pytest
import torch

import test_gpu_logprobs
from test_gpu_paged_weights import BF16, E4M3, F32, INT8, Setup, paged   # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def _layouts(q):
    """The same rows in other places: part of a projection (rows a whole number of heads apart, and not), heads apart, heads
    before rows."""
    n, h, d = q.shape
    for shape, place in (((n, (h + 3) * d), lambda t: t[:, 2 * d:(2 + h) * d].view(n, h, d)),
                         ((n, h * d + 40), lambda t: t[:, 16:16 + h * d].view(n, h, d)),
                         ((n, h + 1, d + 8), lambda t: t[:, 1:, :d]),
                         ((h, n + 1, d), lambda t: t[:, 1:].transpose(0, 1))):
        x = place(torch.full(shape, math.nan, dtype=q.dtype, device="cuda"))
        x.copy_(q)
        yield x


@pytest.mark.parametrize("cache,rows,heads,new", [
    (BF16, BF16, 16, 70), (BF16, BF16, 24, 70), (E4M3, BF16, 16, 70), (INT8, BF16, 24, 50), (F32, F32, 16, 30), (BF16, F32, 16, 30),
    (E4M3, F32, 24, 30), (F32, BF16, 16, 1), (INT8, BF16, 16, 1), (BF16, BF16, 8, 20)])
def test_rows_and_numbers_of_other_strides(paged, cache, rows, heads, new):   # noqa: F811
    """Each kernel of the weights, and the attention's logarithms: the same bits."""
    s = Setup(paged, cache, rows, [900, 333, 1200], [new, new - new // 3, new], heads, 8, 128, 16, 5)
    start = s.weights.clone()
    out, lse = s.c.attention(s.batch, s.q, s.scale, return_lse=True)
    s.c.add_weights(s.batch, s.q, lse, s.scale, s.weights)
    want, turned = s.weights.clone(), torch.empty(heads, len(s.q) + 3, device="cuda").t()[3:]
    for q in _layouts(s.q):
        got, l = s.c.attention(s.batch, q, s.scale, return_lse=True)
        assert torch.equal(got, out) and torch.equal(l, lse)
        turned.copy_(l)
        for order in ((0, 1, 2), (2, 1, 0), (1, 2, 0)):
            held = torch.empty([start.shape[i] for i in order], device="cuda")
            w = held.permute([order.index(i) for i in range(3)])
            w.copy_(start)
            s.c.add_weights(s.batch, q, turned, s.scale, w)
            assert torch.equal(w, want)
    s.c.check()


@pytest.mark.parametrize("cache,rows", [(F32, F32), (BF16, BF16), (E4M3, BF16), (INT8, F32)])
@pytest.mark.parametrize("new", [1, 12, 90])
def test_pages_that_no_row_sees_may_be_missing(paged, cache, rows, new):   # noqa: F811
    """Behind the window and past the sinks, and after the last position."""
    view = dict(window=300, sinks=20)
    s = Setup(paged, cache, rows, [2000, 1500], [new, new], 16, 8, 128, 16, 6)
    lse = s.lse(**view)
    want, tol = s.expect(lse, **view)
    for i, kv in enumerate(s.kv):
        s.batch.block_table[i, 2:(kv - new - 300) // 16] = -1
        s.batch.block_table[i, -(-kv // 16):] = 10 ** 9
    s.c.add_weights(s.batch, s.q, lse, s.scale, s.weights, **view)
    s.c.check()
    assert ((s.weights.double() - want).abs() <= tol).all()


def test_eviction_looks_up_no_page_behind_the_end(paged):   # noqa: F811
    s = Setup(paged, BF16, BF16, [100, 900], [1, 1], 2, 2, 64, 16, 7)
    s.batch.block_table[0, 7:] = -3
    kept = s.c.evict(s.batch, 50, s.weights, first=1, recent=4)
    s.c.check()
    assert s.batch.kv_len.tolist() == [50, 50] and (kept >= 0).all()
    again = s.c.evict(s.batch, 50, s.weights, first=1, recent=4)   # (nothing is left to go)
    assert torch.equal(again, torch.arange(50, device="cuda").int().expand(2, 2, 50))


def test_two_streams_at_once(paged):   # noqa: F811
    """Two caches, each on a stream of its own, many calls of every kind under way together: as one after another."""
    logprobs, rotary = (importlib.import_module("hy_b200." + m) for m in ("logprobs", "rotary"))

    def steps(s, logits, tokens, n):
        w = torch.ones(128, device="cuda")
        cos, sin = torch.full((2048, 128), 0.6, device="cuda"), torch.full((2048, 128), 0.8, device="cuda")
        got = []
        for _ in range(n):
            q, _ = rotary.norm_rotate(s.q, s.q[:, :8], w, w, cos, sin)
            out, lse = s.c.attention(s.batch, q, s.scale, return_lse=True)
            s.c.add_weights(s.batch, q, lse, s.scale, s.weights)
            got += [out, lse, *logprobs.token_logprobs(logits, tokens, 4)]
        got.append(s.c.evict(s.batch, 400, s.weights, recent=50))
        return got + [s.weights, s.c.k, s.batch.kv_len]

    def inputs(seed):
        s = Setup(paged, BF16, BF16, [1500, 700, 2000], [(1, 90)[seed % 2]] * 3, 16, 8, 128, 16, seed)
        logits = torch.randn(40, 50000, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
        return s, logits, torch.arange(40, device="cuda").int()

    want = [steps(*inputs(seed), 6) for seed in (1, 2)]
    held = [inputs(seed) for seed in (1, 2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for x, stream in zip(held, streams):
        with torch.cuda.stream(stream):
            got.append(steps(*x, 6))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_that_are_one_row(pkg, dtype):
    """Expanded logits and heads, positions and tokens given more than once."""
    logprobs, rotary = (importlib.import_module("hy_b200." + m) for m in ("logprobs", "rotary"))
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(1, 9001, generator=gen, device="cuda").to(dtype)
    for rows in (7, 700):
        tokens = torch.full((rows, 5), 17, dtype=torch.int32, device="cuda")
        got = logprobs.token_logprobs(x.expand(rows, -1), tokens, 6)
        # (the rows of a copy start elsewhere in 16 bytes, by which the sums are grouped: the bits are those of one address)
        test_gpu_logprobs._check(got, x.expand(rows, -1), tokens, 6)
        assert all((t == t[:1]).all() for t in got) and (got.logprob == got.logprob[0, 0]).all()
        q = torch.randn(1, 1, 64, generator=gen, device="cuda").to(dtype)
        w, table = torch.rand(64, generator=gen, device="cuda"), torch.randn(3, 64, generator=gen, device="cuda")
        pos = torch.full((rows,), 2, dtype=torch.int32, device="cuda")
        a, b = rotary.norm_rotate(q.expand(rows, 4, 64), q.expand(rows, 2, 64), w, w, table, table[:1].expand(3, 64).contiguous(), pos)
        assert (a == a[0, 0]).all() and (b == a[0, 0]).all()
