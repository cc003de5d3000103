"""Attention weights of cached positions and the eviction by them, on the GPU, against the definitions in 64 bits."""

import importlib
import math

import numpy as np
import pytest
import torch

from paged_reference import LARGEST

pytestmark = pytest.mark.gpu

F32, BF16, E4M3, INT8 = torch.float32, torch.bfloat16, torch.float8_e4m3fn, torch.int8


@pytest.fixture(scope="module")
def paged(pkg):
    return importlib.import_module("hy_b200.paged")


class Setup:
    """A filled cache, a batch over it, rows q and starting weights."""

    def __init__(self, paged, cache, rows, kv_lens, news, heads, kv_heads, dim, page, seed, max_rows=None, scale=None):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.kv, self.new, self.page, self.h = kv_lens, news, page, kv_heads
        width = max(max(-(-max(n, 1) // page) for n in kv_lens), 1)
        self.pages = len(kv_lens) * width + 2
        self.table = torch.randperm(self.pages, generator=gen, device="cuda")[:len(kv_lens) * width].view(len(kv_lens), width).int()
        self.c = paged.PagedKVCache.allocate(self.pages, kv_heads, page, dim, cache)
        for pool, sc in ((self.c.k, self.c.k_scale), (self.c.v, self.c.v_scale)):
            x = torch.randn(pool.shape, generator=gen, device="cuda")
            x *= torch.where(torch.rand(dim, generator=gen, device="cuda") < 0.03, 6.0, 1.0)
            if sc is None:
                pool.copy_(x)
            else:
                s = x.abs().amax(dim=-1) / LARGEST[cache]
                sc.copy_(s)
                y = x / s[..., None]
                pool.copy_(y.round().clamp(-127, 127).to(INT8) if cache == INT8 else y.to(E4M3))
        self.q_start = np.concatenate([[0], np.cumsum(news)]).tolist()
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
        self.batch = paged.PagedBatch(i32(self.q_start), i32(kv_lens), self.table, max_rows=max_rows or max(max(news), 1))
        self.q = torch.randn(self.q_start[-1], heads, dim, generator=gen, device="cuda").to(rows)
        self.scale = scale or 1 / math.sqrt(dim)
        self.weights = torch.rand(self.pages, kv_heads, page, generator=gen, device="cuda")

    def place(self, s):
        j = torch.arange(max(self.kv[s], 0), device="cuda")
        return self.table[s, j // self.page].long(), j % self.page

    def keys(self, s):
        pg, rw = self.place(s)
        k = self.c.k[pg, :, rw].float().double()
        return k if self.c.k_scale is None else k * self.c.k_scale[pg, :, rw].double()[..., None]

    def scores(self, s, causal, window, sinks):
        """(scores, seen, reach) [heads, n, kv] of sequence s."""
        n, kv, k = self.new[s], self.kv[s], self.keys(s)
        q = self.q[self.q_start[s]:self.q_start[s + 1]].double()
        k = k.repeat_interleave(q.shape[1] // self.h, dim=1)
        p = torch.arange(kv - n, kv, device="cuda")[:, None]
        j = torch.arange(kv, device="cuda")[None]
        seen = (j <= p) if causal else (p >= 0).expand(n, kv)
        if window:
            seen = seen & ((p - j < window) | (j < sinks))
        y = torch.einsum("nhd,khd->hnk", q, k) * self.scale
        return y, seen, torch.einsum("nhd,khd->hnk", q.abs(), torch.nan_to_num(k.abs(), 0, 0, 0)) * self.scale

    def lse(self, causal=True, window=0, sinks=0):
        out = torch.zeros(self.q.shape[:2], device="cuda")
        for s in range(len(self.kv)):
            if self.new[s] and self.kv[s] > 0:
                y, seen, _ = self.scores(s, causal, window, sinks)
                out[self.q_start[s]:self.q_start[s + 1]] = torch.logsumexp(y.masked_fill(~seen, -math.inf), dim=-1).T.float()
        return out

    def expect(self, lse, causal=True, window=0, sinks=0):
        """(weights, tolerance). A probability e^d, d = scale q k - lse, is off by: the score's error, products exact to
        2^-21 and the factors' roundings 2^-22, dim of them added up, reach (2^-20 + dim 2^-24); the roundings of d and of
        its multiple, |d| 2^-23; ex2's 2^-22 (and one more of d's). Their sum takes a rounding for each, that with what was
        there one more."""
        want, tol = self.weights.double(), torch.zeros_like(self.weights, dtype=torch.float64)
        dim = self.q.shape[2]
        for s in range(len(self.kv)):
            n, kv = self.new[s], self.kv[s]
            if not n or kv <= 0:
                continue
            y, seen, reach = self.scores(s, causal, window, sinks)
            d = y - lse[self.q_start[s]:self.q_start[s + 1]].T.double()[..., None]
            e = torch.where(seen, d.exp(), 0.0)
            off = torch.where(e > 0, e * (reach * (2.0 ** -20 + dim * 2.0 ** -24) + d.abs() * 2.0 ** -23 + 2.0 ** -21), 0.0)
            total = e.view(self.h, -1, kv).sum(dim=1).T
            pg, rw = self.place(s)
            old = want[pg, :, rw]
            old[torch.arange(kv, device="cuda") >= kv - n] = 0
            want[pg, :, rw] = old + total
            tol[pg, :, rw] = off.view(self.h, -1, kv).sum(dim=1).T + total * (n * len(e) // self.h) * 2.0 ** -24 + (old + total) * 2.0 ** -23
        return want, tol

    def check(self, **view):
        lse = self.lse(**view)
        want, tol = self.expect(lse, **view)
        self.c.add_weights(self.batch, self.q, lse, self.scale, self.weights, **view)
        self.c.check()
        off = (self.weights.double() - want).abs()
        bad = ~(off <= tol)
        assert not bad.any(), (int(bad.sum()), float((off / tol.clamp_min(1e-30))[bad].max()))
        assert torch.equal(self.weights[tol == 0].double(), want[tol == 0])   # nobody's rows, and positions unseen


CACHES = [F32, BF16, E4M3, INT8]
SIZES = [   # kv lengths, new rows, heads, kv heads, dim, page
    ([1], [1], 1, 1, 64, 16), ([33], [1], 2, 1, 128, 16), ([200, 1, 77], [1, 1, 1], 8, 2, 64, 24),
    ([130, 64, 999], [1, 2, 1], 12, 3, 128, 7), ([513, 40, 300], [4, 4, 3], 4, 2, 128, 64),
    ([300, 17, 0, 90], [16, 16, 0, 9], 4, 2, 128, 16), ([2100], [1], 16, 8, 128, 100), ([700, 350], [300, 350], 2, 2, 64, 32),
    ([90], [90], 8, 1, 128, 1),
]


@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("kv,new,heads,kv_heads,dim,page", SIZES)
def test_sizes(paged, cache, rows, kv, new, heads, kv_heads, dim, page):
    Setup(paged, cache, rows, kv, new, heads, kv_heads, dim, page, 1 + sum(kv)).check()


@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 4), (100, 33), (1000, 1), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("kv,new", [([400, 30, 1, 700], [1, 1, 1, 1]), ([500, 130], [37, 130])])
def test_windows(paged, cache, rows, kv, new, window, sinks):
    Setup(paged, cache, rows, kv, new, 4, 2, 128, 16, 5).check(window=window, sinks=sinks)


@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("new", [[1, 2], [16, 40]])
def test_every_key_seen(paged, cache, rows, new):
    Setup(paged, cache, rows, [150, 260], new, 4, 2, 64, 32, 6).check(causal=False)


@pytest.mark.parametrize("cache,rows", [(F32, F32), (BF16, BF16), (E4M3, F32), (INT8, BF16)])
@pytest.mark.parametrize("max_rows", [1, 3, 1000])
def test_another_max_rows_is_as_right(paged, cache, rows, max_rows):
    """Sequences of more (and fewer) rows than the call is laid out for."""
    Setup(paged, cache, rows, [220, 90, 400], [1, 50, 18], 6, 2, 128, 16, 7, max_rows=max_rows).check()


@pytest.mark.parametrize("cache,rows", [(F32, F32), (F32, BF16), (BF16, BF16), (BF16, F32), (E4M3, BF16), (INT8, F32)])
@pytest.mark.parametrize("new", [[1, 1, 1], [20, 20, 5]])
def test_padding_rows_and_long_batches(paged, cache, rows, new):
    s = Setup(paged, cache, rows, [12, 3, 5], [n + 7 for n in new], 4, 2, 64, 4, 8)   # more rows than positions
    s.check()
    many = Setup(paged, cache, rows, [5 + 7 * i % 90 for i in range(70)], [1] * 70, 4, 2, 64, 16, 9)
    many.check()


@pytest.mark.parametrize("cache,rows", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("new", [1, 5, 40])
def test_what_rows_do_not_see_does_not_reach_them(paged, cache, rows, new):
    """Infinities and NaN in keys outside the window, behind a row and in rows of the last page past the end."""
    s = Setup(paged, cache, rows, [300], [new], 4, 2, 128, 16, 10)
    pg, rw = s.place(0)
    s.c.k[pg[20:100], :, rw[20:100]] = math.nan
    s.c.k[pg[100:110], :, rw[100:110]] = math.inf
    s.c.k[pg[-1], :, int(rw[-1]) + 1:] = math.nan
    s.check(window=150, sinks=4)


@pytest.mark.parametrize("cache", [E4M3, INT8])
@pytest.mark.parametrize("new", [1, 40])
def test_a_bad_scale_stays_with_its_key(paged, cache, new):
    s = Setup(paged, cache, BF16, [200], [new], 4, 2, 128, 16, 11)
    pg, rw = s.place(0)
    lse = s.lse()
    want, tol = s.expect(lse)
    s.c.k_scale[pg[50], 1, rw[50]] = math.nan
    s.c.add_weights(s.batch, s.q, lse, s.scale, s.weights)
    got = s.weights.double()
    assert torch.isnan(got[pg[50], 1, rw[50]])
    want[pg[50], 1, rw[50]] = got[pg[50], 1, rw[50]] = 0
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("rows,cache", [(F32, F32), (BF16, E4M3), (BF16, BF16)])
@pytest.mark.parametrize("new", [1, 40])
def test_bad_pages_and_lengths(paged, pkg, rows, cache, new):
    s = Setup(paged, cache, rows, [100, 100, 100], [new] * 3, 4, 2, 64, 16, 12)
    lse = s.lse()
    want, tol = s.expect(lse)
    before = s.weights.clone()
    lost = s.place(0)[0][32:48]
    s.batch.block_table[0, 2] = -5
    s.batch.kv_len[1] = 10 ** 6
    s.c.add_weights(s.batch, s.q, lse, s.scale, s.weights)
    with pytest.raises(pkg.HyError, match="page number.*kv_len"):
        s.c.check()
    want[lost] = before[lost].double()
    own = s.table[1].long()
    want[own] = before[own].double()
    tol[own] = tol[lost] = 0
    assert ((s.weights.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("cache,rows,new", [(BF16, BF16, 1), (E4M3, BF16, 1), (F32, F32, 1), (BF16, BF16, 60)])
def test_the_same_bits_again_captured_and_on_another_stream(paged, cache, rows, new):
    s = Setup(paged, cache, rows, [900, 500], [new, new], 4, 2, 128, 16, 13)
    lse, start = s.lse(), s.weights.clone()
    s.c.add_weights(s.batch, s.q, lse, s.scale, s.weights)
    first = s.weights.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        s.c.add_weights(s.batch, s.q, lse, s.scale, s.weights)
    for _ in range(3):
        s.weights.copy_(start)
        graph.replay()
        assert torch.equal(s.weights, first)


def test_other_strides(paged):
    """Rows as views of a projection, heads before rows, weights and lse in other orders: the same bits."""
    s = Setup(paged, BF16, BF16, [300, 200], [3, 2], 4, 2, 128, 16, 14)
    lse = s.lse()
    held = torch.zeros(s.page, s.h, s.pages, device="cuda").permute(2, 1, 0)
    held.copy_(s.weights)
    s.c.add_weights(s.batch, s.q, lse, s.scale, s.weights)
    wide = torch.zeros(5, 7, 136, dtype=BF16, device="cuda")[:, 2:6, :128]
    wide.copy_(s.q)
    turned = torch.empty(4, 5, device="cuda").t()
    turned.copy_(lse)
    s.c.add_weights(s.batch, wide, turned, s.scale, held)
    assert torch.equal(held, s.weights)


# ---------------------------------------------------------------------------
# The logarithms of the sums that the attention leaves.
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("kv,new,heads,kv_heads,dim,page", SIZES + [([3000, 5000], [1, 1], 4, 2, 128, 16), ([2000], [200], 4, 1, 64, 16)])
def test_lse_of_the_attention(paged, cache, rows, kv, new, heads, kv_heads, dim, page):
    """lse is off by the scores' errors (reach (2^-20 + dim 2^-24)), the exponentials' (2^-20), their sum's (a rounding of
    2^-24 a key at most) and its own; the output is the same with and without it."""
    s = Setup(paged, cache, rows, kv, new, heads, kv_heads, dim, page, 2 + sum(kv))
    for view in (dict(), dict(window=50, sinks=3)):
        out, lse = s.c.attention(s.batch, s.q, s.scale, return_lse=True, **view)
        assert torch.equal(out, s.c.attention(s.batch, s.q, s.scale, **view))
        for i in range(len(kv)):
            if not new[i]:
                continue
            y, seen, reach = s.scores(i, True, view.get("window", 0), view.get("sinks", 0))
            want = torch.logsumexp(y.masked_fill(~seen, -math.inf), dim=-1).T
            far = torch.where(seen, reach, 0.0).amax(dim=-1).T
            tol = far * (2.0 ** -20 + dim * 2.0 ** -24) + 2.0 ** -20 + kv[i] * 2.0 ** -24 + want.abs() * 2.0 ** -22
            got = lse[s.q_start[i]:s.q_start[i + 1]].double()
            assert ((got - want).abs() <= tol).all()


def test_lse_of_rows_that_see_nothing(paged):
    s = Setup(paged, BF16, BF16, [2, 40], [5, 3], 4, 2, 64, 16, 3)
    out, lse = s.c.attention(s.batch, s.q, s.scale, return_lse=True)
    assert (lse[:3] == -math.inf).all() and torch.isfinite(lse[3:]).all() and (out[:3] == 0).all()


# ---------------------------------------------------------------------------
# Eviction.
# ---------------------------------------------------------------------------
def _evicted(s, keep, first, recent):
    """What evict leaves: the state's tensors, kept positions, lengths."""
    held = [t.clone() for t in (s.c.k, s.c.v, s.c.k_scale, s.c.v_scale, s.weights) if t is not None]
    raw = [t.view(torch.uint8) if t.element_size() == 1 else t for t in held]
    kept = torch.full((len(s.kv), s.h, keep), -1, dtype=torch.int32)
    for i, kv in enumerate(s.kv):
        pg, rw = s.place(i)
        for h in range(s.h):
            w = s.weights[pg, h, rw].double().cpu().numpy()
            w = np.where(np.isnan(w), -np.inf, w) + 0.0
            order = np.lexsort((np.arange(kv), np.isnan(s.weights[pg, h, rw].cpu().numpy()), -w))
            safe = [j for j in range(kv) if j < first or j >= kv - recent]
            stay = list(range(kv)) if kv <= keep else sorted(safe + [j for j in order if first <= j < kv - recent][:keep - len(safe)])
            kept[i, h, :len(stay)] = torch.tensor(stay, dtype=torch.int32)
            if kv > keep:
                at = torch.tensor(stay, device="cuda")
                for t in raw:
                    t[pg[:keep], h, rw[:keep]] = t[pg[at], h, rw[at]]
    return held, kept, [min(kv, keep) for kv in s.kv]


def _check_evict(s, keep, first=0, recent=0):
    want, kept, lengths = _evicted(s, keep, first, recent)
    got = s.c.evict(s.batch, keep, s.weights, recent=recent, first=first)
    s.c.check()
    assert torch.equal(got.cpu(), kept)
    assert s.batch.kv_len.tolist() == lengths
    have = [t for t in (s.c.k, s.c.v, s.c.k_scale, s.c.v_scale, s.weights) if t is not None]
    for a, b in zip(have, want):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("kv,kv_heads,dim,page,keep,first,recent", [
    ([2], 1, 64, 16, 1, 0, 0), ([5, 3, 4], 2, 64, 2, 3, 1, 1), ([700, 100, 64], 3, 128, 24, 64, 4, 16),
    ([1100] * 20 + [900], 8, 128, 16, 1024, 4, 256), ([9000, 200], 2, 64, 100, 5000, 0, 7), ([513], 16, 128, 7, 512, 0, 512),
    ([20000], 1, 128, 64, 300, 1, 0), ([600], 8, 64, 64, 500, 500, 0), ([40000, 33000], 1, 64, 64, 900, 1, 5)])
def test_evict(paged, cache, kv, kv_heads, dim, page, keep, first, recent):
    s = Setup(paged, cache, BF16, kv, [1] * len(kv), kv_heads, kv_heads, dim, page, keep)
    _check_evict(s, keep, first, recent)


@pytest.mark.parametrize("kv", [[100, 40], [10000]])
def test_equal_and_odd_weights(paged, kv):
    """Ties stay from the lowest position on; zeros of both signs are equal; NaN and negative ones go first."""
    for kind in range(5):
        s = Setup(paged, F32, F32, kv, [1] * len(kv), 2, 2, 64, 16, 20 + kind)
        w = s.weights
        if kind == 0:
            w.zero_()
        elif kind == 1:
            w.copy_((w * 4).floor())
        elif kind == 2:
            w.copy_(torch.where(w < 0.5, 0.0, -0.0))
        elif kind == 3:
            w.copy_(torch.where(w < 0.7, math.nan, w - 0.8))
        else:
            w.copy_(torch.where(w < 0.3, math.inf, torch.where(w < 0.6, -math.inf, w)))
        _check_evict(s, kv[0] // 2 + 1, 2, 3)


@pytest.mark.parametrize("rising", [True, False])
def test_runs_that_stay_and_runs_that_move(paged, rising):
    """The first positions go, so that everything moves; or the last ones, so that nothing does."""
    s = Setup(paged, BF16, BF16, [3000], [1], 4, 4, 128, 16, 30)
    pg, rw = s.place(0)
    order = torch.arange(3000, device="cuda").float()
    s.weights[pg, :, rw] = (order if rising else -order)[:, None]
    _check_evict(s, 2000)


def test_sequences_that_do_not_hold_are_left(paged, pkg):
    s = Setup(paged, BF16, BF16, [100, 100, 100], [1, 1, 1], 2, 2, 64, 16, 31)
    held = s.c.k.clone()
    s.batch.block_table[0, 3] = 10 ** 6
    s.batch.kv_len[1] = -4
    kept = s.c.evict(s.batch, 50, s.weights)
    with pytest.raises(pkg.HyError, match="page number.*kv_len"):
        s.c.check()
    assert (kept[:2] == -1).all() and s.batch.kv_len.tolist() == [100, -4, 50]
    others = torch.ones(s.pages, dtype=torch.bool)
    others[s.table[2].cpu().long()] = False
    assert torch.equal(s.c.k[others], held[others])


def test_layers_that_share_a_batch(paged):
    """Every layer's cache is cut at the same lengths, which change with the last."""
    layers = [Setup(paged, BF16, BF16, [400, 90, 250], [1] * 3, 2, 2, 64, 16, 50 + i) for i in range(3)]
    batch = layers[0].batch
    for s in layers:
        s.table, s.batch = layers[0].table, batch
    for s in layers:
        want, kept, lengths = _evicted(s, 100, 2, 10)
        last = s is layers[-1]
        assert torch.equal(s.c.evict(batch, 100, s.weights, recent=10, first=2, set_lengths=last).cpu(), kept)
        assert batch.kv_len.tolist() == (lengths if last else s.kv)
        assert all(torch.equal(a, b) for a, b in zip((s.c.k, s.c.v, s.weights), want))


def test_other_layouts_and_capture(paged):
    """Rows before heads in a page, weights in another order; a captured call follows what it finds."""
    s = Setup(paged, BF16, BF16, [400, 90], [1, 1], 4, 4, 64, 16, 32)
    want, kept, lengths = _evicted(s, 200, 1, 5)
    k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (s.c.k, s.c.v))
    w = s.weights.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    other = paged.PagedKVCache(k, v)
    start = [t.clone() for t in (k, v, w, s.batch.kv_len)]
    out = torch.empty(2, 4, 200, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        other.evict(s.batch, 200, w, recent=5, first=1, kept=out)
    for _ in range(2):
        for t, b in zip((k, v, w, s.batch.kv_len), start):
            t.copy_(b)
        graph.replay()
        assert torch.equal(out.cpu(), kept) and s.batch.kv_len.tolist() == lengths
        assert all(torch.equal(a, b) for a, b in zip((k, v, w), want))


def test_refusals_of_tensors(paged, pkg):
    s = Setup(paged, BF16, BF16, [40, 30], [2, 1], 4, 2, 64, 16, 33)
    lse = s.lse()
    bad = [(s.q.half(), lse, s.weights), (s.q[..., :32], lse, s.weights), (s.q, lse.double(), s.weights), (s.q, lse[:2], s.weights),
           (s.q, lse.cpu(), s.weights), (s.q, lse, s.weights.double()), (s.q, lse, s.weights[1:]), (s.q, lse, s.weights.cpu()),
           (s.q.detach().requires_grad_(), lse, s.weights)]
    for q, l, w in bad:
        with pytest.raises(pkg.HyError):
            s.c.add_weights(s.batch, q, l, s.scale, w)
    for kw in (dict(keep=0), dict(keep=4, recent=5), dict(keep=4, first=-1)):
        with pytest.raises(pkg.HyError):
            s.c.evict(s.batch, kw.pop("keep"), s.weights, **kw)
    for kept in (torch.empty(2, 2, 5, dtype=torch.int32, device="cuda"), torch.empty(2, 2, 4, device="cuda"),
                 torch.empty(2, 2, 4, dtype=torch.int32)):
        with pytest.raises(pkg.HyError):
            s.c.evict(s.batch, 4, s.weights, kept=kept)
