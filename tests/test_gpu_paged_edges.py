"""The paged KV cache on the GPU at the edges of what its calls allow: repeated and concurrent calls, scales of
either sign and of every size, windows without end, unmapped pages, padded batches, singleton strides."""

import math
import threading

import numpy as np
import pytest
import torch

import paged_reference as R
from test_gpu_paged import BF16, BLOCKS, CHUNKS, DEV, E4M3, F32, INT8, RAGGED, TYPES, Setup, paged  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", [E4M3, INT8])
@pytest.mark.parametrize("rows", [F32, BF16])
def test_few_sequences_repeat_themselves(paged, cache, rows):
    """Queries whose heads differ by many powers of two, a few sequences of one tile: every warp's share of a
    column's largest magnitude counts, whichever warp is first. The same bits every time, and the right ones."""
    st = Setup(paged, cache, [(2100, 1), (33, 1), (700, 2)], kv_heads=4, seed=31)
    st.fill()
    size = 2.0 ** torch.randint(-18, 3, (st.rows, 8, 8, 1), generator=st.gen)
    q = (torch.randn(st.rows, 8, 8, 16, generator=st.gen) * size).view(st.rows, 8, 128).to(rows).to(DEV)
    first = st.check_attention(8, rows, q=q)
    for _ in range(200):
        assert torch.equal(st.cache.attention(st.batch, q, 1.0 / math.sqrt(128)), first)
    st.cache.check()


@pytest.mark.parametrize("page", [16, 24, 64])
@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_scattered_bad_pages_in_chunks(paged, pkg, cache, page):
    """Pages that are none, scattered over the blocks of keys so that every loading warp's bits differ from block to
    block and end inside one: those keys are not seen, the others are, the same bits every time."""
    kv, n = 2011, 150
    st = Setup(paged, cache, [(kv, n)], kv_heads=4, page=page, seed=32)
    st.fill()
    gone = torch.rand(st.table.shape[1], generator=st.gen) < 0.4
    gone[-1] = False
    st.d_table[0, gone.to(DEV)] = -1
    there = np.repeat(~gone.numpy(), page)[:kv]
    sel = torch.from_numpy(np.flatnonzero(there)).to(DEV)
    before = np.cumsum(there)   # keys that are there up to a position
    q = torch.randn(n, 8, 128, generator=st.gen).to(BF16).to(DEV)
    first = st.cache.attention(st.batch, q, 0.1)
    want, mass, reach = R.attention(q.double(), st.keys[0][sel], st.values[0][sel],
                                    [int(before[p]) - 1 for p in range(kv - n, kv)], 0.1)
    tol = R.tolerance(want, mass, reach, kv, 128, BF16, cache in R.LARGEST)
    assert bool(((first.double() - want).abs() <= tol).all())
    for _ in range(30):
        assert torch.equal(st.cache.attention(st.batch, q, 0.1), first)
    with pytest.raises(pkg.HyError, match="page number"):
        st.cache.check()


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 5, 2 ** 30])
@pytest.mark.parametrize("rows,cache", [(F32, F32), (BF16, BF16), (BF16, E4M3)])
def test_window_without_end_and_padding(paged, rows, cache, window):
    """The largest windows and sinks there are, beside rows that lie far before position 0."""
    for seqs in ([(3, 9), (0, 4), (20, 1)], [(100, 150), (0, 70), (300, 40)]):
        for page in (16, 24):
            for sinks in (0, 3, 2 ** 31 - 1):
                st = Setup(paged, cache, seqs, extra_rows=1, page=page, seed=33)
                st.fill()
                st.check_attention(4, rows, window=window, sinks=sinks)


def test_window_and_sinks_of_any_size(paged, pkg):
    """Numbers past 32 bits are no other numbers: they see what any window as long as the cache sees."""
    st = Setup(paged, BF16, [(300, 5), (90, 1)], seed=38)
    st.fill()
    q = torch.randn(st.rows, 4, 128, generator=st.gen).to(BF16).to(DEV)
    want = st.cache.attention(st.batch, q, 0.1)
    for window, sinks in ((2 ** 31, 0), (2 ** 32 + 5, 2), (10 ** 18, 0), (3, 2 ** 32 + 1), (3, 2 ** 31)):
        out = st.check_attention(4, BF16, scale=0.1, window=window, sinks=sinks, q=q)
        assert torch.equal(out, want)
    for over in (dict(window=-2 ** 32 - 5), dict(window=-1), dict(window=3, sinks=-2 ** 32 + 7)):
        with pytest.raises(pkg.HyError, match="negative"):
            st.cache.attention(st.batch, q, 0.1, **over)


@pytest.mark.parametrize("cache", [E4M3, INT8])
@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("seqs", [RAGGED, BLOCKS, CHUNKS], ids=["tokens", "blocks", "chunks"])
def test_scales_of_either_sign(paged, rows, cache, seqs):
    """A caller's own scales may be negative: a value is code * scale, in attention as in what is read back."""
    st = Setup(paged, cache, seqs, seed=34)
    st.fill()
    for which, held in (("k_scale", st.keys), ("v_scale", st.values)):
        scale = getattr(st.cache, which)
        sign = torch.where(torch.rand(scale.shape, generator=st.gen) < 0.3, -1.0, 1.0)
        scale *= sign.to(DEV)
        for s, kv in enumerate(st.kv):
            p = torch.arange(kv)
            held[s] *= sign[st.table[s, p // st.page].long(), :, p % st.page][..., None].double().to(DEV)
    st.check_attention(4, rows)
    st.check_attention(4, rows, window=100, sinks=3)
    for s, kv in enumerate(st.kv):   # and the same values are read back
        if kv:
            one = paged.PagedBatch(torch.tensor([0, kv], dtype=torch.int32, device=DEV), st.d_kv[s:s + 1], st.d_table[s:s + 1], kv)
            k, v = st.cache.read(one, kv, F32)
            assert torch.equal(k, st.keys[s].float()) and torch.equal(v, st.values[s].float())


@pytest.mark.parametrize("cache", [E4M3, INT8])
def test_quantisation_near_ties_at_tiny_scales(paged, cache):
    """Scales from the smallest, 2^-126, up: quotients just below, at and just above a tie, where the remainder of a
    division lies below the smallest normal number."""
    rng = np.random.default_rng(5)
    rows, dim, top = 4096, 128, R.LARGEST[cache]
    grid = R.e4m3_values() if cache == E4M3 else np.arange(128.0)
    mids = (grid[1:] + grid[:-1]) / 2
    amax = (rng.uniform(1.0, 2.0, rows) * top * 2.0 ** rng.integers(-128, -20, rows)).astype(np.float32)
    scale = np.maximum((amax.astype(np.float64) / top).astype(np.float32), np.float32(2.0 ** -126)).astype(np.float64)
    x = (rng.choice(mids, (rows, dim)) * scale[:, None]).astype(np.float32)
    x = np.nextafter(x, rng.choice([-np.inf, 0, np.inf], (rows, dim)).astype(np.float32), dtype=np.float32)
    x *= rng.choice([-1, 1], (rows, dim)).astype(np.float32)
    x = np.clip(x, -amax[:, None], amax[:, None])
    x[:, 0] = amax
    t = torch.from_numpy(x)[:, None, :].contiguous()
    st = Setup(paged, cache, [(rows, rows)], kv_heads=1)
    st.cache.write(st.batch, t.to(DEV), t.to(DEV))
    st.cache.check()
    code, s = R.quantise(t, cache)
    p = torch.arange(rows)
    at = (st.table[0, p // st.page].long(), slice(None), p % st.page)
    for pool, scales in ((st.cache.k, st.cache.k_scale), (st.cache.v, st.cache.v_scale)):
        assert torch.equal(scales.cpu()[at], s.float())
        assert torch.equal(pool.float().cpu()[at].double(), code)


@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 40, 64])
@pytest.mark.parametrize("window,sinks", [(1024, 4), (1000, 0), (300, 17), (7, 33)])
def test_pages_that_no_row_sees_may_be_unmapped(paged, page, window, sinks):
    """Pages wholly behind the window of a sequence's first row and past the sinks are given back (-1): no row sees
    them, nothing is reported and the outputs are right."""
    for rows, cache, seqs in ((BF16, BF16, [(5000, 300), (2000, 40), (64, 64)]), (BF16, E4M3, [(5000, 300), (2011, 17)]),
                              (F32, BF16, [(3000, 20), (1500, 1)]), (BF16, INT8, [(3001, 1), (1200, 1)])):
        st = Setup(paged, cache, seqs, page=page, seed=35)
        st.fill()
        for s, (kv, n) in enumerate(seqs):
            for x in range(-(-kv // page)):
                if x * page >= sinks and (x + 1) * page - 1 <= kv - n - window:
                    st.d_table[s, x] = -1
        st.check_attention(4, rows, window=window, sinks=sinks)


def test_rows_behind_the_last_sequence_cost_no_walk(paged):
    """Padding rows of a call with many sequences are found to be nobody's about as fast as rows are found."""
    n, rows = 60000, 4096
    kv = torch.zeros(n, dtype=torch.int32, device=DEV)
    kv[-1] = rows
    table = torch.arange(rows // 16, dtype=torch.int32, device=DEV)[None].expand(n, -1)
    starts = torch.zeros(n + 1, dtype=torch.int32, device=DEV)
    cache = paged.PagedKVCache.allocate(rows // 16, 1, 16, 64, BF16)
    k = torch.randn(rows, 1, 64, device=DEV)
    padded = paged.PagedBatch(starts.clone(), kv, table, 1)      # every row lies behind the last sequence
    starts[-1] = rows
    owned = paged.PagedBatch(starts, kv, table, rows)            # every row is the last sequence's

    def time(batch):
        best = math.inf
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(4):
                cache.write(batch, k, k)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    time(owned)
    t_owned, t_padded = time(owned), time(padded)
    cache.check()
    assert t_padded < 2.5 * t_owned, (t_padded, t_owned)


@pytest.mark.parametrize("cache", [E4M3, INT8])
def test_many_light_keys_beside_a_heavy_one(paged, cache):
    """A key with nearly all the weight, some 16000 light ones of 2^-20 each that make up a 64th, and among those, one
    in 128, keys of next to no weight whose values' scale is 2^12 times the others'. In the wide kernel one exponent may
    stand for the scales of a block; the light keys' products must not fall below f16's smallest number for it.

    A key's f16 product carries 2^6, is off by half a step, 2^-11 of it, and at least 2^-25; the running maximum is at most
    2^4 above the row's largest weight times scale (T). So a key adds at most 2^(-25 - 6 + 4) |code| T to the error."""
    seqs, kv, n, dim = 160, 16384, 40, 64   # (more items than CTAs, so that a CTA meets the heavy key and the light ones)
    top = R.LARGEST[cache]
    k, v = torch.zeros(kv, 1, dim), torch.zeros(kv, 1, dim)
    k[:, :, 0] = 100.0
    k[0::128, :, 0] = 80.0
    k[1, :, 0] = 120.0
    v[:, :, 0], v[:, :, 1] = top, 0.5 * top
    v[1], v[0::128] = 0.0, 0.0
    v[1, :, 2], v[0::128, :, 3] = top, top * 2.0 ** 12
    st = Setup(paged, cache, [(kv, kv)], kv_heads=1, dim=dim, page=16, seed=36)
    st.cache.write(st.batch, k.to(DEV), v.to(DEV))
    keys, values = st.stand_for(k), st.stand_for(v)
    scales = R.quantise(v, cache)[1][:, 0].to(DEV)
    q = torch.zeros(seqs * n, 1, dim, dtype=BF16, device=DEV)
    q[:, :, 0] = 1.0
    batch = paged.PagedBatch(torch.arange(0, seqs * n + 1, n, dtype=torch.int32, device=DEV),
                             st.d_kv.expand(seqs).contiguous(), st.d_table.expand(seqs, -1), n)
    scale = math.log(2.0)   # a score is a power of two's exponent
    out = st.cache.attention(batch, q, scale).view(seqs, n, 1, dim).double()
    st.cache.check()
    want, mass, _ = R.attention(q[:n].double(), keys, values, list(range(kv - n, kv)), scale)
    weight = torch.exp2(keys[:, 0, 0] - 120.0)
    weight /= weight.sum()
    codes = (values[:, 0] / scales[:, None]).abs().sum(dim=0)
    tol = 2.0 ** -27 * float((weight * scales).max()) * codes + mass * (2.0 ** -11 + 2.0 ** -16) + want.abs() * 2.0 ** -8
    assert float((tol / want.abs())[..., :2].max()) < 2.0 ** -6   # (nothing like the outputs themselves)
    assert bool(((out - want).abs() <= tol).all()), (out[0, 0, 0, :4], want[0, 0, :4])


@pytest.mark.parametrize("cache", TYPES)
@pytest.mark.parametrize("rows", [F32, BF16])
def test_strides_of_single_entries_do_not_matter(paged, cache, rows):
    """One row, one head, one page: what its stride is has no meaning, so it need not be a multiple of 16 bytes."""
    kv, dim, page = 40, 128, 48
    mem = [torch.zeros(page * dim, dtype=torch.uint8 if cache.itemsize == 1 else cache, device=DEV) for _ in range(2)]
    k, v = (torch.as_strided(m, (1, 1, page, dim), (7, 3, dim, 1)).view(cache) for m in mem)
    scales = [torch.full((1, 1, page), math.nan, device=DEV) for _ in range(2)] if cache.itemsize == 1 else (None, None)
    st = Setup(paged, cache, [(kv, 1)], kv_heads=1, dim=dim, page=page, seed=45, spare_pages=0)
    st.cache = paged.PagedKVCache(k, v, *scales)
    st.fill()
    for heads in (1, 4, 40):
        wide = torch.randn(heads * dim, generator=st.gen).to(rows).to(DEV)
        q = torch.as_strided(wide, (1, heads, dim), (5, dim if heads > 1 else 9, 1))
        out = torch.as_strided(torch.full_like(wide, 77.0), (1, heads, dim), (11, dim if heads > 1 else 1, 1))
        st.check_attention(heads, rows, q=q, out=out)
        st.check_attention(heads, rows, window=9, sinks=2, q=q, out=out)
    back = [torch.as_strided(torch.zeros(dim, device=DEV), (1, 1, dim), (3, 5, 1)) for _ in range(2)]
    st.cache.read(st.batch, 1, F32, out=tuple(back))
    st.cache.check()
    assert torch.equal(back[0][0], st.keys[0][-1].float()) and torch.equal(back[1][0], st.values[0][-1].float())


def test_threads_call_at_once(paged):
    """Calls of four threads on streams of their own overlap: the same bits as alone."""
    sts, qs, want = [], [], []
    for i, (cache, seqs) in enumerate([(BF16, RAGGED), (E4M3, CHUNKS), (F32, BLOCKS), (INT8, [(4000, 1)] * 5)]):
        st = Setup(paged, cache, seqs, kv_heads=2, seed=40 + i)
        st.fill()
        sts.append(st)
        qs.append(torch.randn(st.rows, 4, 128, generator=st.gen).to(F32 if cache == F32 else BF16).to(DEV))
        want.append(st.cache.attention(st.batch, qs[-1], 0.1))
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for r in range(50):
                got = sts[i].cache.attention(sts[i].batch, qs[i], 0.1)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(got, want[i]):
                    bad.append((i, r))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for st in sts:
        st.cache.check()
    assert not bad
