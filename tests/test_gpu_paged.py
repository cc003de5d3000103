"""The paged KV cache on the GPU: rows written (quantised) and read back, attention over the pages, windows with
sinks, against plain 64-bit forms. Codes and scales are exact; tolerances of the attention are derived in
paged_reference.tolerance."""

import math

import numpy as np
import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu

F32, BF16, E4M3, INT8 = torch.float32, torch.bfloat16, torch.float8_e4m3fn, torch.int8
TYPES = [F32, BF16, E4M3, INT8]
DEV = "cuda"


@pytest.fixture(scope="module")
def paged(pkg):
    import importlib
    return importlib.import_module("hy_b200.paged")


class Setup:
    """Sequences of (kv_len, rows) in a shuffled pool whose unused rows hold NaN (E4M3 / INT8: NaN scales)."""

    def __init__(self, paged, dtype, seqs, kv_heads=2, dim=128, page=16, seed=0, extra_rows=0, layout="phrd",
                 spare_pages=3):
        self.paged, self.dtype, self.page, self.kv_heads, self.dim = paged, dtype, page, kv_heads, dim
        self.gen = torch.Generator().manual_seed(seed)
        need = [-(-kv // page) for kv, _ in seqs]
        pages = sum(need) + spare_pages
        order = torch.randperm(pages, generator=self.gen).int()
        width = max(need + [1])
        table = torch.full((len(seqs), width), -7, dtype=torch.int32)   # unused entries are no pages
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n]
            at += n
        self.kv = [kv for kv, _ in seqs]
        self.n = [n for _, n in seqs]
        self.starts = np.concatenate([[0], np.cumsum(self.n)]).astype(np.int64).tolist()
        self.rows = self.starts[-1] + extra_rows
        self.table = table
        perm = {"phrd": (0, 1, 2, 3), "prhd": (0, 2, 1, 3)}[layout]   # memory order of (page, head, row, dim)
        shape = (pages, kv_heads, page, dim)
        mem = [shape[i] for i in perm]
        back = [perm.index(i) for i in range(4)]

        def pool():
            if dtype.itemsize == 1:
                return torch.zeros(mem, dtype=torch.uint8, device=DEV).view(dtype).permute(back)
            return torch.full(mem, math.nan, dtype=dtype, device=DEV).permute(back)

        k, v = pool(), pool()
        scales = [torch.full(shape[:3], math.nan, device=DEV) for _ in range(2)] if dtype.itemsize == 1 else [None] * 2
        self.cache = paged.PagedKVCache(k, v, *scales)
        self.d_starts = torch.tensor(self.starts, dtype=torch.int32, device=DEV)
        self.d_kv = torch.tensor(self.kv, dtype=torch.int32, device=DEV)
        self.d_table = table.to(DEV)
        self.batch = paged.PagedBatch(self.d_starts, self.d_kv, self.d_table, max(self.n + [0]))

    def fill(self, spread=1.0, octaves=0):
        """Writes every position of every sequence (values times a power of two of the position, up to 2^octaves
        either way); keeps what the cache then stands for in 64 bits."""
        total = sum(self.kv)
        k = torch.randn(total, self.kv_heads, self.dim, generator=self.gen) * spread
        v = torch.randn(total, self.kv_heads, self.dim, generator=self.gen)
        if octaves:
            v = v * 2.0 ** torch.randint(-octaves, octaves + 1, (total, 1, 1), generator=self.gen)
        starts = torch.tensor(np.concatenate([[0], np.cumsum(self.kv)]), dtype=torch.int32, device=DEV)
        whole = self.paged.PagedBatch(starts, self.d_kv, self.d_table, max(self.kv + [0]))
        self.cache.write(whole, k.to(DEV), v.to(DEV))
        self.cache.check()
        self.keys, self.values = ([x for x in self.stand_for(t).split(self.kv)] for t in (k, v))

    def stand_for(self, x):
        if self.dtype in R.LARGEST:
            code, scale = R.quantise(x, self.dtype)
            return (code * scale[..., None]).to(DEV)
        return x.to(self.dtype).double().to(DEV)

    def check_attention(self, q_heads, q_dtype, scale=None, causal=True, window=0, sinks=0, q=None, out=None):
        scale = scale if scale is not None else 1.0 / math.sqrt(self.dim)
        if q is None:
            q = torch.randn(self.rows, q_heads, self.dim, generator=self.gen).to(q_dtype).to(DEV)
        if out is None:
            out = torch.full_like(q, 77.0)
        got = self.cache.attention(self.batch, q, scale, causal=causal, window=window, sinks=sinks, out=out)
        self.cache.check()
        assert got is out
        self.compare(q, out, scale, causal, window, sinks)
        return out

    def compare(self, q, out, scale, causal=True, window=0, sinks=0):
        for s, (kv, n) in enumerate(zip(self.kv, self.n)):
            r0, r1 = self.starts[s], self.starts[s + 1]
            if n == 0:
                continue
            pos = list(range(kv - n, kv))
            for a in range(0, n, 256):
                b = min(n, a + 256)
                want, mass, reach = R.attention(q[r0 + a:r0 + b].double(), self.keys[s], self.values[s], pos[a:b],
                                                scale, causal, window, sinks)
                have = out[r0 + a:r0 + b].double()
                tol = R.tolerance(want, mass, reach, kv, self.dim, q.dtype, self.dtype in R.LARGEST)
                off = torch.nan_to_num((have - want).abs() - tol, nan=0.0)
                assert torch.equal(torch.isnan(have), torch.isnan(want)), s
                assert float(off.max()) <= 0, (s, float((have - want).abs().max()), float(tol.min()))
        if self.rows > self.starts[-1]:
            assert bool((out[self.starts[-1]:] == 77.0).all())


# ---------------------------------------------------------------------------
# Write and read back.
# ---------------------------------------------------------------------------
def _pool_positions(st, which):
    """Every row's (page, row) contents after a write: [rows, heads, dim]."""
    out = []
    for pos in R.positions(st.starts, st.kv, st.rows):
        if pos is None or pos[1] < 0:
            out.append(None)
            continue
        s, p = pos
        out.append((int(st.table[s, p // st.page]), p % st.page))
    return out


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("cache", TYPES)
@pytest.mark.parametrize("rows", [F32, BF16])
def test_write_is_exact_and_reads_back(paged, cache, rows, dim):
    st = Setup(paged, cache, [(37, 37), (0, 0), (50, 3), (1, 1), (2, 5)], kv_heads=3, dim=dim, page=24, extra_rows=2)
    k, v = (torch.randn(st.rows, 3, dim, generator=st.gen).to(rows) for _ in range(2))
    k[0, 0] = 0                                     # a row of zeros
    k[1, 1] = torch.randn(dim, generator=st.gen).to(rows) * 1e-38   # below the smallest scale
    k[2, 2] = 2.0 ** torch.randint(-30, 30, (dim,), generator=st.gen).to(rows)   # far below the largest: subnormal codes
    k[3, 0] = torch.arange(dim).to(rows) * 0.5      # ties
    k[4, 1, 5] = math.inf
    v[4, 2, 6] = math.nan
    before = [t.clone() for t in (st.cache.k.view(torch.uint8) if cache.itemsize == 1 else st.cache.k,)]
    st.cache.write(st.batch, k.to(DEV), v.to(DEV))
    got = st.cache.read(st.batch, st.rows, rows, out=tuple(torch.full((st.rows, 3, dim), 55.0, dtype=rows, device=DEV)
                                                            for _ in range(2)))
    st.cache.check()
    places = _pool_positions(st, "k")
    assert places.count(None) == 3 + 2   # two past the last sequence, three before position 0
    for x, pool, scales, back in ((k, st.cache.k, st.cache.k_scale, got[0]), (v, st.cache.v, st.cache.v_scale, got[1])):
        if cache in R.LARGEST:
            code, scale = R.quantise(x, cache)
            want = (code.float() * scale.float()[..., None])
        else:
            want = x.to(cache).float()
        for r, at in enumerate(places):
            if at is None:
                assert bool((back[r] == 55.0).all())
                continue
            if cache in R.LARGEST:
                held = pool[at[0], :, at[1]].float().cpu().double()
                assert torch.equal(held, code[r]), r
                assert np.array_equal(scales[at[0], :, at[1]].cpu().numpy(), scale[r].float().numpy(), equal_nan=True)
            else:
                assert torch.equal(pool[at[0], :, at[1]].float().cpu().nan_to_num(9), want[r].nan_to_num(9))
            assert torch.equal(back[r].float().cpu().nan_to_num(9), want[r].to(rows).float().nan_to_num(9)), r
    # Nothing else was written.
    touched = torch.zeros(st.cache.k.shape[0], st.page, dtype=torch.bool)
    for at in places:
        if at is not None:
            touched[at] = True
    now = st.cache.k.view(torch.uint8) if cache.itemsize == 1 else st.cache.k
    same = (now.cpu().float().nan_to_num(9) == before[0].cpu().float().nan_to_num(9)).all(dim=3).all(dim=1)
    assert bool(same[~touched].all())


@pytest.mark.parametrize("cache", [E4M3, INT8])
def test_quantisation_near_ties(paged, cache):
    """Quotients next to a tie: x just below, at and just above (n + 1/2) scale for scales of every kind, where the
    product with a rounded reciprocal falls on either side."""
    rng = np.random.default_rng(3)
    rows, dim, top = 512, 128, R.LARGEST[cache]
    grid = R.e4m3_values() if cache == E4M3 else np.arange(128.0)
    mids = (grid[1:] + grid[:-1]) / 2
    amax = rng.uniform(0.5, 2.0, rows).astype(np.float32) * np.float32(2.0) ** rng.integers(-20, 20, rows)
    amax = amax.astype(np.float32)
    scale = (amax.astype(np.float64) / top).astype(np.float32).astype(np.float64)
    x = (rng.choice(mids, (rows, dim)) * scale[:, None]).astype(np.float32)
    x = np.nextafter(x, rng.choice([-np.inf, 0, np.inf], (rows, dim)).astype(np.float32) * 1, dtype=np.float32)
    x *= rng.choice([-1, 1], (rows, dim)).astype(np.float32)
    x = np.clip(x, -amax[:, None], amax[:, None])
    x[:, 0] = amax
    t = torch.from_numpy(x)[:, None, :].contiguous()
    st = Setup(paged, cache, [(rows, rows)], kv_heads=1)
    st.cache.write(st.batch, t.to(DEV), t.to(DEV))
    k, _ = st.cache.read(st.batch, rows, F32)
    code, s = R.quantise(t, cache)
    assert torch.equal(k.cpu(), code.float() * s.float()[..., None])


@pytest.mark.parametrize("layout", ["phrd", "prhd"])
def test_write_and_read_strided_rows(paged, layout):
    """Rows inside a wider projection buffer [rows, q | k | v], pages in either order, the pools of k and v one tensor."""
    st = Setup(paged, BF16, [(70, 70), (9, 4)], kv_heads=8, layout=layout)
    qkv = torch.randn(st.rows, 32, 128, generator=st.gen).to(DEV)
    k, v = qkv[:, 16:24], qkv[:, 24:]
    st.cache.write(st.batch, k, v)
    out = torch.full((st.rows, 32, 128), 5.0, device=DEV)
    st.cache.read(st.batch, st.rows, F32, out=(out[:, 16:24], out[:, 24:]))
    st.cache.check()
    assert bool((out[:, :16] == 5.0).all())
    assert torch.equal(out[:, 16:], qkv[:, 16:].bfloat16().float())


def test_one_tensor_for_keys_and_values(paged):
    """A pool [pages, 2, heads, rows, dim]: k and v are strided views of it."""
    pool = torch.zeros(6, 2, 2, 16, 64, device=DEV)
    cache = paged.PagedKVCache(pool[:, 0], pool[:, 1])
    t = torch.tensor([[4, 2]], dtype=torch.int32, device=DEV)
    b = paged.PagedBatch(torch.tensor([0, 20], dtype=torch.int32, device=DEV),
                         torch.tensor([20], dtype=torch.int32, device=DEV), t, 20)
    k, v = torch.randn(2, 20, 2, 64, device=DEV)
    cache.write(b, k, v)
    assert torch.equal(pool[4, 0].transpose(0, 1), k[:16]) and torch.equal(pool[2, 1, :, :4].transpose(0, 1), v[16:])
    assert bool((pool[[0, 1, 3, 5]] == 0).all())


# ---------------------------------------------------------------------------
# Attention.
# ---------------------------------------------------------------------------
RAGGED = [(1, 1), (17, 1), (0, 0), (300, 1), (64, 1), (1000, 1)]
BLOCKS = [(16, 16), (333, 16), (40, 7), (129, 1), (5, 5)]
CHUNKS = [(200, 130), (513, 65), (1, 1), (700, 300), (64, 64)]


@pytest.mark.parametrize("seqs", [RAGGED, BLOCKS, CHUNKS], ids=["tokens", "blocks", "chunks"])
@pytest.mark.parametrize("cache", TYPES)
@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_types(paged, rows, cache, dim, seqs):
    st = Setup(paged, cache, seqs, kv_heads=2, dim=dim, page=16, extra_rows=3)
    st.fill()
    st.check_attention(4, rows)


@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (5, 5), (8, 1), (12, 4), (20, 2), (40, 1), (16, 8)])
@pytest.mark.parametrize("seqs", [RAGGED, BLOCKS, CHUNKS], ids=["tokens", "blocks", "chunks"])
def test_attention_heads(paged, q_heads, kv_heads, seqs):
    for rows, cache in ((F32, F32), (BF16, BF16)):
        st = Setup(paged, cache, seqs, kv_heads=kv_heads, page=32, seed=2)
        st.fill()
        st.check_attention(q_heads, rows)


@pytest.mark.parametrize("page", [1, 3, 8, 24, 100, 128, 1000])
@pytest.mark.parametrize("seqs", [RAGGED, BLOCKS, CHUNKS], ids=["tokens", "blocks", "chunks"])
def test_attention_page_sizes(paged, page, seqs):
    for cache, rows in ((BF16, BF16), (E4M3, F32)):
        st = Setup(paged, cache, seqs, page=page, seed=3)
        st.fill()
        st.check_attention(4, rows)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (64, 4), (100, 33), (128, 200), (5000, 4), (333, 1)])
@pytest.mark.parametrize("seqs", [RAGGED, BLOCKS, CHUNKS], ids=["tokens", "blocks", "chunks"])
def test_attention_window(paged, window, sinks, seqs):
    for cache, rows in ((BF16, BF16), (INT8, BF16), (F32, F32)):
        st = Setup(paged, cache, seqs, seed=4)
        st.fill()
        st.check_attention(4, rows, window=window, sinks=sinks)


@pytest.mark.parametrize("seqs", [RAGGED, BLOCKS, CHUNKS], ids=["tokens", "blocks", "chunks"])
@pytest.mark.parametrize("rows", [F32, BF16])
def test_attention_without_mask(paged, rows, seqs):
    st = Setup(paged, BF16, seqs, seed=5)
    st.fill()
    st.check_attention(4, rows, causal=False)


@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("cache", [F32, BF16, E4M3])
def test_rows_that_see_nothing(paged, rows, cache):
    """Rows before position 0 (more rows than cache positions) give zeros; empty sequences change nothing."""
    for seqs in ([(3, 9), (0, 4), (0, 0), (20, 1)], [(100, 150), (0, 70)]):
        st = Setup(paged, cache, seqs, extra_rows=1, seed=6)
        st.fill()
        out = st.check_attention(4, rows)
        n0 = seqs[0][1] - seqs[0][0]
        assert bool((out[:n0] == 0).all()) and bool((out[st.starts[1]:st.starts[2]] == 0).all())


@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_items_that_see_nothing_between_others(paged, cache):
    """Wide tiles of padding rows only, several to a CTA and between real ones, with and without whole pages of 16;
    repeated, and the same bits every time."""
    for page in (16, 24):
        seqs = [(0, 70), (400, 300), (0, 130), (5, 200), (1000, 129), (0, 40), (257, 64)] * 6
        st = Setup(paged, cache, seqs, kv_heads=4, page=page, seed=18)
        st.fill()
        out = st.check_attention(8, BF16)
        q = torch.randn(st.rows, 8, 128, generator=st.gen).to(BF16).to(DEV)
        first = st.cache.attention(st.batch, q, 0.1)
        for _ in range(20):
            assert torch.equal(st.cache.attention(st.batch, q, 0.1), first)
        st.cache.check()
        assert bool((out[:70] == 0).all())


@pytest.mark.parametrize("seqs", [[(50, 16)], [(300, 200)], [(700, 300)]], ids=["block", "chunk", "long"])
@pytest.mark.parametrize("rows,cache", [(F32, F32), (BF16, BF16), (F32, BF16), (BF16, F32), (BF16, E4M3)])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_values_that_a_row_does_not_see(paged, rows, cache, seqs, value):
    """An infinity or NaN in a key or value reaches the rows that see its position, and no others."""
    st = Setup(paged, cache, seqs, seed=7)
    st.fill()
    kv, n = seqs[0]
    for which, p, d in (("v", kv - 3, 5), ("v", kv - n + 2, 17), ("k", kv - 6, 100)):
        page, row = int(st.table[0, p // st.page]), p % st.page
        (st.values if which == "v" else st.keys)[0][p, 1, d] = math.nan
        if cache == E4M3:
            (st.cache.v_scale if which == "v" else st.cache.k_scale)[page, 1, row] = math.nan
            (st.values if which == "v" else st.keys)[0][p, 1] = math.nan
        else:
            # (an infinite key gives infinite scores of either sign: only a NaN is sure to show)
            (st.cache.v if which == "v" else st.cache.k)[page, 1, row, d] = value if which == "v" else math.nan
    q = torch.randn(st.rows, 4, 128, generator=st.gen).to(rows).to(DEV)
    out = st.cache.attention(st.batch, q, 0.09)
    have = torch.where(torch.isfinite(out), out, math.nan)   # an infinite output is as good as a NaN
    st.compare(q, have, 0.09)
    # With a window that has passed the bad positions nothing of them is left.
    if n < 100:
        st2 = st.cache.attention(st.batch, q, 0.09, window=2, sinks=4)
        assert bool(torch.isfinite(st2[-1]).all())


@pytest.mark.parametrize("rows", [F32, BF16])
@pytest.mark.parametrize("seqs", [RAGGED, BLOCKS, CHUNKS], ids=["tokens", "blocks", "chunks"])
def test_large_scores(paged, rows, seqs):
    """Scores of several hundred: one position takes all the weight, nothing overflows."""
    st = Setup(paged, BF16, seqs, seed=8)
    st.fill(spread=30.0)
    out = st.check_attention(4, rows, scale=0.5)
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("scale", [1e-45, 1e-30, 1e30])
@pytest.mark.parametrize("seqs", [RAGGED, BLOCKS, CHUNKS], ids=["tokens", "blocks", "chunks"])
def test_queries_of_zeros(paged, seqs, scale):
    """Every score is zero at any scale: the mean of the visible values."""
    for rows, cache in ((F32, F32), (F32, E4M3), (BF16, BF16), (BF16, INT8)):
        st = Setup(paged, cache, seqs, seed=23)
        st.fill()
        st.check_attention(4, rows, scale=scale, window=50, sinks=2, q=torch.zeros(st.rows, 4, 128, dtype=rows, device=DEV))


def test_long_sequence_few_rows(paged):
    """The keys of one sequence split over the whole GPU and joined."""
    for rows, cache, seqs, heads in ((F32, F32, [(20001, 1)], (2, 1)), (BF16, E4M3, [(33333, 2)], (8, 1)),
                                     (BF16, BF16, [(30000, 40), (7, 7)], (4, 2)), (F32, BF16, [(9000, 200)], (2, 1)),
                                     (BF16, BF16, [(30000, 200)], (2, 1))):
        st = Setup(paged, cache, seqs, kv_heads=heads[1], page=16, seed=9)
        st.fill()
        st.check_attention(heads[0], rows)
        st.check_attention(heads[0], rows, window=20000, sinks=5)


def test_many_sequences(paged):
    rng = np.random.default_rng(1)
    for rows, cache in ((BF16, INT8), (F32, BF16)):
        seqs = [(int(rng.integers(0, 90)), int(rng.integers(0, 3))) for _ in range(700)]
        seqs = [(max(kv, n), n) for kv, n in seqs]
        st = Setup(paged, cache, seqs, kv_heads=1, dim=64, page=16, seed=10)
        st.fill()
        st.check_attention(2, rows)


def test_many_blocks(paged):
    """More sequences than a CTA's threads look at in one round, tiles of 256 columns."""
    rng = np.random.default_rng(2)
    for cache in (BF16, E4M3):
        seqs = [(int(rng.integers(0, 90)), int(rng.integers(0, 40))) for _ in range(900)]
        st = Setup(paged, cache, seqs, kv_heads=1, dim=64, page=16, seed=19, extra_rows=4)
        st.fill()
        st.check_attention(4, BF16)


@pytest.mark.parametrize("octaves", [5, 6, 7, 30])
@pytest.mark.parametrize("cache", [E4M3, INT8])
def test_values_of_many_sizes(paged, cache, octaves):
    """8-bit caches whose value scales lie close together and far apart within a block of keys."""
    for seqs in (RAGGED, BLOCKS, CHUNKS):
        for rows in (F32, BF16):
            st = Setup(paged, cache, seqs, seed=20)
            st.fill(octaves=octaves)
            st.check_attention(4, rows)
            st.check_attention(4, rows, window=100, sinks=3)


@pytest.mark.parametrize("q_heads,kv_heads", [(64, 1), (1024, 1), (1024, 1024), (99, 3)])
def test_many_heads(paged, q_heads, kv_heads):
    """Groups of more heads than a tile has columns; as many KV heads as there may be."""
    for rows, cache in ((BF16, BF16), (BF16, INT8), (F32, E4M3)):
        st = Setup(paged, cache, [(300, 1), (0, 0), (20, 2)], kv_heads=kv_heads, dim=64, page=16, seed=21)
        st.fill()
        st.check_attention(q_heads, rows)


@pytest.mark.parametrize("cache", TYPES)
def test_shared_pages_and_interleaved_pools(paged, cache):
    """Sequences that share the pages of a prefix, and keys and values that alternate page by page in one tensor,
    give the same bits as separate ones."""
    for n, page in ((1, 16), (5, 16), (90, 16), (90, 24)):
        st = Setup(paged, cache, [(400, n), (400, n), (400, n)], page=page, seed=22)
        rows = [torch.randn(400, 2, 128, generator=st.gen).to(DEV) for _ in range(2)]
        starts = torch.tensor([0, 400, 800, 1200], dtype=torch.int32, device=DEV)
        whole = paged.PagedBatch(starts, st.d_kv, st.d_table, 400)
        st.cache.write(whole, *(t.repeat(3, 1, 1) for t in rows))
        for q_dtype in (F32, BF16):
            q = torch.randn(3 * n, 4, 128, generator=st.gen).to(q_dtype).to(DEV)
            want = st.cache.attention(st.batch, q, 0.1)
            shared = paged.PagedBatch(st.d_starts, st.d_kv, st.d_table[:1].expand(3, -1), n)
            assert torch.equal(st.cache.attention(shared, q, 0.1), want)
            c = st.cache

            def alternate(x, y):
                return [t.view(x.dtype) for t in torch.stack((x.view(torch.uint8) if cache.itemsize == 1 else x,
                                                              y.view(torch.uint8) if cache.itemsize == 1 else y), 1).unbind(1)]

            k, v = alternate(c.k, c.v)
            scales = torch.stack((c.k_scale, c.v_scale), -1).unbind(-1) if cache.itemsize == 1 else (None, None)
            other = paged.PagedKVCache(k, v, *scales)
            assert not k.is_contiguous()
            assert torch.equal(other.attention(st.batch, q, 0.1), want)
            other.check()
        st.cache.check()


def test_offsets_past_32_bits(paged):
    """Pages beyond 2^31 elements of a pool."""
    page, heads = 64, 8
    pages = (1 << 31) // (page * heads * 128) + 40
    k, v = (torch.zeros((pages, heads, page, 128), dtype=torch.int8, device=DEV) for _ in range(2))
    scales = [torch.zeros((pages, heads, page), device=DEV) for _ in range(2)]
    st = Setup(paged, INT8, [(100, 100), (150, 5)], kv_heads=heads, page=page)
    st.cache = paged.PagedKVCache(k, v, *scales)
    st.table[0, :2] = torch.tensor([pages - 1, pages - 30])
    st.table[1, :3] = torch.tensor([pages - 2, 0, pages - 9])
    st.d_table.copy_(st.table)
    st.fill()
    got, _ = st.cache.read(st.batch, st.rows, F32)
    assert torch.equal(got[:100].cpu(), st.keys[0].float().cpu())
    st.check_attention(16, BF16)
    st.check_attention(16, F32)


def test_strided_rows_in_attention(paged):
    """q inside a projection buffer, the output inside another, block table rows with slack."""
    for rows in (F32, BF16):
        for seqs in (RAGGED, CHUNKS):
            st = Setup(paged, BF16, seqs, kv_heads=8, layout="prhd", seed=11)
            st.fill()
            wide = torch.full((len(seqs), st.d_table.shape[1] + 5), 9999, dtype=torch.int32, device=DEV)
            wide[:, :st.d_table.shape[1]] = st.d_table
            st.batch = paged.PagedBatch(st.d_starts, st.d_kv, wide[:, :st.d_table.shape[1]], 1)
            qkv = torch.randn(st.rows, 32, 128, generator=st.gen).to(rows).to(DEV)
            out = torch.full((16, st.rows, 128), 3.0, dtype=rows, device=DEV).transpose(0, 1)
            st.check_attention(16, rows, q=qkv[:, :16], out=out)


def test_max_rows_is_only_a_hint(paged):
    for hint in (0, 1, 5, 100000):
        for rows in (F32, BF16):
            st = Setup(paged, BF16, CHUNKS, seed=12)
            st.fill()
            st.batch = paged.PagedBatch(st.d_starts, st.d_kv, st.d_table, hint)
            st.check_attention(4, rows)


# ---------------------------------------------------------------------------
# Streams, graphs, devices' state, refusals on the device.
# ---------------------------------------------------------------------------
def test_captured_call_follows_the_arrays(paged):
    """A captured write + attention replayed with other lengths, pages and rows; two graphs in turn."""
    st = Setup(paged, E4M3, [(40, 1), (200, 1)], seed=13)
    st.fill()
    q = torch.randn(2, 4, 128, generator=st.gen).to(BF16).to(DEV)
    k, v = (torch.randn(2, 2, 128, generator=st.gen).to(BF16).to(DEV) for _ in range(2))
    out = torch.full_like(q, 77.0)
    other = torch.full_like(q, 77.0)

    def step(o, window):
        st.cache.write(st.batch, k, v)
        st.cache.attention(st.batch, q, 0.1, out=o, window=window, sinks=2)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(out, 0)
    torch.cuda.synchronize()
    graphs = []
    for o, w in ((out, 0), (other, 50)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(o, w)
        graphs.append(g)
    for lens in ([40, 200], [39, 77], [1, 161]):
        st.d_kv.copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(torch.randn(2, 4, 128, generator=st.gen))
        k.copy_(torch.randn(2, 2, 128, generator=st.gen))
        for g in graphs + graphs:
            g.replay()
        torch.cuda.synchronize()
        st.cache.check()
        newk, newv = st.stand_for(k.cpu()), st.stand_for(v.cpu())
        keys, values = [], []
        for s, n in enumerate(lens):
            st.keys[s][n - 1], st.values[s][n - 1] = newk[s], newv[s]
            keys.append(st.keys[s][:n])
            values.append(st.values[s][:n])
        whole = (st.keys, st.values, st.kv)
        st.keys, st.values, st.kv = keys, values, lens
        st.compare(q, out, 0.1)
        st.compare(q, other, 0.1, window=50, sinks=2)
        st.keys, st.values, st.kv = whole


def test_two_streams_at_once(paged):
    """Calls on two streams that overlap, each with its own cache and workspace, repeated: the same bits every time."""
    sts = [Setup(paged, BF16, [(5000, 1), (300, 1)], seed=14), Setup(paged, E4M3, [(700, 300), (6000, 9)], seed=15)]
    qs, first = [], []
    for st in sts:
        st.fill()
        qs.append(torch.randn(st.rows, 4, 128, generator=st.gen).to(BF16).to(DEV))
        first.append(st.cache.attention(st.batch, qs[-1], 0.1))
        st.compare(qs[-1], first[-1], 0.1)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sts]
    for _ in range(20):
        outs = []
        for st, q, s in zip(sts, qs, streams):
            with torch.cuda.stream(s):
                outs.append(st.cache.attention(st.batch, q, 0.1))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, first))


def test_bad_arrays_are_reported_and_skipped(paged, pkg):
    for rows in (F32, BF16):
        for n in (1, 130):
            st = Setup(paged, BF16, [(200, n), (200, n), (200, n)], seed=16)
            st.fill()
            q = torch.randn(st.rows, 4, 128, generator=st.gen).to(rows).to(DEV)
            good = st.cache.attention(st.batch, q, 0.1)

            def run(what, match, sane):
                out = torch.full_like(q, 77.0)
                st.cache.attention(st.batch, q, 0.1, out=out)
                with pytest.raises(pkg.HyError, match=match):
                    st.cache.check()
                st.cache.check()   # cleared
                for s in sane:
                    assert torch.equal(out[s * n:(s + 1) * n], good[s * n:(s + 1) * n]), what
                return out

            st.d_table[1, 2] = 10 ** 6   # positions 32..47 of sequence 1 are not seen
            out = run("page", "page number", (0, 2))
            keep = [st.keys[1], st.values[1]]
            sel = [j for j in range(200) if not 32 <= j < 48]
            want, mass, reach = R.attention(q[n:n + 1].double(), keep[0][sel], keep[1][sel],
                                            [sum(j <= 200 - n for j in sel) - 1], 0.1)
            tol = R.tolerance(want, mass, reach, 200, 128, rows)
            assert bool(((out[n:n + 1].double() - want).abs() <= tol).all())
            st.d_table[1, 2] = -1
            run("page", "page number", (0, 2))
            st.d_table.copy_(st.table)
            for bad in (-1, 10 ** 6):
                st.d_kv[2] = bad
                out = run("length", "kv_len", (0, 1))
                assert bool((out[2 * n:] == 77.0).all())
                st.d_kv[2] = 200
            st.d_starts[3] = 10 ** 6
            out = run("rows", "q_start", (0, 1))
            assert bool((out[2 * n:] == 77.0).all())
            st.d_starts[3] = 3 * n
            st.d_starts[1] = -5
            out = run("rows", "q_start", (2,))
            k = torch.zeros(st.rows, 2, 128, device=DEV)
            st.d_starts[1] = n
            st.d_table[0, :] = -3
            st.cache.write(st.batch, k, k)   # sequence 0's rows go nowhere
            back = torch.full((st.rows, 2, 128), 4.0, device=DEV)
            st.cache.read(st.batch, st.rows, F32, out=(back, back.clone()))
            with pytest.raises(pkg.HyError, match="page number"):
                st.cache.check()
            assert bool((back[:n] == 4.0).all()) and bool((back[n:] == 0).all())


def test_call_refusals_with_tensors(paged, pkg):
    st = Setup(paged, BF16, [(20, 2)])
    q = torch.zeros(2, 4, 128, dtype=BF16, device=DEV)
    for bad, match in ((q.half(), "float32 or bfloat16"), (q.cpu(), "float32 or bfloat16"), (q[..., :64], "128"),
                       (q[:, :3], "multiple"), (q.transpose(1, 2).contiguous().transpose(1, 2), "contiguous")):
        with pytest.raises(pkg.HyError, match=match):
            st.cache.attention(st.batch, bad, 0.1)
    with pytest.raises(pkg.HyError, match="overlap"):
        st.cache.attention(st.batch, q, 0.1, out=q)
    with pytest.raises(pkg.HyError, match="causal"):
        st.cache.attention(st.batch, q, 0.1, causal=False, window=3)
    with pytest.raises(pkg.HyError, match="gradient"):
        st.cache.attention(st.batch, q.float().requires_grad_(), 0.1)
    with pytest.raises(pkg.HyError, match="16 bytes"):
        st.cache.attention(st.batch, torch.zeros(2 * 4 * 128 + 8, dtype=BF16, device=DEV)[1:1025].view(2, 4, 128), 0.1)
    k = torch.zeros(2, 2, 128, device=DEV)
    with pytest.raises(pkg.HyError, match="one shape"):
        st.cache.write(st.batch, k, k.bfloat16())
    with pytest.raises(pkg.HyError, match="scales"):
        paged.PagedKVCache(st.cache.k.view(torch.int8)[..., :128], st.cache.v.view(torch.int8)[..., :128]).write(
            st.batch, k, k)
    with pytest.raises(pkg.HyError, match="int32"):
        paged.PagedBatch(st.d_starts.long(), st.d_kv, st.d_table, 2)
    assert st.cache.attention(paged.PagedBatch(st.d_starts[:1], st.d_kv[:0], st.d_table[:0], 0), q[:0], 0.1).shape[0] == 0


@pytest.mark.parametrize("cache", TYPES)
def test_prompt_then_tokens(paged, cache):
    """The calls together, as a server makes them: prompts written in chunks with attention over what is there, then
    tokens of all sequences at once through a window with sinks, each step against the 64-bit form of what was fed."""
    rng = torch.Generator().manual_seed(17)
    lens, heads, kvh, dim, page = [150, 37], 8, 4, 128, 16
    total = [n + 12 for n in lens]
    cache_ = paged.PagedKVCache.allocate(40, kvh, page, dim, cache)
    order = torch.randperm(40, generator=rng)[:2 * 12].view(2, 12).int().to(DEV)
    ref = Setup(paged, cache, [(1, 1)], kv_heads=kvh)
    K = [torch.randn(n, kvh, dim, generator=rng) for n in total]
    V = [torch.randn(n, kvh, dim, generator=rng) for n in total]
    k64, v64 = [ref.stand_for(x) for x in K], [ref.stand_for(x) for x in V]
    at = [0, 0]

    def step(counts, window, rows):
        starts = torch.tensor([0] + np.cumsum(counts).tolist(), dtype=torch.int32, device=DEV)
        now = [a + c for a, c in zip(at, counts)]
        b = paged.PagedBatch(starts, torch.tensor(now, dtype=torch.int32, device=DEV), order, max(counts))
        k, v = (torch.cat([x[a:a + c] for x, a, c in zip(X, at, counts)]).to(DEV) for X in (K, V))
        q = torch.randn(sum(counts), heads, dim, generator=rng).to(rows).to(DEV)
        cache_.write(b, k, v)
        out = cache_.attention(b, q, 0.0883883, window=window, sinks=4 if window else 0)
        cache_.check()
        r = 0
        for s, c in enumerate(counts):
            want, mass, reach = R.attention(q[r:r + c].double(), k64[s][:now[s]], v64[s][:now[s]],
                                            list(range(at[s], now[s])), 0.0883883, True, window, 4)
            tol = R.tolerance(want, mass, reach, now[s], dim, rows)
            assert bool(((out[r:r + c].double() - want).abs() <= tol).all())
            r += c
        at[:] = now

    for rows in (F32, BF16):
        step([60, 37 if rows == F32 else 0], 0, rows)
    step([30, 0], 0, F32)
    for i in range(12):
        step([1, 1], 32 if i % 2 else 0, BF16 if i % 3 else F32)


def test_prefix_moves_between_contexts_by_pages(paged, pkg):
    """A context's prefilled KV rows into pages and from there into another context, which then decodes the same
    tokens (fp32 pages are exact); 8-bit pages bring back code * scale of the same rows."""
    cfg = dict(num_layers=2, vocab_size=4096, max_context=256, max_prefill=192, max_tokens=64)
    rng = np.random.default_rng(5)
    seq = 150
    embeds = rng.standard_normal((seq, 1024)).astype(np.float32) * 0.02
    cos, sin = pkg.rope_rows(0, seq, True), pkg.rope_rows(0, seq, False)
    table = torch.randperm(12, generator=torch.Generator().manual_seed(1)).int().to(DEV)[None]
    batch = paged.PagedBatch(torch.tensor([0, seq], dtype=torch.int32, device=DEV),
                             torch.tensor([seq], dtype=torch.int32, device=DEV), table, seq)
    with pkg.TextRuntime.synthetic(seed=3, norm_std=0.1, **cfg) as a, pkg.TextRuntime.synthetic(seed=3, norm_std=0.1, **cfg) as b:
        a.prefill(embeds, cos, sin)
        rows = [a.kv_read(layer, 0, seq) for layer in range(2)]
        pages = [paged.PagedKVCache.allocate(12, 8, 16, 128, F32) for _ in range(2)]
        for layer in range(2):
            a.store_kv_pages(layer, pages[layer], batch, seq)
        a.set_history([])
        want, _ = a.generate(7, 7, 24, 1.08)
        b.reset()
        for layer in range(2):
            b.load_kv_pages(layer, pages[layer], batch, seq)
        b.prefill(embeds[:1], cos[:1], sin[:1])   # any sequence of its own: the length is set below
        for layer in range(2):
            b.load_kv_pages(layer, pages[layer], batch, seq)
            pages[layer].check()
            k, v = b.kv_read(layer, 0, seq)
            assert np.array_equal(k, rows[layer][0]) and np.array_equal(v, rows[layer][1])
        b.set_length(seq)
        b.set_history([])
        got, _ = b.generate(7, 7, 24, 1.08)
        assert got == want
        small = paged.PagedKVCache.allocate(12, 8, 16, 128, INT8)
        a.store_kv_pages(1, small, batch, seq)
        b.load_kv_pages(1, small, batch, seq)
        small.check()
        back = b.kv_read(1, 0, seq)
        for x, y in zip(rows[1], back):
            code, scale = R.quantise(torch.from_numpy(x), INT8)
            assert np.array_equal(y, (code.float() * scale.float()[..., None]).numpy())
        with pytest.raises(pkg.HyError, match="capacity"):
            a.store_kv_pages(0, pages[0], batch, 257)
        with pytest.raises(pkg.HyError, match="layer"):
            a.store_kv_pages(2, pages[0], batch, seq)
