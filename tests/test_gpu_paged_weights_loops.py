"""Attention weights where every block of threads has many tiles, on the GPU: rings and buffers that are filled again, a
second and third item, the walk into the next head and the next sequence. Against the definition in 64 bits, with the
tolerances of test_gpu_paged_weights."""

import random

import pytest
import torch

from test_gpu_paged_weights import BF16, E4M3, F32, INT8, Setup, paged   # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

SMS = 148


def _lengths(n, lo, hi, seed):
    rng = random.Random(seed)
    return [rng.randint(lo, hi) for _ in range(n)]


def _tiles(kv, new, keys, kv_heads):
    return sum(-(-n // keys) for n, m in zip(kv, new) if m) * kv_heads


# ---------------------------------------------------------------------------
# Many bf16 rows (tcgen05): items of up to two blocks of 128 keys, tiles of 128 columns.
# ---------------------------------------------------------------------------
CHUNKS = [   # cache, dim, query heads, kv heads, page, kv, new, view
    (BF16, 128, 16, 8, 16, (6, 2000, 5000), (130, 300), {}),
    (BF16, 128, 24, 8, 24, (6, 2000, 5000), (20, 200), {}),                                # 128 is no multiple of the group
    (BF16, 64, 12, 12, 64, (5, 2500, 5000), (40, 400), dict(window=2300, sinks=5)),
    (BF16, 64, 32, 8, 7, (12, 900, 2100), (9, 60), dict(causal=False)),
    (E4M3, 128, 16, 8, 64, (6, 2000, 5000), (100, 300), {}),
    (E4M3, 128, 24, 8, 100, (6, 2000, 5000), (50, 200), dict(window=1500, sinks=130)),     # sinks that end inside a block
    (E4M3, 64, 36, 12, 16, (5, 2000, 4500), (40, 250), {}),
    (E4M3, 64, 16, 8, 1, (6, 2000, 4000), (300, 700), dict(causal=False)),
    (INT8, 128, 24, 8, 32, (6, 2000, 5000), (40, 300), {}),
    (INT8, 128, 8, 8, 16, (10, 2000, 5000), (130, 1100), dict(window=1000)),
    (INT8, 64, 64, 8, 48, (7, 1500, 4500), (5, 40), dict(window=2000, sinks=1)),
    (INT8, 64, 16, 16, 128, (4, 2000, 4000), (40, 900), {}),
]


@pytest.mark.parametrize("cache,dim,heads,kv_heads,page,kv,new,view", CHUNKS)
def test_many_rows(paged, cache, dim, heads, kv_heads, page, kv, new, view):   # noqa: F811
    seed = dim + heads + page
    lens, rows = _lengths(*kv, seed), _lengths(kv[0], *new, seed + 1)
    at = 2 + seed % 2
    lens[at:at], rows[at:at] = [0, 50, 333], [0, 60, 0]   # nothing; more rows than positions; no rows
    seen = [min(n, view.get("window", n) + m) for n, m in zip(lens, rows)]
    assert _tiles(seen, rows, 256, kv_heads) > 2 * SMS and max(rows) * heads // kv_heads > 32
    Setup(paged, cache, BF16, lens, rows, heads, kv_heads, dim, page, seed).check(**view)


def test_more_columns_than_rings_hold(paged):   # noqa: F811
    """A block of keys with 32 tiles of columns, and one with a few behind it."""
    Setup(paged, BF16, BF16, [2500, 4300], [2048, 77], 16, 8, 128, 16, 5).check()


# ---------------------------------------------------------------------------
# Columns past what the ring kernel takes, by mma.sync: tiles of 128 keys (8-bit caches: 256), 32 columns at a time. With
# at most 148 (sequence, head) pairs a block has one run of tiles of one; with more it goes on into the next ones.
# ---------------------------------------------------------------------------
WIDE = [(F32, F32), (F32, BF16), (BF16, F32), (E4M3, F32), (INT8, F32)]   # cache, rows


@pytest.mark.parametrize("cache,rows", WIDE)
@pytest.mark.parametrize("dim,kv_heads,group,page,kv,new,view", [
    (128, 8, 2, 16, (6, 3000, 6000), (10, 130), {}),
    (64, 4, 3, 24, (9, 4000, 9000), (12, 40), dict(window=3500, sinks=40)),
    (128, 8, 2, 32, (20, 1000, 2500), (17, 90), {}),
    (64, 16, 3, 100, (30, 200, 1400), (11, 50), dict(causal=False)),
])
def test_wide(paged, cache, rows, dim, kv_heads, group, page, kv, new, view):   # noqa: F811
    seed = dim + page
    lens, n = _lengths(*kv, seed), _lengths(kv[0], *new, seed + 1)
    n[1] = 0
    assert _tiles(lens, n, 256 if cache in (E4M3, INT8) else 128, kv_heads) > 2 * SMS
    Setup(paged, cache, rows, lens, n, kv_heads * group, kv_heads, dim, page, seed).check(**view)


@pytest.mark.parametrize("cache", [BF16, E4M3, INT8])
def test_verify_blocks(paged, cache):   # noqa: F811
    """bf16 rows of 9 to 32 columns."""
    lens = _lengths(40, 500, 2600, 3)
    assert _tiles(lens, lens, 256, 8) > 4 * SMS
    Setup(paged, cache, BF16, lens, [16 - i % 9 for i in range(40)], 16, 8, 128, 16, 4).check()


# ---------------------------------------------------------------------------
# Few columns: rings of four steps in each warp, three blocks to an SM, tiles of 32 to 128 keys.
# ---------------------------------------------------------------------------
FEW = [(c, r) for c in (F32, BF16, E4M3, INT8) for r in (F32, BF16)]


@pytest.mark.parametrize("cache,rows", FEW)
@pytest.mark.parametrize("dim,kv_heads,group,page,kv,view", [
    (128, 8, 2, 16, (40, 1500, 5000), {}),                               # a share that goes on into other heads and sequences
    (64, 8, 3, 24, (50, 1500, 5000), dict(window=2000, sinks=3)),
    (64, 4, 4, 64, (45, 4000, 8000), dict(causal=False)),
    (128, 2, 1, 100, (2, 40000, 60000), {}),                             # one run of tiles each
    (64, 3, 2, 16, (2, 60000, 90000), dict(window=50000, sinks=2000)),
])
def test_few_columns(paged, cache, rows, dim, kv_heads, group, page, kv, view):   # noqa: F811
    seed = dim + page
    lens = _lengths(*kv, seed)
    seen = [min(n, view.get("window") or n) for n in lens]
    assert _tiles(seen, seen, 128, kv_heads) > (8 if kv[0] > 32 else 2) * 3 * SMS or kv[0] == 2
    assert _tiles(seen, seen, 64 if dim == 64 else 32, kv_heads) > 6 * 3 * SMS or cache != F32
    Setup(paged, cache, rows, lens, [1] * kv[0], kv_heads * group, kv_heads, dim, page, seed).check(**view)


@pytest.mark.parametrize("cache,rows", FEW)
def test_few_columns_laid_out_for_fewer(paged, cache, rows):   # noqa: F811
    """Sequences of more columns than a pass takes: every tile of a run is passed over again.

    A pass takes 2 columns (fp32 caches; 8 over others) and adds their sum to what is there, so the weight w of a position is
    rounded once for every pass instead of once: (passes - 1) 2^-24 w on top of the tolerance of one pass. 11 rows of two
    heads are 11 passes."""
    lens, new = _lengths(36, 1500, 4000, 7), [1 + 5 * (i % 3) for i in range(36)]
    s = Setup(paged, cache, rows, lens, new, 8, 4, 64, 16, 8, max_rows=1)
    lse = s.lse()
    want, tol = s.expect(lse)
    for i, n in enumerate(new):
        pg, rw = s.place(i)
        passes = -(-2 * n // (2 if cache == F32 else 8))
        tol[pg, :, rw] += (passes - 1) * 2.0 ** -24 * want[pg, :, rw].abs()
    s.c.add_weights(s.batch, s.q, lse, s.scale, s.weights)
    s.c.check()
    assert ((s.weights.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("cache,rows,heads,new", [(BF16, BF16, 16, 200), (E4M3, BF16, 24, 90), (BF16, F32, 16, 40), (E4M3, BF16, 16, 1)])
def test_the_same_bits_again(paged, cache, rows, heads, new):   # noqa: F811
    s = Setup(paged, cache, rows, _lengths(36, 600, 3000, 9), [new] * 36, heads, 8, 128, 16, 10)
    lse, start = s.lse(), s.weights.clone()
    s.c.add_weights(s.batch, s.q, lse, s.scale, s.weights)
    first = s.weights.clone()
    for _ in range(3):
        s.weights.copy_(start)
        s.c.add_weights(s.batch, s.q, lse, s.scale, s.weights)
        assert torch.equal(s.weights, first)
    s.c.check()
