"""How near the paged attention comes to the 64-bit form: bounds that are a small share of the outputs, so that a
part of the keys lost, or a term of the products, would show."""

import math

import pytest
import torch

import paged_reference as R
from test_gpu_paged import BF16, BLOCKS, CHUNKS, DEV, E4M3, F32, INT8, RAGGED, TYPES, Setup, paged  # noqa: F401

pytestmark = pytest.mark.gpu

LONG = [[(9000, 1)], [(33333, 2)], [(30000, 200)]]
CASES = [RAGGED, BLOCKS, CHUNKS] + LONG
IDS = ["tokens", "blocks", "chunks", "9000", "33333", "30000x200"]


def ordinary_bound(rows):
    """Of the error's root mean square over the outputs', rows and keys of unit variance. bf16 rows: weights and outputs
    are off by up to 2^-9 of a power of two above them, some 2^-10 on average; 2^-8 leaves a factor of 2 over both.

    fp32 rows: products exact to 2^-21; a score adds up 128 of them, a few units large, in 8 steps of up to 6 products
    whose sums are cut at 2^-23 of them, and is then scaled by 0.09: some 2^-20. With weights and sums of 2^-21, 2^-18
    leaves a factor of 2. Sums over the keys are rounded from step to step and so stay at that however many there are.
    (Splitting q, k and v into two bf16 terms instead of three costs 2.3e-5.)"""
    return 2.0 ** -8 if rows == BF16 else 2.0 ** -18


@pytest.mark.parametrize("seqs", CASES, ids=IDS)
@pytest.mark.parametrize("cache", TYPES)
@pytest.mark.parametrize("rows", [F32, BF16])
def test_error_of_ordinary_data(paged, rows, cache, seqs):
    st = Setup(paged, cache, seqs, kv_heads=1, seed=37)
    st.fill()
    scale = 1 / math.sqrt(128)
    for window, sinks in ((0, 0), (200, 5)):
        q = torch.randn(st.rows, 2, 128, generator=st.gen).to(rows).to(DEV)
        out = st.cache.attention(st.batch, q, scale, window=window, sinks=sinks)
        st.cache.check()
        err = ref = 0.0
        for s, (kv, n) in enumerate(seqs):
            a, b = st.starts[s], st.starts[s + 1]
            want, _, _ = R.attention(q[a:b].double(), st.keys[s], st.values[s], list(range(kv - n, kv)), scale, True,
                                     window, sinks)
            err += float((out[a:b].double() - want).square().sum())
            ref += float(want.square().sum())
        assert math.sqrt(err / ref) <= ordinary_bound(rows), math.sqrt(err / ref)


def code_tolerance(want, mass, reach, t, codes, length, dim, dtype, wide):
    """At every output, over 8-bit caches. Scores and sums as in paged_reference.tolerance, with products exact to 2^-21.
    A weight times its value's scale is an f16 number (fp32 rows: two), off by 2^-11 (2^-22) of itself, or by 2^-25 in the
    unit it carries, 2^14 (tiles of 256 columns: 2^6, and the maximum up to 2^4 too large): so by 2^-39 (2^-27) of the
    row's largest such product t, times the codes of the keys that the row sees. bf16 rows: the output half a step more."""
    rel = 2 * reach * (2.0 ** -21 + dim * 2.0 ** -24) + 2.0 ** -20 + length * 2.0 ** -24
    rel = rel + (2.0 ** -11 if dtype == BF16 else 2.0 ** -22)
    tol = mass * rel + 2.0 ** (-27 if wide else -39) * t * codes + 2.0 ** -126
    return tol + (want.abs() + tol) * 2.0 ** -8 if dtype == BF16 else tol


@pytest.mark.parametrize("octaves", [0, 2, 5, 30])
@pytest.mark.parametrize("seqs", CASES, ids=IDS)
@pytest.mark.parametrize("cache", [E4M3, INT8])
@pytest.mark.parametrize("rows", [F32, BF16])
def test_every_output_over_codes(paged, rows, cache, seqs, octaves):
    st = Setup(paged, cache, seqs, kv_heads=1, seed=39)
    st.fill(octaves=octaves)
    scale, heads = 1 / math.sqrt(128), 2
    q = torch.randn(st.rows, heads, 128, generator=st.gen).to(rows).to(DEV)
    out = st.cache.attention(st.batch, q, scale)
    st.cache.check()
    wide = rows == BF16 and max(n for _, n in seqs) * heads > 32
    for s, (kv, n) in enumerate(seqs):
        a, b = st.starts[s], st.starts[s + 1]
        if n == 0:
            continue
        pos = list(range(kv - n, kv))
        want, mass, reach = R.attention(q[a:b].double(), st.keys[s], st.values[s], pos, scale)
        p = torch.arange(kv)
        vs = st.cache.v_scale[st.table[s, p // st.page].long().to(DEV), 0, (p % st.page).to(DEV)].double()
        seen = torch.arange(kv, device=DEV)[None] <= torch.tensor(pos, device=DEV)[:, None]
        scores = torch.einsum("nhd,ld->nhl", q[a:b].double(), st.keys[s][:, 0]) * scale
        weights = torch.softmax(scores.masked_fill(~seen[:, None], -math.inf), dim=-1)
        t = (weights * vs).amax(dim=-1, keepdim=True)
        codes = (seen.double() @ (st.values[s][:, 0] / vs[:, None]).abs())[:, None]
        tol = code_tolerance(want, mass, reach, t, codes, kv, 128, rows, wide)
        assert float((tol.norm(dim=-1) / want.norm(dim=-1)).max()) < 0.4   # (nothing like the outputs themselves)
        off = (out[a:b].double() - want).abs() - tol
        assert float(off.max()) <= 0, (s, float(off.max()))


@pytest.mark.parametrize("cache", TYPES)
def test_long_chains_of_additions(paged, cache):
    """One block adds up a whole long item (more items than blocks): some 250 steps of 16 keys to a sum in a warp. Rounded
    additions of the steps leave errors of either sign, so that the bound of fp32 rows is that of short sequences."""
    seqs, heads, kv_heads = [(16000 + 7 * i, 20) for i in range(8)], 32, 8
    st = Setup(paged, cache, seqs, kv_heads=kv_heads, dim=64, page=64, seed=46)
    st.fill()
    q = torch.randn(st.rows, heads, 64, generator=st.gen).to(DEV)
    out = st.cache.attention(st.batch, q, 0.125)
    st.cache.check()
    err = ref = 0.0
    for s in (0, 3, 7):
        kv, n = seqs[s]
        a, b = st.starts[s], st.starts[s + 1]
        want, _, _ = R.attention(q[a:b].double(), st.keys[s], st.values[s], list(range(kv - n, kv)), 0.125)
        err += float((out[a:b].double() - want).square().sum())
        ref += float(want.square().sum())
    assert math.sqrt(err / ref) <= ordinary_bound(F32), math.sqrt(err / ref)


@pytest.mark.parametrize("cache", TYPES)
def test_scores_of_loud_dimensions(paged, cache):
    """fp32 rows in tiles of 32 columns over keys with four dimensions eight times the others: scores of some 2 units,
    up to 10. The tensor cores cut a sum at every product (by 2^-24 of it on average): through all 24 of a score over BF16
    pages (48 over F32) the same arithmetic on the CPU is off by 1.8e-6 in the outputs, through the 8 that matter by
    6e-7; the bound leaves a factor of 2 over that."""
    seqs = [(1500, 16), (2600, 16), (1800, 16), (2111, 16)]
    st = Setup(paged, cache, seqs, kv_heads=8, seed=47)
    loud = torch.ones(128)
    loud[[3, 40, 77, 126]] = 8.0
    k, v = (torch.randn(sum(st.kv), 8, 128, generator=st.gen) * loud for _ in range(2))
    starts = torch.tensor([0, 1500, 4100, 5900, 8011], dtype=torch.int32, device=DEV)
    st.cache.write(paged.PagedBatch(starts, st.d_kv, st.d_table, 2600), k.to(DEV), v.to(DEV))
    keys, values = (st.stand_for(x).split(st.kv) for x in (k, v))
    q = torch.randn(st.rows, 16, 128, generator=st.gen).to(DEV)
    out = st.cache.attention(st.batch, q, 0.0883883)
    st.cache.check()
    err = ref = 0.0
    for s, (kv, n) in enumerate(seqs):
        a, b = st.starts[s], st.starts[s + 1]
        want, _, _ = R.attention(q[a:b].double(), keys[s], values[s], list(range(kv - n, kv)), 0.0883883)
        err += float((out[a:b].double() - want).square().sum())
        ref += float(want.square().sum())
    assert math.sqrt(err / ref) <= 1.25 * 2.0 ** -20, math.sqrt(err / ref)
