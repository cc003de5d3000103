"""Norms of heads with the rotation, on the GPU, against the formula in 64 bits."""

import importlib

import numpy as np
import pytest
import torch

from paged_reference import LARGEST, positions

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rotary(pkg):
    return importlib.import_module("hy_b200.rotary")


@pytest.fixture(scope="module")
def paged(pkg):
    return importlib.import_module("hy_b200.paged")


def _angles(rows, dim, gen):
    """A table whose halves differ, as mRoPE's do."""
    angle = torch.rand(rows, dim, generator=gen, device="cuda", dtype=torch.float64) * 6.28
    return angle.cos().float(), angle.sin().float()


def _inputs(rows, heads, kv_heads, dim, dtype, seed, table=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, heads + 2 * kv_heads, dim, generator=gen, device="cuda")
    x *= torch.where(torch.rand(dim, generator=gen, device="cuda") < 0.05, 8.0, 1.0)
    x = x.to(dtype)
    cos, sin = _angles(table or max(rows, 1), dim, gen)
    pos = torch.randint(table, (rows,), generator=gen, device="cuda", dtype=torch.int32) if table else None
    weights = [1 + 0.2 * torch.randn(dim, generator=gen, device="cuda") for _ in range(2)]
    return x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:], weights, cos, sin, pos


def _formula(x, w, cos, sin, pos, eps, rotate_first):
    """(result, reach): reach is |w| r (|lo c| + |hi s|), what the roundings are relative to."""
    x, w, h = x.double(), w.double(), x.shape[-1] // 2
    at = torch.arange(len(x), device=x.device) if pos is None else pos.long()
    c, s = cos.double()[at][:, None], sin.double()[at][:, None]

    def turn(y, sign=-1.0):
        return y * c + torch.cat([sign * y[..., h:], y[..., :h]], dim=-1) * s

    def reach(y):
        return y.abs() * c.abs() + torch.cat([y[..., h:], y[..., :h]], dim=-1).abs() * s.abs()

    if rotate_first:
        y = turn(x)
        r = 1 / torch.sqrt((y * y).mean(dim=-1, keepdim=True) + eps)
        return y * r * w, reach(x) * r * w.abs()
    y = x * w / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + eps)
    return turn(y), reach(y)


def _tolerance(want, reach, dtype):
    """In units of 2^-24 of reach: the rotation 2 (a product and a fused sum), the weight 1, the factor's product 1; the
    factor itself: half of the sum of squares' error (at most 24 additions of a lane and its mates, 12; the rotated
    values' errors in it, 3), rsqrtf's 2 units in the last place, 4; norm first rounds x w once more, 1. 24 in all. bf16
    rounds that once."""
    tol = reach * 24 * 2.0 ** -24
    return tol + (want.abs() + tol) * 2.0 ** -8 if dtype == torch.bfloat16 else tol


CASES = [(1, 16, 8, 128), (3, 1, 1, 64), (16, 16, 8, 128), (37, 5, 1, 64), (64, 32, 4, 128), (591, 6, 3, 64),
         (592, 16, 8, 128), (1777, 3, 3, 64), (4099, 7, 1, 128)]


@pytest.mark.parametrize("rotate_first", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,heads,kv_heads,dim", CASES)
def test_rows(rotary, rows, heads, kv_heads, dim, dtype, rotate_first):
    q, k, _, (qw, kw), cos, sin, pos = _inputs(rows, heads, kv_heads, dim, dtype, rows + dim, table=None if rows % 2 else 5000)
    got = rotary.norm_rotate(q, k, qw, kw, cos, sin, pos, eps=1e-5, rotate_first=rotate_first)
    for x, w, y in ((q, qw, got[0]), (k, kw, got[1])):
        want, reach = _formula(x, w, cos, sin, pos, 1e-5, rotate_first)
        assert y.dtype == dtype and (y.double() - want).abs().le(_tolerance(want, reach, dtype)).all()


@pytest.mark.parametrize("rows", [5, 700])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_in_place_and_other_layouts(rotary, rows, dtype):
    """The outputs in the place of the inputs, and heads before rows: the same bits."""
    q, k, _, (qw, kw), cos, sin, pos = _inputs(rows, 16, 8, 128, dtype, 3, table=100)
    want = rotary.norm_rotate(q, k, qw, kw, cos, sin, pos)
    other = [torch.empty(h, rows, 136, dtype=dtype, device="cuda")[..., :128].transpose(0, 1) for h in (16, 8)]
    rotary.norm_rotate(q, k, qw, kw, cos, sin, pos, out=other)
    held = q._base.clone() if q._base is not None else None
    assert held is not None
    qi, ki = held[:, :16], held[:, 16:24]
    rotary.norm_rotate(qi, ki, qw, kw, cos, sin, pos, out=(qi, ki))
    for a, b, c in zip(want, other, (qi, ki)):
        assert torch.equal(a, b) and torch.equal(a, c)
    assert torch.equal(held[:, 24:], q._base[:, 24:])   # the values beside them are as they were


def test_positions_outside_the_table_are_reported(rotary):
    q, k, _, (qw, kw), cos, sin, pos = _inputs(6, 4, 2, 64, torch.float32, 9, table=50)
    good = rotary.norm_rotate(q, k, qw, kw, cos, sin, pos)
    pos[1], pos[4] = 50, -1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = rotary.norm_rotate(q, k, qw, kw, cos, sin, pos, status=status)
    for a, b in zip(good, got):
        assert torch.isnan(b[[1, 4]]).all()
        assert torch.equal(a[[0, 2, 3, 5]], b[[0, 2, 3, 5]])
    assert status.item() == 16


def test_extreme_rows(rotary):
    """A row of zeros stays zero; an infinity or a NaN stays within its head."""
    q, k, _, (qw, kw), cos, sin, _ = _inputs(4, 2, 1, 128, torch.float32, 5)
    q = q.contiguous()
    q[0, 0] = 0
    q[1, 1, 5] = float("nan")
    q[2, 0, 7] = float("inf")
    out = rotary.norm_rotate(q, k, qw, kw, cos, sin)[0]
    assert (out[0, 0] == 0).all()
    assert torch.isnan(out[1, 1]).all() and torch.isfinite(out[1, 0]).all()
    assert torch.isfinite(out[2, 1]).all() and not torch.isfinite(out[2, 0]).all()
    assert torch.isfinite(out[3]).all()


# ---------------------------------------------------------------------------
# Into the paged cache.
# ---------------------------------------------------------------------------
CACHES = [torch.float32, torch.bfloat16, torch.float8_e4m3fn, torch.int8]


def _paged(paged, cache, kv_lens, news, kv_heads, dim, page, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    width = max(-(-n // page) for n in kv_lens) + 1
    pages = len(kv_lens) * width + 2
    table = torch.randperm(pages, generator=gen, device="cuda")[:len(kv_lens) * width].view(len(kv_lens), width).int()
    c = paged.PagedKVCache.allocate(pages, kv_heads, page, dim, cache)
    q_start = np.concatenate([[0], np.cumsum(news)]).tolist()
    batch = paged.PagedBatch(torch.tensor(q_start, dtype=torch.int32, device="cuda"),
                             torch.tensor(kv_lens, dtype=torch.int32, device="cuda"), table, max_rows=max(news))
    return c, batch, q_start


@pytest.mark.parametrize("rotate_first", [True, False])
@pytest.mark.parametrize("rows_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("kv_lens,news,heads,kv_heads,dim,page", [
    ([5], [1], 16, 8, 128, 16), ([40, 3, 17], [16, 3, 1], 6, 2, 64, 24), ([700, 900], [650, 500], 4, 1, 128, 7),
    ([0, 9, 0], [0, 5, 0], 3, 3, 64, 4)])
def test_into_pages(rotary, paged, cache, rows_dtype, kv_lens, news, heads, kv_heads, dim, page, rotate_first):
    c, batch, q_start = _paged(paged, cache, kv_lens, news, kv_heads, dim, page, 11)
    rows = q_start[-1]
    q, k, v, (qw, kw), cos, sin, pos = _inputs(rows, heads, kv_heads, dim, rows_dtype, 7, table=2000)
    out = c.write_rotated(batch, q, k, v, qw, kw, cos, sin, pos, rotate_first=rotate_first)
    c.check()
    # q, v, and (fp32 rows) k of a plain write of rows that were normed and rotated in fp32, bit by bit; a lane adds up
    # twice as many squares of a bf16 row, in another order, so k of those is held to the formula alone.
    plain, _, _ = _paged(paged, cache, kv_lens, news, kv_heads, dim, page, 11)
    want_q, _ = rotary.norm_rotate(q, k, qw, kw, cos, sin, pos, rotate_first=rotate_first)
    assert torch.equal(out, want_q)
    _, k32 = rotary.norm_rotate(q.float(), k.float(), qw, kw, cos, sin, pos, rotate_first=rotate_first)
    plain.write(batch, k32, v.float())
    same = [torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in ((c.v, plain.v), (c.k, plain.k))]
    if cache in LARGEST:
        same += [torch.equal(c.v_scale, plain.v_scale), torch.equal(c.k_scale, plain.k_scale)]
    assert all(same if rows_dtype == torch.float32 else same[::2])
    # And against the formula, as the cache gives it back.
    got = c.read(batch, rows, torch.float32)[0].double()
    want, reach = _formula(k, kw, cos, sin, pos, 1e-5, rotate_first)
    tol = reach * 24 * 2.0 ** -24
    if cache == torch.bfloat16:
        tol = tol + (want.abs() + tol) * 2.0 ** -8
    elif cache in LARGEST:
        # A code is off by half a step: 2^-4 of itself or, below the normal numbers, 2^-10 (E4M3); 1/2 (INT8). The scale
        # carries the largest element's error.
        scale = want.abs().amax(dim=-1, keepdim=True) / LARGEST[cache]
        step = want.abs() * 2.0 ** -4 + scale * 2.0 ** -10 if cache == torch.float8_e4m3fn else scale / 2
        tol = 2 * tol + step * 1.001 + want.abs() * (tol.amax(dim=-1, keepdim=True) / (scale * LARGEST[cache]) + 2.0 ** -22)
    assert (got - want).abs().le(tol).all()


def test_rows_of_no_sequence_and_padding_stay_as_they_were(rotary, paged):
    c, _, _ = _paged(paged, torch.bfloat16, [4, 6], [2, 2], 2, 64, 8, 3)
    table = torch.tensor([[0], [1]], dtype=torch.int32, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
    batch = paged.PagedBatch(i32(1, 5, 7), i32(2, 6), table, max_rows=4)   # rows 1, 2 are padding; 0, 7, 8 nobody's
    q, k, v, (qw, kw), cos, sin, pos = _inputs(9, 4, 2, 64, torch.float32, 2, table=64)
    out = torch.full_like(q, 7.0, memory_format=torch.contiguous_format)
    c.write_rotated(batch, q, k, v, qw, kw, cos, sin, pos, out=out)
    c.check()
    want = rotary.norm_rotate(q, k, qw, kw, cos, sin, pos)[0]
    assert (out[[0, 1, 2, 7, 8]] == 7).all()
    assert torch.equal(out[3:7], want[3:7])
    assert (c.k[0, :, 2:] == 0).all() and (c.k[1, :, :4] == 0).all() and (c.k[1, :, 4:6] != 0).any()
    assert [p for _, p in filter(None, positions([1, 5, 7], [2, 6], 9))] == [-2, -1, 0, 1, 4, 5]


def test_a_bad_page_takes_its_keys_alone(rotary, paged):
    c, batch, _ = _paged(paged, torch.float32, [10, 10], [3, 3], 1, 64, 16, 4)
    batch.block_table[1, 0] = 10 ** 6
    q, k, v, (qw, kw), cos, sin, pos = _inputs(6, 2, 1, 64, torch.float32, 2, table=64)
    out = c.write_rotated(batch, q, k, v, qw, kw, cos, sin, pos)
    assert torch.equal(out, rotary.norm_rotate(q, k, qw, kw, cos, sin, pos)[0])
    with pytest.raises(Exception, match="page number"):
        c.check()
    assert int((c.k != 0).any(dim=-1).sum()) == 3


def test_captured_and_on_another_stream(rotary, paged):
    c, batch, _ = _paged(paged, torch.float8_e4m3fn, [30, 40], [4, 4], 2, 128, 16, 5)
    q, k, v, (qw, kw), cos, sin, pos = _inputs(8, 4, 2, 128, torch.bfloat16, 6, table=256)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = torch.empty(8, 4, 128, dtype=torch.bfloat16, device="cuda")
    with torch.cuda.stream(side):
        c.write_rotated(batch, q, k, v, qw, kw, cos, sin, pos, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            c.write_rotated(batch, q, k, v, qw, kw, cos, sin, pos, out=out)
    torch.cuda.synchronize()
    # The next step: later positions, other angles, read on the device.
    batch.kv_len += 4
    pos += 4
    graph.replay()
    torch.cuda.synchronize()
    fresh, _, _ = _paged(paged, torch.float8_e4m3fn, [30, 40], [4, 4], 2, 128, 16, 5)
    want = fresh.write_rotated(batch, q, k, v, qw, kw, cos, sin, pos)
    assert torch.equal(out, want)
    assert all(torch.equal(x, y) for x, y in zip(c.read(batch, 8), fresh.read(batch, 8)))


def test_refusals_of_tensors(rotary, pkg):
    q, k, _, (qw, kw), cos, sin, pos = _inputs(4, 4, 2, 64, torch.float32, 2, table=16)
    for args, kw_ in (((q, k[:3], qw, kw, cos, sin, pos), {}), ((q, k.bfloat16(), qw, kw, cos, sin, pos), {}),
                      ((q, k, qw[:32], kw, cos, sin, pos), {}), ((q, k, qw, kw.double(), cos, sin, pos), {}),
                      ((q, k, qw, kw, cos[:, :32], sin, pos), {}), ((q, k, qw, kw, cos, sin[:5], pos), {}),
                      ((q, k, qw, kw, cos, sin, pos.long()), {}), ((q, k, qw, kw, cos, sin, pos[:3]), {}),
                      ((q, k, qw, kw, cos[:3], sin[:3], None), {}), ((q.cpu(), k, qw, kw, cos, sin, pos), {}),
                      ((q.half(), k.half(), qw, kw, cos, sin, pos), {}), ((q, k, qw, kw, cos, sin, pos), {"eps": -1.0}),
                      ((q.detach().requires_grad_(), k, qw, kw, cos, sin, pos), {})):
        with pytest.raises(pkg.HyError):
            rotary.norm_rotate(*args, **kw_)
