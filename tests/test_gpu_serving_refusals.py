"""Calls of the norms, the paged cache and the log probabilities that are refused, and ones beside them that are not, on the
GPU."""

import importlib

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mods(pkg):
    return [importlib.import_module("hy_b200." + m) for m in ("paged", "rotary", "logprobs")]


def _projection(rows, heads, dim, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(rows, heads, dim, generator=gen, device="cuda").to(dtype)


def _angles(rows, dim):
    a = torch.arange(rows, device="cuda")[:, None] * (1 + torch.arange(dim, device="cuda") % (dim // 2)) * 0.01
    return a.cos(), a.sin()


def test_forward_mode_tangents(mods, pkg):
    _, rotary, logprobs = mods
    x = _projection(3, 6, 64, torch.float32, 1)
    cos, sin = _angles(3, 64)
    w = torch.ones(64, device="cuda")
    q, k = x[:, :4], x[:, 4:]
    logits, tokens = _projection(3, 1, 100, torch.float32, 2)[:, 0], torch.zeros(3, dtype=torch.int32, device="cuda")
    with forward_ad.dual_level():
        for args in ((forward_ad.make_dual(q, q), k), (q, forward_ad.make_dual(k, k))):
            with pytest.raises(pkg.HyError, match="tangent"):
                rotary.norm_rotate(*args, w, w, cos, sin)
        out = forward_ad.make_dual(torch.empty_like(q), torch.empty_like(q))
        with pytest.raises(pkg.HyError, match="tangent"):
            rotary.norm_rotate(q, k, w, w, cos, sin, out=(out, torch.empty_like(k)))
        with pytest.raises(pkg.HyError, match="tangent"):
            logprobs.token_logprobs(forward_ad.make_dual(logits, logits), tokens)
        got = rotary.norm_rotate(q, k, w, w, cos, sin)   # (a level alone refuses nothing)
    assert all(torch.equal(a, b) for a, b in zip(got, rotary.norm_rotate(q, k, w, w, cos, sin)))
    assert logprobs.token_logprobs(logits, tokens).logprob.shape == (3,)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 50, 700])
def test_outputs_beside_their_inputs_in_one_projection(mods, pkg, rows, dtype):
    """Interleaved views share no element and are right; those that share some are refused."""
    _, rotary, _ = mods
    x = _projection(rows, 13, 64, dtype, rows)
    cos, sin = _angles(rows, 64)
    w = torch.rand(64, device="cuda") + 0.5
    q, k = x[:, :4], x[:, 4:6]
    want = rotary.norm_rotate(q, k, w, w, cos, sin)
    held = x.clone()
    for a, b in ((6, 11), (0, 4), (8, 4), (0, 11)):   # first heads of the outputs
        x.copy_(held)
        out = x[:, a:a + 4], x[:, b:b + 2]
        rotary.norm_rotate(q, k, w, w, cos, sin, out=out)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        rest = [h for h in range(13) if not a <= h < a + 4 and not b <= h < b + 2]
        assert torch.equal(x[:, rest], held[:, rest])
    x.copy_(held)
    for a, b in ((7, 0), (2, 11), (1, 4), (6, 5), (6, 3), (6, 9)):
        with pytest.raises(pkg.HyError, match="overlap"):
            rotary.norm_rotate(q, k, w, w, cos, sin, out=(x[:, a:a + 4], x[:, b:b + 2]))
    assert torch.equal(x, held)


def test_a_table_without_rows(mods):
    """No rows give nothing; rows whose positions lie outside the empty table are NaN, and reported."""
    paged, rotary, _ = mods
    x = _projection(3, 6, 64, torch.float32, 1)
    cos = torch.ones(0, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    a, b = rotary.norm_rotate(x[:0, :4], x[:0, 4:], w, w, cos, cos)
    assert a.shape == (0, 4, 64) and b.shape == (0, 2, 64)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    a, b = rotary.norm_rotate(x[:, :4], x[:, 4:], w, w, cos, cos, torch.zeros(3, dtype=torch.int32, device="cuda"), status=status)
    assert torch.isnan(a).all() and torch.isnan(b).all() and status.item() == 16
    cache = paged.PagedKVCache.allocate(2, 2, 16, 64, torch.float32)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
    batch = paged.PagedBatch(i32(0, 0), i32(0), i32(0)[:, None], 1)
    assert cache.write_rotated(batch, x[:0, :2], x[:0, 2:4], x[:0, 4:], w, w, cos, cos).shape == (0, 2, 64)
