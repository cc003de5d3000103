"""Log probabilities, entropy and alternatives on the GPU, against the definitions in 64 bits."""

import importlib
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

INF = math.inf


@pytest.fixture(scope="module")
def call(pkg):
    return importlib.import_module("hy_b200.logprobs").token_logprobs


def _reference(x, tokens, top):
    """(values, tolerances) of a call, per output. With d = x - max, s, t and u the sums of e^d, |d| e^d and d^2 e^d over
    the logits below the largest, c the count of the largest: an exponential is off by 2^-22 (ex2) and 2^-23 |d| (its
    argument), once more at each of at most 2^5 rescalings, and s collects at most 2^6 roundings of 2^-24; so s is off by
    at most s 2^-16 + t 2^-20 and t by t 2^-16 + u 2^-20. log(c + s) and the rest: a few roundings of themselves."""
    x = x.double()
    m = x.amax(dim=1, keepdim=True)
    d = x - m
    e = torch.where(d < 0, torch.exp(d), 0.0)
    c = (d == 0).sum(dim=1).double()
    dd = torch.where(e > 0, -d, 0.0)
    s, t, u = e.sum(dim=1), (dd * e).sum(dim=1), (dd * dd * e).sum(dim=1)
    less = torch.log1p(s + (c - 1))
    err_s, err_t = s * 2.0 ** -16 + t * 2.0 ** -20, t * 2.0 ** -16 + u * 2.0 ** -20
    err_less = err_s / (c + s) + less * 2.0 ** -22
    entropy = less + t / (c + s)
    err_entropy = err_less + err_t / (c + s) + t / (c + s) * err_s / (c + s) + entropy * 2.0 ** -22
    lp = torch.where(((tokens >= 0) & (tokens < x.shape[1])),
                     d.gather(1, tokens.long().clamp(0, x.shape[1] - 1)) - less[:, None], math.nan)
    ids = np.array([np.lexsort((np.arange(x.shape[1]), -r))[:top] for r in x.cpu().numpy()]).reshape(len(x), top)
    ids = torch.from_numpy(ids).to(x.device)
    alt = d.gather(1, ids) - less[:, None]
    ids = torch.where(torch.isinf(alt), -1, ids)
    err = [(err_less[:, None] + torch.where(torch.isfinite(v), v.abs(), 0.0) * 2.0 ** -22) for v in (lp, alt)]
    return (lp, entropy, ids, alt), (err[0], err_entropy, err[1])


def _check(got, x, tokens, top):
    tok = tokens if tokens.dim() == 2 else tokens[:, None]
    (lp, entropy, ids, alt), (e_lp, e_h, e_alt) = _reference(x, tok, top)

    def near(a, b, tol):
        a = a.double()
        same = (a == b) | (torch.isnan(a) & torch.isnan(b))
        assert (same | ((a - b).abs() <= tol)).all(), float(torch.nan_to_num(a - b).abs().max())

    near(got.logprob.view(lp.shape), lp, e_lp)
    near(got.entropy, entropy, e_h)
    if top:
        assert torch.equal(got.top_ids.long(), ids)
        near(got.top_logprobs, alt, e_alt)
    else:
        assert got.top_ids is None and got.top_logprobs is None


def _logits(rows, vocab, dtype, seed, spread=2.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=gen, device="cuda") * spread).to(dtype)
    return x, torch.randint(vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (3, 2, 2), (2, 7, 0), (5, 64, 64), (1, 257, 20), (4, 2047, 5), (1, 4099, 64), (9, 8193, 1), (1, 120818, 20),
    (16, 120818, 5), (700, 5003, 8), (2, 262147, 3), (1, 1 << 20, 64)])
def test_sizes(call, rows, vocab, top, dtype):
    x, tokens = _logits(rows, vocab, dtype, rows + vocab)
    _check(call(x, tokens, top), x, tokens, top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", range(0, 8))
def test_rows_at_any_address(call, dtype, shift):
    """Rows that start and end inside 16 bytes, with what must not be read around them."""
    held = torch.full((5, 1031), INF, dtype=dtype, device="cuda")
    x, tokens = _logits(5, 1001, dtype, shift)
    view = held[:, shift:shift + 1001]
    view.copy_(x)
    _check(call(view, tokens, 7), x, tokens, 7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_tokens(call, dtype):
    x, tokens = _logits(6, 9000, dtype, 1)
    gen = torch.Generator(device="cuda").manual_seed(2)
    x[:3] = x[:3].masked_fill(torch.rand(3, 9000, generator=gen, device="cuda") < 0.5, -INF)
    x[3, 3:] = -INF               # fewer left than alternatives asked for
    x[4] = -INF
    x[4, 8999] = -3.0             # one alone
    x[5, 100:] = torch.finfo(dtype).min   # masked by the type's lowest value
    tokens[:] = torch.tensor([0, 1, 2, 7000, 8999, 50])
    got = call(x, tokens, 5)
    _check(got, x, tokens, 5)
    assert got.logprob[4] == 0 and got.entropy[4] == 0 and got.logprob[3] == -INF
    assert got.top_ids[4].tolist() == [8999, -1, -1, -1, -1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("split", [1, 700])   # eight CTAs a row, and one
def test_equal_logits(call, dtype, split):
    """Ties go to the lower token: a few, many more than any list holds, zeros of both signs."""
    x = torch.zeros(split + 4, 20000, dtype=dtype, device="cuda")
    x[0, 5000:9000] = 1.0
    x[1, ::2] = -0.0
    x[2, 19990:] = 2.0
    x[3, 1::3] = 4.0
    tokens = torch.full((split + 4,), 5000, dtype=torch.int32, device="cuda")
    _check(call(x, tokens, 20), x, tokens, 20)


def test_strided_masks_that_leave_few_threads_anything(call):
    """What is left lies in one thread's share of the row: more of it than the list holds."""
    x = torch.full((1, 120818), -INF, device="cuda")
    kept = torch.arange(120818, device="cuda") % 1024 < 4
    x[0, kept] = torch.randn(int(kept.sum()), device="cuda")
    rows = x.expand(600, -1).contiguous()   # (one CTA a row)
    for y in (x, rows):
        tokens = torch.zeros(len(y), dtype=torch.int32, device="cuda")
        got = call(y, tokens, 64)
        _check(type(got)(*(t[:1] for t in got)), y[:1], tokens[:1], 64)
        assert (got.top_ids == got.top_ids[0]).all()


def test_rising_and_falling_logits(call):
    up = torch.arange(50000, device="cuda").float() * 1e-3
    x = torch.stack([up, up.flip(0), up.abs().sin() * 5])
    tokens = torch.tensor([0, 49999, 7], dtype=torch.int32, device="cuda")
    _check(call(x, tokens, 10), x, tokens, 10)


def test_near_certain_tokens_keep_their_precision(call):
    x, tokens = _logits(8, 3000, torch.float32, 3, spread=1.0)
    x[torch.arange(8), tokens.long()] = torch.arange(8, device="cuda") * 5.0 + 10.0
    got = call(x, tokens, 2)
    _check(got, x, tokens, 2)
    # (log_softmax loses this in 64 bits too: 1 plus what is left, 1e-16, is 1)
    others = x.double() - x.double().gather(1, tokens.long()[:, None])
    others[torch.arange(8), tokens.long()] = -INF
    want = -torch.log1p(others.exp().sum(dim=1))
    assert -1e-15 < want[-1] < 0 and bool(((got.logprob.double() - want).abs() <= 1e-4 * want.abs()).all())


def test_rows_without_an_answer(call):
    """NaN, +infinity, nothing above -infinity: NaN and -1, whatever their place; other rows are as ever."""
    x, tokens = _logits(12, 30000, torch.float32, 4)
    x[0, 0] = math.nan
    x[1, 29999] = math.nan
    x[2, 15000] = INF
    x[3] = -INF
    x[4] = math.nan
    x[5, 7], x[5, 20000] = INF, math.nan
    for y in (x, x.repeat(60, 1)):
        tok = tokens.repeat(len(y) // 12)
        got = call(y, tok, 3)
        bad = torch.arange(len(y), device="cuda") % 12 < 6
        assert torch.isnan(got.logprob[bad]).all() and torch.isnan(got.entropy[bad]).all()
        assert (got.top_ids[bad] == -1).all() and torch.isnan(got.top_logprobs[bad]).all()
        _check(type(got)(*(t[~bad] for t in got)), y[~bad], tok[~bad], 3)


def test_several_tokens_a_row_and_tokens_outside(call):
    x, _ = _logits(7, 500, torch.float32, 5)
    gen = torch.Generator(device="cuda").manual_seed(1)
    tokens = torch.randint(-20, 520, (7, 300), generator=gen, device="cuda", dtype=torch.int32)
    tokens[0, :3] = torch.tensor([-1, 500, 2 ** 31 - 1])
    _check(call(x, tokens, 0), x, tokens, 0)
    none = call(x, tokens[:, :0].contiguous(), 4)
    assert none.logprob.shape == (7, 0) and none.top_ids.shape == (7, 4)
    empty = call(x[:0], tokens[:0], 4)
    assert empty.logprob.shape == (0, 300) and empty.top_ids.shape == (0, 4)


def test_captured_and_repeated(call):
    x, tokens = _logits(20, 120818, torch.bfloat16, 6)
    first = call(x, tokens, 8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call(x, tokens, 8)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(first, held))
    x.copy_(x.roll(1, 0))
    tokens.copy_(tokens.roll(1))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(call(x, tokens, 8), held))   # what the arrays hold now
    assert torch.equal(held.top_ids, first.top_ids.roll(1, 0))


def test_refusals_of_tensors(call, pkg):
    x, tokens = _logits(3, 100, torch.float32, 7)
    for a in ((x.half(), tokens), (x.cpu(), tokens), (x.t(), tokens), (x, tokens.long()), (x, tokens[:2]), (x[0], tokens),
              (x, tokens.cpu()), (x.detach().requires_grad_(), tokens)):
        with pytest.raises(pkg.HyError):
            call(*a)
    for top in (-1, 65, 101):
        with pytest.raises(pkg.HyError):
            call(x, tokens, top)


def test_behind_a_runtimes_lm_head(pkg):
    """hy_lm_head_logprobs against the logits that the same head gives."""
    rt = pkg.TextRuntime.synthetic(seed=3, std=0.02, norm_std=0.1, num_layers=1, vocab_size=4099, max_context=64,
                                   max_prefill=32, max_tokens=16, device=0)
    try:
        rng = np.random.default_rng(1)
        for rows in (1, 5, 16):
            hidden = rng.standard_normal((rows, 1024)).astype(np.float32) * 3
            tokens = rng.integers(0, 4099, rows).astype(np.int32)
            _, raw, logits = rt.select_logit_rows(hidden, 1.0, want_logits=True)
            lp, entropy, ids, alt = rt.lm_head_logprobs(hidden, tokens, top=4)
            x = torch.from_numpy(logits)
            got = importlib.import_module("hy_b200.logprobs").TokenLogprobs(*(torch.from_numpy(t) for t in (lp, entropy, ids, alt)))
            _check(got, x, torch.from_numpy(tokens), 4)
            assert (ids[:, 0] == raw).all()
            none, entropy2, no_ids, no_alt = rt.lm_head_logprobs(hidden)
            assert none is None and no_ids is None and no_alt is None and (entropy2 == entropy).all()
        with pytest.raises(pkg.HyError):
            rt.lm_head_logprobs(hidden, tokens[:3])
        with pytest.raises(pkg.HyError):
            rt.lm_head_logprobs(hidden, tokens, top=65)
        with pytest.raises(pkg.HyError):
            rt.lm_head_logprobs(np.zeros((17, 1024), np.float32))
    finally:
        rt.close()
