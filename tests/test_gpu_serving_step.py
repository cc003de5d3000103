"""The operators of a server's step together, as they are used: projections of a layer -> norms and rotation on the way into
pages -> attention with its sums' logarithms -> attention weights -> eviction, step by step, and log probabilities behind
the LM head; against the same steps written out in 64 bits over plain lists of keys."""

import importlib
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, KEEP, RECENT, FIRST, SCALE = 4, 2, 64, 24, 8, 2, 0.125


@pytest.fixture(scope="module")
def mods(pkg):
    return [importlib.import_module("hy_b200." + m) for m in ("paged", "rotary", "logprobs")]


class Plain:
    """One sequence in 64 bits: per KV head its keys, values and their weights."""

    def __init__(self):
        self.k = [torch.zeros(0, DIM, dtype=torch.float64, device="cuda") for _ in range(KV)]
        self.v = [x.clone() for x in self.k]
        self.w = [torch.zeros(0, dtype=torch.float64, device="cuda") for _ in range(KV)]

    def step(self, q, k, v):
        """q, k normed and rotated [n, heads, dim]; the attention's output."""
        n, out = len(q), torch.zeros_like(q)
        for h in range(KV):
            self.k[h], self.v[h] = torch.cat([self.k[h], k[:, h]]), torch.cat([self.v[h], v[:, h]])
            old = len(self.w[h])
            self.w[h] = torch.cat([self.w[h], torch.zeros(n, dtype=torch.float64, device="cuda")])
            seen = torch.arange(old + n, device="cuda")[None] <= torch.arange(old, old + n, device="cuda")[:, None]
            for g in range(HEADS // KV):
                s = (q[:, h * (HEADS // KV) + g] @ self.k[h].T * SCALE).masked_fill(~seen, -math.inf)
                p = torch.softmax(s, dim=1)
                out[:, h * (HEADS // KV) + g] = p @ self.v[h]
                self.w[h] = self.w[h] + p.sum(dim=0)
        return out

    def evict(self):
        kept = []
        for h in range(KV):
            n = len(self.w[h])
            w = self.w[h].clone()
            w[:FIRST] = w[n - RECENT:] = math.inf
            at = torch.sort(w, descending=True, stable=True).indices[:KEEP].sort().values
            kept.append(at)
            self.k[h], self.v[h], self.w[h] = self.k[h][at], self.v[h][at], self.w[h][at]
        return torch.stack(kept)


def _formula(x, w, cos, sin, eps):
    c, s = cos.double()[:, None], sin.double()[:, None]
    y = x.double() * c + torch.cat([-x[..., DIM // 2:], x[..., :DIM // 2]], dim=-1).double() * s
    return y * w.double() / torch.sqrt((y * y).mean(dim=-1, keepdim=True) + eps)


def test_steps_of_two_records(mods):
    paged, rotary, logprobs = mods
    gen = torch.Generator(device="cuda").manual_seed(5)

    def rand(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    hidden, vocab, page = 96, 500, 8
    wqkv, wo, head = rand(hidden, (HEADS + 2 * KV) * DIM) / 10, rand(HEADS * DIM, hidden) / 16, rand(hidden, vocab) / 10
    qw, kw = 1 + 0.1 * rand(DIM), 1 + 0.1 * rand(DIM)
    angle = torch.arange(200, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-(torch.arange(DIM, device="cuda") % 32) / 32.0)
    cos, sin = angle.cos().float(), angle.sin().float()
    cache = paged.PagedKVCache.allocate(40, KV, page, DIM, torch.float32)
    weights = cache.allocate_weights()
    table = torch.randperm(40, generator=gen, device="cuda")[:40].view(2, 20).int()
    kv_len = torch.zeros(2, dtype=torch.int32, device="cuda")
    plain, position, evictions = [Plain(), Plain()], [0, 0], 0
    for step in range(40):
        new = [31, 12] if step == 0 else [1, 1]   # the prompts, then a token each
        q_start = torch.tensor([0, new[0], sum(new)], dtype=torch.int32, device="cuda")
        kv_len += torch.tensor(new, dtype=torch.int32, device="cuda")
        batch = paged.PagedBatch(q_start, kv_len, table, max_rows=max(new))
        where = torch.cat([torch.arange(p, p + n) for p, n in zip(position, new)]).int().cuda()
        x = rand(sum(new), hidden)
        rows = (x @ wqkv).view(sum(new), HEADS + 2 * KV, DIM)
        q, k, v = rows[:, :HEADS], rows[:, HEADS:HEADS + KV], rows[:, HEADS + KV:]
        turned = cache.write_rotated(batch, q, k, v, qw, kw, cos, sin, where)
        out, lse = cache.attention(batch, turned, SCALE, return_lse=True)
        cache.add_weights(batch, turned, lse, SCALE, weights)
        got = logprobs.token_logprobs(out.reshape(sum(new), -1) @ wo @ head, torch.full((sum(new),), 7, dtype=torch.int32, device="cuda"), top=3)
        kept = cache.evict(batch, KEEP, weights, recent=RECENT, first=FIRST) if step % 10 == 9 else None
        cache.check()
        # ---- the same in 64 bits ----
        at = where.long()
        q64, k64 = _formula(q, qw, cos[at], sin[at], 1e-5), _formula(k, kw, cos[at], sin[at], 1e-5)
        for s, (a, b) in enumerate(((0, new[0]), (new[0], sum(new)))):
            want = plain[s].step(q64[a:b], k64[a:b], v[a:b].double())
            # (fp32 throughout, keys of unit variance: 2^-12 is a thousand times the parts' tolerances)
            assert (out[a:b].double() - want).abs().max() < 2.0 ** -12
            if kept is not None and len(plain[s].w[0]) > KEEP:
                assert torch.equal(kept[s].long(), plain[s].evict())
                evictions += 1
            n = len(plain[s].w[0])
            assert kv_len[s] == n
            j = torch.arange(n, device="cuda")
            held = weights[table[s, j // page].long(), :, j % page]
            assert (held.double() - torch.stack(plain[s].w, dim=1)).abs().max() < 2.0 ** -12
        want = torch.log_softmax((out.reshape(sum(new), -1) @ wo @ head).double(), dim=1)
        assert (got.logprob.double() - want[:, 7]).abs().max() < 1e-5
        assert torch.equal(got.top_ids.long(), torch.topk(want, 3, dim=1).indices)
        position = [p + n for p, n in zip(position, new)]
    assert evictions >= 6


def test_a_captured_step_follows_lengths_and_positions(mods):
    """norms + write, attention, weights and log probabilities of a token in one graph, replayed as the records grow."""
    paged, rotary, logprobs = mods
    gen = torch.Generator(device="cuda").manual_seed(6)
    cos, sin = (torch.randn(64, DIM, generator=gen, device="cuda") for _ in range(2))
    w = torch.ones(DIM, device="cuda")
    table = torch.arange(12, device="cuda").view(3, 4).int()
    q_start = torch.arange(4, device="cuda").int()
    x = torch.empty(3, HEADS + 2 * KV, DIM, device="cuda")

    def build():
        cache = paged.PagedKVCache.allocate(12, KV, 16, DIM, torch.bfloat16)
        kv_len = torch.tensor([1, 5, 17], dtype=torch.int32, device="cuda")
        return cache, cache.allocate_weights(), paged.PagedBatch(q_start, kv_len, table, 1), torch.zeros(3, dtype=torch.int32, device="cuda")

    def step(cache, weights, batch, where):
        q = cache.write_rotated(batch, x[:, :HEADS], x[:, HEADS:HEADS + KV], x[:, HEADS + KV:], w, w, cos, sin, where)
        out, lse = cache.attention(batch, q, SCALE, return_lse=True)
        cache.add_weights(batch, q, lse, SCALE, weights)
        return out, logprobs.token_logprobs(out.view(3, -1), where, top=2).top_logprobs

    one, two = build(), build()
    x.normal_(generator=gen)
    step(*build())   # (kernels are loaded before the capture)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(*one)
    for _ in range(6):
        x.normal_(generator=gen)
        graph.replay()
        want = step(*two)
        assert all(torch.equal(a, b) for a, b in zip(held, want))
        assert torch.equal(one[1], two[1]) and torch.equal(one[0].k, two[0].k)
        for _, _, batch, where in (one, two):
            batch.kv_len += 1
            where += 1
