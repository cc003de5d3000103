"""Cases of the operators around the paged KV cache and behind the LM head: norms of the query and key
heads with the position rotation in the same pass (alone, and on the way into the cache), attention
weights added up for every cached position, eviction of the positions with the least of it, and log
probabilities of given tokens with entropy and top alternatives.

A case's `kind` is "rotate" (norm and rotation of rows), "enter" (the same, k and v written to pages),
"weigh" (attention weights of new rows added to what the cached positions have), "evict" (the cache cut to
`keep` positions of a head) or "score" (log probabilities). Where there is a cache, sequence s has
kv_len[s] rows in it, the last n[s] of them new; both are drawn from the case's `lens`.
"""

import math
import random

import numpy as np
import torch

own = False

HEADS, KV_HEADS, DIM = 16, 8, 128   # the decoder's attention geometry
SCALE = 0.0883883                   # the decoder's attention scale at 128 dimensions
VOCAB = 120818                      # the decoder's vocabulary
CONTEXT = 8256                      # positions of its rotation table
EPS = 1e-5
THETA = 10000.0
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
LARGEST = {"e4m3": 448.0, "int8": 127.0}
TINY = 2.0 ** -126


def _heads(name, kind, rows, heads=HEADS, kv_heads=KV_HEADS, dim=DIM):
    return {"name": name, "kind": kind, "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim}


def _cached(name, kind, cache, rows, seqs, kv, new, page=16, lens=1, **more):
    geometry = {k: more.pop(k) for k in ("heads", "kv_heads", "dim") if k in more}
    return {**_heads(name, kind, rows, **geometry), "cache": cache, "seqs": seqs, "kv_min": kv[0], "kv_max": kv[1],
            "new_min": new[0], "new_max": new[1], "page": page, "lens": lens, **more}


def _scored(name, rows, count, top, vocab=VOCAB, masked=0.0):
    return {"name": name, "kind": "score", "rows": rows, "count": count, "vocab": vocab, "top": top, "masked": masked}


def listed():
    return [
        # One decode step of one record: rotation first, then the norm, rows of the fp32 projections. Latency alone.
        {**_heads("rotate_token_f32", "rotate", "f32"), "count": 1, "rotate_first": True, "table": CONTEXT},
        # Prompts of many records, other heads (eight query heads per KV head of 64), norm first, an odd count.
        {**_heads("rotate_prompts_bf16", "rotate", "bf16", 32, 4, 64), "count": 20011, "rotate_first": False,
         "table": CONTEXT},
        # Verify blocks of 16 rows of four records into a bf16 cache.
        _cached("enter_verify", "enter", "bf16", "f32", 4, (1500, 2600), (16, 16), lens=2, rotate_first=True),
        # Prompts of 16 records admitted together, odd lengths, bf16 rows, an 8-bit cache.
        _cached("enter_prompts_e4m3", "enter", "e4m3", "bf16", 16, (700, 4096), (700, 4096), lens=3,
                rotate_first=True),
        # One AR token of one record at 2048 rows, fp32 throughout.
        _cached("weigh_token_f32", "weigh", "f32", "f32", 1, (2048, 2048), (1, 1), window=0, sinks=0),
        # 64 records at long contexts, one token each, 8-bit cache: the serving step that memory bounds.
        _cached("weigh_serving_e4m3", "weigh", "e4m3", "bf16", 64, (1024, 8192), (1, 1), page=64, lens=4, window=0,
                sinks=0),
        # Prompt chunks of four records behind long prefixes: what the tensor cores bound.
        _cached("weigh_chunks", "weigh", "bf16", "bf16", 4, (6000, 8192), (1000, 1024), lens=5, window=0, sinks=0),
        # One record's prompt cut to 1024 positions of a head.
        _cached("evict_prompt", "evict", "bf16", "f32", 1, (4111, 4111), (1, 1), lens=6, keep=1024, recent=256,
                first=4),
        # 64 records that have grown by up to 128 tokens since they were last cut; some are short still.
        _cached("evict_records_e4m3", "evict", "e4m3", "bf16", 64, (900, 1152), (1, 1), page=64, lens=7, keep=1024,
                recent=256, first=4),
        # One step's token of one record, with the alternatives that an API shows.
        _scored("score_token", "f32", 1, 20),
        # A step of a batch, bf16 logits, some tokens masked out.
        _scored("score_batch_bf16", "bf16", 16, 5, masked=0.02),
        # Every token of a long prompt.
        _scored("score_prompt", "f32", 1024, 8),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    top = {f: max(work(c)[f] for c in listed()) for f in ("bytes", "flops")}
    while True:
        kind = rng.choice(["rotate", "enter", "weigh", "weigh", "evict", "score"])
        rows = rng.choice(["f32", "bf16"])
        kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
        heads = kv_heads * rng.choice([1, 2, 2, 4, 5, 8])
        dim = rng.choice([64, 128])
        if kind == "rotate":
            case = {**_heads("", kind, rows, heads, kv_heads, dim), "count": log(1, 20000),
                    "rotate_first": rng.random() < 0.5, "table": rng.choice([0, CONTEXT])}
        elif kind == "score":
            case = _scored("", rows, log(1, 1024), rng.choice([0, 1, 5, 8, 20]), vocab=log(500, 200000),
                          masked=rng.choice([0.0, 0.02, 0.5]))
        else:
            cache = rng.choice(["f32", "bf16", "e4m3"] + (["int8"] if kind == "weigh" else []))
            kv_max = log(2, 16384)
            kv_min = rng.randint(1, kv_max)
            new = (1, 1)
            if kind == "weigh":
                new_max = min(kv_max, rng.choice([1, 1, log(2, 40), log(16, 2048)]))
                new = (rng.randint(1, new_max), new_max)
                window = rng.choice([0, 0, log(16, 4096)])
                more = {"window": window, "sinks": rng.choice([0, 4, 33]) if window else 0}
            elif kind == "enter":
                new_max = log(1, kv_max)
                new = (rng.randint(1, new_max), new_max)
                more = {"rotate_first": rng.random() < 0.5}
            else:
                keep = log(2, kv_max)
                recent = rng.randint(0, keep)
                more = {"keep": keep, "recent": recent, "first": rng.randint(0, min(keep - recent, 8))}
            case = _cached("", kind, cache, rows, log(1, 64), (kv_min, kv_max), new,
                           page=rng.choice([1, 8, 16, 16, 24, 32, 64, 100, 128]), lens=rng.randint(1, 10 ** 6),
                           heads=heads, kv_heads=kv_heads, dim=dim, **more)
        del case["name"]
        w = work(case)
        # (the plain form holds scores and keys padded to the longest sequence)
        wide = case["seqs"] * case["kv_max"] if "seqs" in case else 0
        if (w["bytes"] <= top["bytes"] and w["flops"] <= top["flops"] and wide * kv_heads * dim <= 6e8 and
                wide * heads * case.get("new_max", 1) <= 7e8):
            return case


def lengths(case):
    """kv_len and the count of new rows of every sequence."""
    rng = random.Random(case["lens"])
    kv = [rng.randint(case["kv_min"], case["kv_max"]) for _ in range(case["seqs"])]
    if case["new_min"] == case["kv_min"] and case["new_max"] == case["kv_max"]:
        return kv, list(kv)   # whole sequences
    return kv, [min(n, rng.randint(case["new_min"], case["new_max"])) for n in kv]


def _visible(case, kv, n):
    """Keys that each of the n new rows sees, added up, and the keys that any of them sees."""
    w, s = case["window"], case["sinks"]
    p = np.arange(kv - n, kv, dtype=np.int64)
    if not w:
        return int((p + 1).sum()), kv
    first = np.maximum(p - w + 1, 0)
    return int((p + 1 - first + np.minimum(first, s)).sum()), int(kv - first[0] + min(int(first[0]), s))


def work(case):
    e_rows = TYPES[case["rows"]].itemsize
    if case["kind"] == "score":
        n, top = case["count"], case["top"]
        return {"bytes": n * (case["vocab"] * e_rows + 12 + 8 * top), "flops": 5 * n * case["vocab"]}
    h, hq, d = case["kv_heads"], case["heads"], case["dim"]
    if case["kind"] == "rotate":   # rows in and out, their angles (a table's rows once at most), the norms' weights
        n = case["count"]
        angles = min(n, case["table"]) if case["table"] else n
        return {"bytes": 2 * n * (hq + h) * d * e_rows + 8 * angles * d + 8 * d, "flops": 8 * n * (hq + h) * d}
    kv, new = lengths(case)
    row = h * (d * TYPES[case["cache"]].itemsize + (4 if case["cache"] in LARGEST else 0))   # one position's keys
    if case["kind"] == "enter":
        n = sum(new)
        return {"bytes": n * ((2 * hq + 2 * h) * d * e_rows + 2 * row + 8 * d) + 8 * d, "flops": n * d * (8 * hq + 10 * h)}
    if case["kind"] == "evict":
        keep = case["keep"]
        # Of sequences that are cut, the kept rows behind the first position that goes move (it lies, on the average,
        # where (kv + 1) / (gone + 1) does); weights are read, those of kept positions and the list of these written.
        moved = [keep - min(keep, (n + 1) / (n - keep + 1)) for n in kv if n > keep]
        cut = [n for n in kv if n > keep]
        return {"bytes": sum(moved) * 4 * row + 4 * h * (sum(cut) + keep * (len(cut) + len(kv))), "flops": 4 * h * sum(cut)}
    seen = [_visible(case, a, b) for a, b in zip(kv, new)]
    keys = sum(k for _, k in seen)
    return {"bytes": keys * (row + 8 * h) + sum(new) * hq * (d * e_rows + 4), "flops": 2 * d * hq * sum(t for t, _ in seen)}


# ---------------------------------------------------------------------------
# The plain form.
# ---------------------------------------------------------------------------
def _rotated(st, x, weight):
    """Heads x [n, heads, dim], normed and rotated in 32 bits."""
    x, half = x.float(), x.shape[-1] // 2
    cos, sin = st["cos"], st["sin"]
    if st["positions"] is not None:
        cos, sin = cos[st["positions"]], sin[st["positions"]]
    cos, sin = cos[:, None], sin[:, None]

    def turn(y):
        return y * cos + torch.cat([-y[..., half:], y[..., :half]], dim=-1) * sin

    def norm(y):
        return y * torch.rsqrt((y * y).mean(dim=-1, keepdim=True) + EPS) * weight

    return norm(turn(x)) if st["rotate_first"] else turn(norm(x))


def _scales(x, cache):
    """Scale of every row: its largest magnitude over the type's largest value, never below 2^-126."""
    amax = x.float().abs().amax(dim=-1)
    return (amax / torch.full_like(amax, LARGEST[cache])).clamp_min(TINY)


def _codes(x, scale, cache):
    """x / scale rounded to the 8-bit type, ties to even; the quotient in 64 bits, so that it is never rounded onto a tie."""
    y = x.double() / scale.double()[..., None]
    if cache == "int8":
        return y.round().to(torch.int8)
    # E4M3: a step of 2^(e - 3), e the value's exponent, not below 2^-9.
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return ((y / step).round() * step).float().to(torch.float8_e4m3fn)


def _bytes(x):
    """8-bit floats as bytes: what indexes and copies them."""
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def _sequence(counts, total, first):
    """Sequence of every one of `total` entries, and its number in it; first: where each sequence's entries start."""
    seq = torch.repeat_interleave(torch.arange(len(counts), device=counts.device), counts, output_size=total)
    return seq, torch.arange(total, device=counts.device) - first[seq]


def _enter(st):
    seq, i = _sequence(st["new"], st["total"], st["q_start"][:-1])
    at = i + (st["kv_len"] - st["new"])[seq]
    pages, rows = st["table"][seq, at // st["page"]].long(), at % st["page"]
    q = _rotated(st, st["q"], st["q_weight"]).to(st["q"].dtype)
    for which, x in (("k", _rotated(st, st["k_rows"], st["k_weight"])), ("v", st["v_rows"])):
        if st["cache"] in LARGEST:
            scale = _scales(x, st["cache"])
            st[which + "_scale"][pages, :, rows] = scale
            _bytes(st[which])[pages, :, rows] = _bytes(_codes(x, scale, st["cache"]))
        else:
            st[which][pages, :, rows] = x.to(st[which].dtype)
    return q


def _weigh(st):
    page, heads, h, n = st["page"], st["q"].shape[1], st["k"].shape[1], st["most"]
    kv, new = st["kv_len"].long(), st["new"]
    dev, s = kv.device, len(kv)
    # Keys of all sequences [s, h, dim, longest], rows [s, h, group * n, dim], both padded.
    j = torch.arange(st["longest"], device=dev)
    pages, rows = st["table"][:, j // page].long(), j % page
    k = st["k"][pages, :, rows].float()
    if st["k_scale"] is not None:
        k = k * st["k_scale"][pages, :, rows][..., None]
    k = k.permute(0, 2, 3, 1)
    i = torch.arange(n, device=dev)
    r = (st["q_start"][:-1, None] + i).clamp_max(st["total"] - 1)
    q = st["q"][r].float().view(s, n, h, heads // h, -1).permute(0, 2, 3, 1, 4)
    lse = st["lse"][r].view(s, n, h, heads // h).permute(0, 2, 3, 1)
    y = q.reshape(s, h, -1, q.shape[-1]) @ k * st["scale"]
    y = torch.exp(y.view(s, h, heads // h, n, -1) - lse[..., None])
    p = (kv - new)[:, None] + i
    seen = (j <= p[..., None]) & (i < new[:, None])[..., None]
    if st["window"]:
        seen &= (p[..., None] - j < st["window"]) | (j < st["sinks"])
    y = y.masked_fill(~seen[:, None, None], 0.0).sum(dim=(2, 3))
    # Every position of the cache once: what it had, if it is not a new row's, and the sum.
    seq, at = _sequence(st["kv_len"], st["cached"], st["kv_start"])
    pages, rows = st["table"][seq, at // page].long(), at % page
    old = st["weights"][pages, :, rows]
    old = old.masked_fill((at >= (kv - new)[seq])[:, None], 0.0)
    st["weights"][pages, :, rows] = old + y.transpose(1, 2)[seq, at]
    return st["weights"]


def _evict(st):
    page, h, keep = st["page"], st["k"].shape[1], st["keep"]
    kv = st["kv_len"].long()
    dev = kv.device
    head = torch.arange(h, device=dev)
    j = torch.arange(max(st["longest"], keep), device=dev)
    pages = st["table"][:, (j // page).clamp_max(st["table"].shape[1] - 1)].long()
    w = st["weights"][pages, :, j % page].transpose(1, 2)
    safe = (j < st["first"]) | (j >= (kv - st["recent"])[:, None])
    w = w.masked_fill(safe[:, None], math.inf).masked_fill((j >= kv[:, None])[:, None], -math.inf)
    kept = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :keep].sort(dim=-1).values
    kept = torch.where(kept < kv[:, None, None], kept, -1)   # [s, h, keep]
    # The rows that stay, to the front. (Sequences that are short enough write what is there.)
    seq, i = _sequence(kv.clamp_max(keep), st["staying"], st["staying_start"])
    src = kept[seq, :, i]
    to = (st["table"][seq, i // page].long()[:, None], head, (i % page)[:, None])
    from_ = (st["table"][seq[:, None], src // page].long(), head, src % page)
    for which in ("k", "v", "k_scale", "v_scale", "weights"):
        if st[which] is not None:
            _bytes(st[which])[to] = _bytes(st[which])[from_]
    st["kv_len"].clamp_max_(keep)
    return kept.int()


def _score(st):
    x, tokens, top = st["logits"].float(), st["tokens"].long(), st["top"]
    m = x.amax(dim=-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.sum(dim=-1, keepdim=True)
    less = torch.log(total)
    entropy = less[:, 0] - (e * d.clamp_min(-1e30)).sum(dim=-1) / total[:, 0]   # (0 times what is masked is 0)
    out = [(d.gather(1, tokens[:, None]) - less)[:, 0], entropy]
    if top:
        # Ordered by value, then by the lower index: unique whole numbers.
        bits = x.view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long() << 32
        order = order | (0x7fffffff - torch.arange(x.shape[1], device=x.device))
        ids = torch.topk(order, top, dim=-1).indices
        out += [ids.int(), d.gather(1, ids) - less]
    return out


# ---------------------------------------------------------------------------
# Inputs.
# ---------------------------------------------------------------------------
def _values(gen, shape, dtype, dev):
    """Rows as the decoder has them: unit variance, a few dimensions eight times as large."""
    x = torch.randn(shape, generator=gen, device=dev)
    loud = torch.rand(shape[-1], generator=gen, device=dev) < 0.03
    return (x * torch.where(loud, 8.0, 1.0)).to(dtype)


def _angles(rows, dim, dev):
    """cos and sin [rows, dim] of the positions 0 .. rows - 1, computed in 64 bits."""
    freq = THETA ** (-(torch.arange(dim, device=dev, dtype=torch.float64) % (dim // 2)) * 2 / dim)
    angle = torch.arange(rows, device=dev, dtype=torch.float64)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _rotation(case, gen, dev, st, positions):
    d = case["dim"]
    st["cos"], st["sin"] = _angles(int(case.get("table") or positions.shape[0]) if case["kind"] == "rotate" else CONTEXT * 2, d, dev)
    st["positions"] = positions.int() if case["kind"] == "enter" or case["table"] else None
    for w in ("q_weight", "k_weight"):
        st[w] = 1 + 0.1 * torch.randn(d, generator=gen, device=dev)
    st["rotate_first"] = case["rotate_first"]


def _projections(case, gen, dev, st, n, v):
    """q, k (and v) heads as views of one projection's rows."""
    hq, h, d = case["heads"], case["kv_heads"], case["dim"]
    x = _values(gen, (n, hq + (2 if v else 1) * h, d), TYPES[case["rows"]], dev)
    st["q"], st["k_rows"] = x[:, :hq], x[:, hq:hq + h]
    if v:
        st["v_rows"] = x[:, hq + h:]


def _prepare_score(case, gen, dev):
    n, v = case["count"], case["vocab"]
    x = torch.randn(n, v, generator=gen, device=dev).mul_(2.5)
    # Peaks as a trained model has them, in some rows far above all else.
    peaks = torch.randint(v, (n, 4), generator=gen, device=dev)
    height = torch.rand(n, 4, generator=gen, device=dev) * 20
    x.scatter_(1, peaks, height)
    tokens = torch.where(torch.rand(n, generator=gen, device=dev) < 0.7, peaks[:, 0],
                         torch.randint(v, (n,), generator=gen, device=dev))
    if case["masked"]:
        x.masked_fill_(torch.rand(v, generator=gen, device=dev) < case["masked"], -math.inf)
        x[:, :2] = height[:, :2]   # (something is always left)
        tokens = torch.where(torch.isinf(x.gather(1, tokens[:, None])[:, 0]), 0, tokens)
    return {"kind": "score", "logits": x.to(TYPES[case["rows"]]), "tokens": tokens.int(),
            "top": min(case["top"], v)}


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    if own:
        from __graft_entry__ import load_package
        load_package()
        from hy_b200 import logprobs, paged, rotary
    if case["kind"] == "score":
        st = _prepare_score(case, gen, dev)
        if own:
            st["call"] = logprobs.token_logprobs
        return st
    if case["kind"] == "rotate":
        st = {"kind": "rotate"}
        _projections(case, gen, dev, st, case["count"], False)
        positions = torch.randint(max(1, case["table"]), (case["count"],), generator=gen, device=dev)
        _rotation(case, gen, dev, st, positions)
        if own:
            st["call"] = rotary.norm_rotate
        return st
    kv, new = lengths(case)
    page, h, d = case["page"], case["kv_heads"], case["dim"]
    need = [-(-n // page) for n in kv]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device=dev).int()
    table = torch.zeros(len(kv), max(need), dtype=torch.int32, device=dev)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n

    def starts(counts):
        return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=dev)

    st = {"kind": case["kind"], "cache": case["cache"], "page": page, "table": table, "total": sum(new),
          "most": max(new), "longest": max(kv), "cached": sum(kv),
          "scale": SCALE if d == DIM else 1.0 / math.sqrt(d), "k_scale": None, "v_scale": None,
          "kv_len": torch.tensor(kv, dtype=torch.int32, device=dev), "kv_start": starts(kv)[:-1],
          "new": torch.tensor(new, device=dev), "q_start": starts(new)}
    dtype = TYPES[case["cache"]]
    for which in ("k", "v"):
        pool = torch.empty(pages, h, page, d, dtype=dtype, device=dev)
        scale = torch.empty(pages, h, page, device=dev) if case["cache"] in LARGEST else None
        some = max(1, (1 << 25) // (h * page * d))
        for p0 in range(0, pages, some):   # a part of the pool at a time: the values are made in 32 bits
            x = _values(gen, (min(some, pages - p0), h, page, d), torch.float32, dev)
            if scale is None:
                pool[p0:p0 + some] = x.to(dtype)
            else:
                scale[p0:p0 + some] = _scales(x, case["cache"])
                pool.view(torch.uint8)[p0:p0 + some] = _codes(x, scale[p0:p0 + some], case["cache"]).view(torch.uint8)
        st[which], st[which + "_scale"] = pool, scale
    if case["kind"] == "enter":
        _projections(case, gen, dev, st, sum(new), True)
        seq, i = _sequence(st["new"], st["total"], st["q_start"][:-1])
        _rotation(case, gen, dev, st, i + (st["kv_len"] - st["new"])[seq])
    else:
        # What a position has got so far: a few hold most of it.
        st["weights"] = torch.rand(pages, h, page, generator=gen, device=dev).pow_(8).mul_(500.0 / max(kv))
    if case["kind"] == "weigh":
        st["window"], st["sinks"] = case["window"], case["sinks"]
        st["q"] = torch.randn(sum(new), case["heads"], d, generator=gen, device=dev).to(TYPES[case["rows"]])
        st["lse"] = _log_sums(st)
    if case["kind"] == "evict":
        staying = [min(n, case["keep"]) for n in kv]
        st.update(keep=case["keep"], recent=case["recent"], first=case["first"], staying=sum(staying),
                  staying_start=starts(staying)[:-1], came={"kv_len": st["kv_len"].clone(), "weights": st["weights"].clone()})
    if own:
        st["pages"] = paged.PagedKVCache(st["k"], st["v"], st["k_scale"], st["v_scale"])
        st["batch"] = paged.PagedBatch(st["q_start"], st["kv_len"], table, max_rows=st["most"])
    return st


def _log_sums(st):
    """Logarithm of the softmax sum of every row and head, as the attention of these rows gives it."""
    q, h, page = st["q"], st["k"].shape[1], st["page"]
    heads = q.shape[1]
    lse = torch.empty(q.shape[:2], device=q.device)
    start = 0
    for s, (kv, n) in enumerate(zip(st["kv_len"].tolist(), st["new"].tolist())):
        j = torch.arange(kv, device=q.device)
        pages, rows = st["table"][s, j // page].long(), j % page
        k = st["k"][pages, :, rows].float()
        if st["k_scale"] is not None:
            k = k * st["k_scale"][pages, :, rows][..., None]
        x = q[start:start + n].float().view(n, h, heads // h, -1).permute(1, 2, 0, 3)
        y = (x.reshape(h, -1, x.shape[-1]) @ k.permute(1, 2, 0) * st["scale"]).view(h, heads // h, n, kv)
        p = torch.arange(kv - n, kv, device=q.device)[:, None]
        seen = j <= p
        if st["window"]:
            seen &= (p - j < st["window"]) | (j < st["sinks"])
        lse[start:start + n] = torch.logsumexp(y.masked_fill(~seen, -math.inf), dim=-1).permute(2, 0, 1).reshape(n, heads)
        start += n
    return lse


def run(state):
    kind = state["kind"]
    if kind == "score":
        if own:
            got = state["call"](state["logits"], state["tokens"], top=state["top"])
            return [got.logprob, got.entropy] + ([got.top_ids, got.top_logprobs] if state["top"] else [])
        return _score(state)
    if kind == "rotate":
        if own:
            return list(state["call"](state["q"], state["k_rows"], state["q_weight"], state["k_weight"], state["cos"],
                                      state["sin"], state["positions"], eps=EPS, rotate_first=state["rotate_first"]))
        return [_rotated(state, x, w).to(x.dtype) for x, w in ((state["q"], state["q_weight"]),
                                                                (state["k_rows"], state["k_weight"]))]
    held = [state[w] for w in ("k", "v", "k_scale", "v_scale") if state[w] is not None]
    if kind == "enter":
        if own:
            q = state["pages"].write_rotated(state["batch"], state["q"], state["k_rows"], state["v_rows"],
                                             state["q_weight"], state["k_weight"], state["cos"], state["sin"],
                                             state["positions"], eps=EPS, rotate_first=state["rotate_first"])
        else:
            q = _enter(state)
        return [q] + held
    if kind == "weigh":
        if own:
            state["pages"].add_weights(state["batch"], state["q"], state["lse"], state["scale"], state["weights"],
                                       window=state["window"], sinks=state["sinks"])
            return state["weights"]
        return _weigh(state)
    # The lengths and weights that the records come with: a pass starts from them.
    state["kv_len"].copy_(state["came"]["kv_len"])
    state["weights"].copy_(state["came"]["weights"])
    if own:
        kept = state["pages"].evict(state["batch"], state["keep"], state["weights"], recent=state["recent"],
                                    first=state["first"])
    else:
        kept = _evict(state)
    return held + [state["weights"], state["kv_len"], kept]


# ---------------------------------------------------------------------------
# The definitions in 64 bits, written apart from the above.
# ---------------------------------------------------------------------------
def _exact_heads(st, x, weight):
    """Rows x [n, heads, dim] as 64-bit values: pairs of dimensions as complex numbers where the angles allow it."""
    n, heads, dim = x.shape
    at = torch.arange(n, device=x.device) if st["positions"] is None else st["positions"].long()
    c, s = st["cos"].double()[at].unsqueeze(1), st["sin"].double()[at].unsqueeze(1)
    half = dim // 2
    y = x.double()
    if not st["rotate_first"]:
        y = weight.double() * y / torch.sqrt(torch.linalg.vector_norm(y, dim=2, keepdim=True) ** 2 / dim + EPS)
    a, b = y[:, :, :half], y[:, :, half:]
    y = torch.cat([a * c[..., :half] - b * s[..., :half], b * c[..., half:] + a * s[..., half:]], dim=2)
    if st["rotate_first"]:
        y = weight.double() * y / torch.sqrt(torch.linalg.vector_norm(y, dim=2, keepdim=True) ** 2 / dim + EPS)
    return y


def _e4m3_grid(dev):
    """The non-negative values of the type, by its definition: 3 bits of fraction, exponents from -6, 448 the largest."""
    return torch.tensor([m / 8 * 2.0 ** -6 for m in range(8)] +
                        [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8) if (e, m) != (8, 7)],
                        dtype=torch.float64, device=dev)


def _exact_codes(x):
    """(codes, scales) of rows x [..., dim] in E4M3: the scale is the 32-bit number that the cache keeps."""
    scale = torch.maximum((x.abs().max(dim=-1).values / LARGEST["e4m3"]).float(),
                          torch.tensor(TINY, device=x.device)).double()
    y = x / scale.unsqueeze(-1)
    grid = _e4m3_grid(x.device)
    hi = torch.searchsorted(grid, y.abs()).clamp(1, len(grid) - 1)
    below, above = grid[hi - 1], grid[hi]
    mid = (below + above) / 2
    up = (y.abs() > mid) | ((y.abs() == mid) & (hi % 2 == 0))   # even code = even fraction
    return torch.where(up, above, below) * torch.sign(y), scale


def _exact_place(st, s, idx):
    """Pages and rows of positions idx of sequence s."""
    idx = torch.as_tensor(idx, device=st["table"].device, dtype=torch.int64)
    return st["table"][s].long()[torch.div(idx, st["page"], rounding_mode="floor")], torch.remainder(idx, st["page"])


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "score":
        x = st["logits"].double()
        logp = x - torch.logsumexp(x, dim=1, keepdim=True)
        out = [logp[torch.arange(len(x), device=x.device), st["tokens"].long()],
               -torch.special.xlogy(logp.exp(), logp.exp()).sum(dim=1)]
        if st["top"]:
            values = torch.sort(x, dim=1, descending=True).values[:, :st["top"]]
            out += [None, values - torch.logsumexp(x, dim=1, keepdim=True)]
        return out
    if kind == "rotate":
        return [_exact_heads(st, st["q"], st["q_weight"]), _exact_heads(st, st["k_rows"], st["k_weight"])]
    kv, new = lengths(case)
    if kind == "enter":
        names = [w for w in ("k", "v", "k_scale", "v_scale") if st[w] is not None]
        held = {w: st[w].float().double() for w in names}
        k, v = _exact_heads(st, st["k_rows"], st["k_weight"]), st["v_rows"].double()
        r = 0
        for s, n in enumerate(new):
            pg, rw = _exact_place(st, s, range(kv[s] - n, kv[s]))
            for w, x in (("k", k[r:r + n]), ("v", v[r:r + n])):
                if case["cache"] in LARGEST:
                    x, held[w + "_scale"][pg, :, rw] = _exact_codes(x)
                held[w][pg, :, rw] = x
            r += n
        return [_exact_heads(st, st["q"], st["q_weight"])] + [held[w] for w in names]
    if kind == "evict":
        names = [w for w in ("k", "v", "k_scale", "v_scale", "weights") if st[w] is not None]
        held = {w: st[w].float().double() for w in names}
        weights, keep = st["weights"].cpu().numpy(), st["keep"]
        table = st["table"].cpu().numpy()
        for s, n in enumerate(kv):
            if n <= keep:
                continue
            at = np.arange(n)
            for h in range(case["kv_heads"]):
                w = weights[table[s, at // st["page"]], h, at % st["page"]].astype(np.float64)
                w[:st["first"]] = np.inf
                w[n - st["recent"]:] = np.inf
                stay = np.sort(np.lexsort((at, -w))[:keep])
                (pg, rw), (pg0, rw0) = _exact_place(st, s, stay), _exact_place(st, s, at[:keep])
                for w in names:
                    held[w][pg0, h, rw0] = held[w][pg, h, rw]
        return [held[w] for w in names] + [None, None]   # (the lengths and the list are whole numbers)
    if work(case)["flops"] > 1e12:
        return None
    group = case["heads"] // case["kv_heads"]
    out = st["weights"].double()
    r = 0
    for s, n in enumerate(new):
        first = max(0, kv[s] - n - case["window"] + 1) if case["window"] else 0
        idx = list(range(min(first, case["sinks"]))) + list(range(first, kv[s]))
        pg, rw = _exact_place(st, s, idx)
        j = torch.tensor(idx, device=out.device)
        k = st["k"][pg, :, rw].float().double()
        if st["k_scale"] is not None:
            k *= st["k_scale"][pg, :, rw].double().unsqueeze(-1)
        total = torch.zeros(len(idx), case["kv_heads"], dtype=torch.float64, device=out.device)
        for i0 in range(0, n, 512):
            i1 = min(n, i0 + 512)
            p = kv[s] - n + torch.arange(i0, i1, device=out.device)
            apart = p[:, None] - j[None, :]
            mask = apart >= 0
            if case["window"]:
                mask = mask & ((apart < case["window"]) | (j < case["sinks"])[None, :])
            for head in range(case["heads"]):
                a = torch.matmul(st["q"][r + i0:r + i1, head].double(), k[:, head // group].T) * st["scale"]
                a = torch.exp(a - st["lse"][r + i0:r + i1, head].double().unsqueeze(1))
                total[:, head // group] += torch.where(mask, a, torch.zeros_like(a)).sum(dim=0)
        keep = (j < kv[s] - n).double().unsqueeze(1)
        out[pg, :, rw] = out[pg, :, rw] * keep + total
        r += n
    return out
