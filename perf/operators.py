"""Cases of the paged KV cache: rows quantised as they are written and read back, the attention
of new rows over the pages, and the same attention with a sliding window and sinks.

A case's `kind` is "store" (write the batch's new rows, read them back), "fetch" (read the rows of
whole sequences), "attend" (attention of the new rows over the cache) or "window" (the same with a
window and sinks). Sequence s of a case has kv_len[s] rows in the cache, the last n[s] of them new;
both are drawn from the case's `lens` between the case's bounds.
"""

import math
import random

import numpy as np
import torch

own = False

HEADS, KV_HEADS, DIM = 16, 8, 128   # the decoder's attention geometry
SCALE = 0.0883883                   # the decoder's attention scale at 128 dimensions
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
LARGEST = {"e4m3": 448.0, "int8": 127.0}
TINY = 2.0 ** -126


def _case(name, kind, cache, rows, seqs, kv, new, page=16, heads=HEADS, kv_heads=KV_HEADS, dim=DIM, window=0,
          sinks=0, lens=1):
    return {"name": name, "kind": kind, "cache": cache, "rows": rows, "seqs": seqs, "kv_min": kv[0], "kv_max": kv[1],
            "new_min": new[0], "new_max": new[1], "page": page, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "window": window, "sinks": sinks, "lens": lens}


def listed():
    return [
        # One decode step of one record: its key / value row joins an 8-bit cache. Latency alone.
        _case("store_token_e4m3", "store", "e4m3", "f32", 1, (2048, 2048), (1, 1)),
        # A prompt of 1024 rows (the decoder's fp32 projections) into an 8-bit integer cache.
        _case("store_prompt_int8", "store", "int8", "f32", 1, (1024, 1024), (1024, 1024)),
        # Prompts of 16 records admitted together, odd lengths, bf16 rows.
        _case("store_prompts_e4m3", "store", "e4m3", "bf16", 16, (700, 4096), (700, 4096), lens=2),
        # One record's prefix brought back as fp32 rows (a cache handed to a contiguous slot).
        _case("fetch_prefix_e4m3", "fetch", "e4m3", "f32", 1, (1111, 1111), (1111, 1111)),
        # 64 records of up to 8192 rows read back whole.
        _case("fetch_records_int8", "fetch", "int8", "bf16", 64, (100, 8192), (100, 8192), page=64, lens=3),
        # One AR token of one record at 2048 rows, fp32 throughout: the decoder's parity types.
        _case("attend_token_f32", "attend", "f32", "f32", 1, (2048, 2048), (1, 1)),
        # 16 records, one token each, other heads (four query heads per KV head of 64), pages of 24 rows, ragged.
        _case("attend_records_odd", "attend", "bf16", "bf16", 16, (1, 2500), (1, 1), page=24, heads=32, dim=64, lens=4),
        # 64 records at long contexts, one token each, 8-bit cache: the serving step that memory bounds.
        _case("attend_serving_e4m3", "attend", "e4m3", "bf16", 64, (1024, 8192), (1, 1), page=64, lens=5),
        # Verify blocks of 16 rows of four records, fp32 rows over a bf16 cache.
        _case("attend_verify", "attend", "bf16", "f32", 4, (1500, 2600), (16, 16), lens=6),
        # Prompt chunks of four records behind long prefixes: what the tensor cores bound.
        _case("attend_chunks", "attend", "bf16", "bf16", 4, (6000, 8192), (1000, 1024), lens=7),
        # 16 long generations, one token each, window of 1024 and 4 sinks.
        _case("window_records", "window", "bf16", "bf16", 16, (900, 16384), (1, 1), window=1024, sinks=4, lens=8),
        # Chunks of up to 2048 rows in long sequences, window of 1024 and 4 sinks, integer cache.
        _case("window_chunks_int8", "window", "int8", "bf16", 4, (8000, 16384), (1500, 2048), page=32, window=1024,
              sinks=4, lens=9),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    top = {f: max(work(c)[f] for c in listed()) for f in ("bytes", "flops")}
    while True:
        kind = rng.choice(["store", "fetch", "attend", "attend", "window"])
        cache = rng.choice(["f32", "bf16", "e4m3", "int8"])
        rows = rng.choice(["f32", "bf16"])
        kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
        group = rng.choice([1, 2, 2, 4, 5, 8]) if kind in ("attend", "window") else 1
        seqs = log(1, 64)
        kv_max = log(1, 16384)
        kv_min = rng.randint(1, kv_max)
        if kind in ("attend", "window"):
            new_max = min(kv_max, rng.choice([1, 1, log(2, 40), log(16, 2048)]))
        else:
            new_max = log(1, kv_max)
        new_min = rng.randint(1, new_max)
        window = log(16, 4096) if kind == "window" else 0
        sinks = rng.choice([0, 1, 4, 33]) if kind == "window" else 0
        case = _case("", kind, cache, rows, seqs, (kv_min, kv_max), (new_min, new_max),
                     page=rng.choice([1, 8, 16, 16, 24, 32, 64, 100, 128]), heads=kv_heads * group, kv_heads=kv_heads,
                     dim=rng.choice([64, 128]), window=window, sinks=sinks, lens=rng.randint(1, 10 ** 6))
        del case["name"]
        w = work(case)
        pool = 2 * sum(lengths(case)[0]) * kv_heads * case["dim"] * (1 if cache in LARGEST else TYPES[cache].itemsize)
        if w["bytes"] <= top["bytes"] and w["flops"] <= top["flops"] and pool <= top["bytes"]:
            return case


def lengths(case):
    """kv_len and the count of new rows of every sequence."""
    rng = random.Random(case["lens"])
    kv = [rng.randint(case["kv_min"], case["kv_max"]) for _ in range(case["seqs"])]
    if case["kind"] == "fetch" or case["new_min"] == case["kv_min"] and case["new_max"] == case["kv_max"]:
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
    kv, new = lengths(case)
    h, d = case["kv_heads"], case["dim"]
    e_cache = TYPES[case["cache"]].itemsize
    e_rows = TYPES[case["rows"]].itemsize
    row = h * (2 * d * e_cache + (8 if case["cache"] in LARGEST else 0))   # one position's keys and values
    if case["kind"] == "store":   # rows in, pages out; pages in, rows out
        return {"bytes": sum(new) * (2 * row + 4 * h * d * e_rows), "flops": sum(new) * h * d * 4}
    if case["kind"] == "fetch":
        return {"bytes": sum(new) * (row + 2 * h * d * e_rows), "flops": sum(new) * h * d * 2}
    seen = [_visible(case, a, b) for a, b in zip(kv, new)]
    return {"bytes": sum(k for _, k in seen) * row + 2 * sum(new) * case["heads"] * d * e_rows,
            "flops": 4 * d * case["heads"] * sum(t for t, _ in seen)}


# ---------------------------------------------------------------------------
# The plain form.
# ---------------------------------------------------------------------------
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


def _places(st):
    """Page and row in it of every new row, in the order of the rows."""
    kv, n, table, page = st["kv_len"], st["new"], st["table"], st["page"]
    total = st["total"]
    seq = torch.repeat_interleave(torch.arange(len(n), device=n.device), n, output_size=total)
    at = torch.arange(total, device=n.device) - st["q_start"][:-1][seq] + (kv - n)[seq]
    return table[seq, at // page].long(), at % page


def _stored(st, which, pages, rows, heads=slice(None)):
    """The values that the cache holds at (pages, rows): [positions, heads, dim] in 32 bits."""
    x = st[which][pages, heads, rows].float()
    scale = st[which + "_scale"]
    return x if scale is None else x * scale[pages, heads, rows][..., None]


def _store(st):
    pages, rows = _places(st)
    for which, x in (("k", st["k_rows"]), ("v", st["v_rows"])):
        if st["cache"] in LARGEST:
            scale = _scales(x, st["cache"])
            code = _codes(x, scale, st["cache"])
            st[which + "_scale"][pages, :, rows] = scale
            if st["cache"] == "e4m3":
                st[which].view(torch.uint8)[pages, :, rows] = code.view(torch.uint8)
            else:
                st[which][pages, :, rows] = code
        else:
            st[which][pages, :, rows] = x.to(st[which].dtype)


def _fetch(st):
    pages, rows = _places(st)
    return tuple(_stored(st, w, pages, rows).to(st["rows"]) for w in ("k", "v"))


def _attend(st):
    q, page = st["q"], st["page"]
    heads, h = q.shape[1], st["k"].shape[1]
    out = torch.empty_like(q)
    start = 0
    for s, (kv, n) in enumerate(zip(st["kv_host"], st["new_host"])):
        for r0 in range(0, n, 512):   # a block of rows at a time: the scores are kept whole
            r1 = min(n, r0 + 512)
            p = torch.arange(kv - n + r0, kv - n + r1, device=q.device)
            hi = kv - n + r1
            lo = max(0, kv - n + r0 - st["window"] + 1) if st["window"] else 0
            j = torch.arange(lo, hi, device=q.device)
            if min(lo, st["sinks"]):
                j = torch.cat([torch.arange(min(lo, st["sinks"]), device=q.device), j])
            pages, rows = st["table"][s, j // page].long(), j % page
            k = _stored(st, "k", pages, rows).permute(1, 2, 0)   # [kv heads, dim, keys]
            v = _stored(st, "v", pages, rows).transpose(0, 1)    # [kv heads, keys, dim]
            x = q[start + r0:start + r1].float().view(r1 - r0, h, heads // h, -1).permute(1, 2, 0, 3)
            y = x.reshape(h, -1, x.shape[-1]) @ k * st["scale"]
            seen = j[None, :] <= p[:, None]
            if st["window"]:
                seen &= (p[:, None] - j[None, :] < st["window"]) | (j[None, :] < st["sinks"])
            y = y.view(h, heads // h, r1 - r0, -1).masked_fill(~seen, -math.inf)
            y = torch.exp(y - y.amax(dim=-1, keepdim=True))
            o = (y.reshape(h, -1, y.shape[-1]) @ v).view(h, heads // h, r1 - r0, -1) / y.sum(dim=-1, keepdim=True)
            out[start + r0:start + r1] = o.permute(2, 0, 1, 3).reshape(r1 - r0, heads, -1).to(q.dtype)
        start += n
    return out


# ---------------------------------------------------------------------------
# Inputs.
# ---------------------------------------------------------------------------
def _values(gen, shape, dtype, dev):
    """Rows as the decoder has them: unit variance, a few dimensions eight times as large."""
    x = torch.randn(shape, generator=gen, device=dev)
    loud = torch.rand(shape[-1], generator=gen, device=dev) < 0.03
    return (x * torch.where(loud, 8.0, 1.0)).to(dtype)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
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
    st = {"cache": case["cache"], "page": page, "window": case["window"], "sinks": case["sinks"],
          "rows": TYPES[case["rows"]], "scale": SCALE if d == DIM else 1.0 / math.sqrt(d), "kind": case["kind"],
          "kv_host": kv, "new_host": new, "total": sum(new), "most": max(new), "table": table,
          "kv_len": torch.tensor(kv, dtype=torch.int32, device=dev), "new": torch.tensor(new, device=dev),
          "q_start": torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=dev),
          "k_scale": None, "v_scale": None}
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
    if case["kind"] == "store":
        st["k_rows"] = _values(gen, (sum(new), h, d), st["rows"], dev)
        st["v_rows"] = _values(gen, (sum(new), h, d), st["rows"], dev)
    if case["kind"] in ("attend", "window"):
        st["q"] = torch.randn(sum(new), case["heads"], d, generator=gen, device=dev).to(st["rows"])
    if own:
        from __graft_entry__ import load_package
        load_package()
        from hy_b200 import paged
        st["pages"] = paged.PagedKVCache(st["k"], st["v"], st["k_scale"], st["v_scale"])
        st["batch"] = paged.PagedBatch(st["q_start"], st["kv_len"], table, max_rows=st["most"])
    return st


def run(state):
    kind = state["kind"]
    if kind == "store":
        if own:
            state["pages"].write(state["batch"], state["k_rows"], state["v_rows"])
            rows = state["pages"].read(state["batch"], state["total"], state["rows"])
        else:
            _store(state)
            rows = _fetch(state)
        if state["cache"] in LARGEST:   # the codes are in `rows`, as the values they stand for
            return [*rows, state["k_scale"], state["v_scale"]]
        return [*rows, state["k"], state["v"]]
    if kind == "fetch":
        if own:
            return list(state["pages"].read(state["batch"], state["total"], state["rows"]))
        return list(_fetch(state))
    if own:
        return state["pages"].attention(state["batch"], state["q"], state["scale"], window=state["window"],
                                        sinks=state["sinks"])
    return _attend(state)


# ---------------------------------------------------------------------------
# The definition in 64 bits, position by position.
# ---------------------------------------------------------------------------
def _e4m3_grid(dev):
    """The non-negative values of the type, by its definition: 3 bits of fraction, exponents from -6, 448 the largest."""
    return torch.tensor([m / 8 * 2.0 ** -6 for m in range(8)] +
                        [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8) if (e, m) != (8, 7)],
                        dtype=torch.float64, device=dev)


def _exact_quantised(x, cache):
    """(values, scales) of rows x [..., dim]: the scale is the 32-bit number that the cache keeps."""
    x = x.double()
    scale = torch.maximum((x.abs().max(dim=-1).values / LARGEST[cache]).float(),
                          torch.tensor(TINY, device=x.device)).double()
    y = x / scale.unsqueeze(-1)
    if cache == "int8":
        c = torch.floor(y)
        f = y - c
        c = c + ((f > 0.5) | ((f == 0.5) & (c % 2 != 0))).double()
    else:
        grid = _e4m3_grid(x.device)
        hi = torch.searchsorted(grid, y.abs()).clamp(1, len(grid) - 1)
        below, above = grid[hi - 1], grid[hi]
        mid = (below + above) / 2
        up = (y.abs() > mid) | ((y.abs() == mid) & (hi % 2 == 0))   # even code = even fraction
        c = torch.where(up, above, below) * torch.sign(y)
    return c * scale.unsqueeze(-1), scale


def exact(case, seed):
    if case["kind"] in ("attend", "window") and work(case)["flops"] > 2e12:
        return None
    st = prepare(case, seed)
    dev = st["table"].device
    table = st["table"].tolist()
    page, kv, new = st["page"], st["kv_host"], st["new_host"]

    def position(which, s, idx):
        """Rows idx of sequence s as 64-bit values [kv heads, len(idx), dim]."""
        pg = torch.tensor([table[s][j // page] for j in idx], device=dev)
        rw = torch.tensor([j % page for j in idx], device=dev)
        x = st[which].transpose(1, 2)[pg, rw].to(torch.float32).double()
        if st[which + "_scale"] is not None:
            x *= st[which + "_scale"].transpose(1, 2)[pg, rw].double().unsqueeze(-1)
        return x.transpose(0, 1)

    if case["kind"] == "fetch":
        return [torch.cat([position(w, s, range(kv[s])).transpose(0, 1) for s in range(len(kv))]) for w in ("k", "v")]
    if case["kind"] == "store":
        rows, held = [], []
        for w in ("k", "v"):
            x = st[w + "_rows"]
            if case["cache"] in LARGEST:
                value, scale = _exact_quantised(x, case["cache"])
                pool = st[w + "_scale"].double()
                put = scale
            else:
                value = x.to(st[w].dtype).double()
                pool = st[w].double()
                put = value
            r = 0
            for s, n in enumerate(new):
                pg = torch.tensor([table[s][j // page] for j in range(kv[s] - n, kv[s])], device=dev)
                rw = torch.tensor([j % page for j in range(kv[s] - n, kv[s])], device=dev)
                pool[pg, :, rw] = put[r:r + n]
                r += n
            rows.append(value)
            held.append(pool)
        return rows + held
    q = st["q"].double()
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros_like(q)
    r = 0
    for s, n in enumerate(new):
        first = max(0, kv[s] - n - case["window"] + 1) if case["window"] else 0
        idx = list(range(min(first, case["sinks"]))) + list(range(first, kv[s]))
        k, v = position("k", s, idx), position("v", s, idx)
        j = torch.tensor(idx, device=dev)
        for i0 in range(0, n, 256):
            i1 = min(n, i0 + 256)
            p = kv[s] - n + torch.arange(i0, i1, device=dev)
            d = p[:, None] - j[None, :]
            mask = d >= 0
            if case["window"]:
                mask = mask & ((d < case["window"]) | (j < case["sinks"])[None, :])
            for head in range(case["heads"]):
                a = torch.matmul(q[r + i0:r + i1, head], k[head // group].T) * st["scale"]
                a = torch.softmax(torch.where(mask, a, torch.full_like(a, -math.inf)), dim=-1)
                out[r + i0:r + i1, head] = torch.matmul(a, v[head // group])
        r += n
    return out
