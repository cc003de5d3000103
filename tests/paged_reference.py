"""The paged cache's operators in 64 bits, for the tests: plain loops over sequences, from the definitions."""

import math

import numpy as np
import torch

LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def positions(q_start, kv_len, rows):
    """(sequence, position) of every row, None where no sequence holds it."""
    out = [None] * rows
    for s, kv in enumerate(kv_len):
        n = q_start[s + 1] - q_start[s]
        for i in range(n):
            out[q_start[s] + i] = (s, kv - n + i)
    return out


def e4m3_values():
    v = [m / 8 * 2.0 ** -6 for m in range(8)]
    v += [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8) if (e, m) != (8, 7)]
    return np.array(v)


def quantise(x: torch.Tensor, dtype):
    """(codes' values, scales) of x [..., dim], codes by exact comparison with the two neighbours."""
    x = x.double().cpu().numpy()
    bad = ~np.isfinite(x).all(axis=-1)
    amax = np.abs(np.where(np.isfinite(x), x, 0)).max(axis=-1)
    scale = np.maximum((amax / LARGEST[dtype]).astype(np.float32), np.float32(2.0 ** -126)).astype(np.float64)
    with np.errstate(invalid="ignore"):
        y = x / scale[..., None]
    grid = e4m3_values() if dtype == torch.float8_e4m3fn else np.arange(128.0)
    a = np.where(np.isfinite(y), np.abs(y), 0)
    hi = np.clip(np.searchsorted(grid, a), 1, len(grid) - 1)
    mid = (grid[hi - 1] + grid[hi]) / 2
    up = (a > mid) | ((a == mid) & (hi % 2 == 0))
    code = np.where(up, grid[hi], grid[hi - 1]) * np.where(y < 0, -1.0, 1.0)
    code[bad] = 0
    scale = np.where(bad, np.nan, scale)
    return torch.from_numpy(code), torch.from_numpy(scale)


def attention(q, keys, values, positions_, scale, causal=True, window=0, sinks=0):
    """One sequence: q [n, Q, D] at positions_ [n], keys / values [L, H, D], all float64. Returns (out, weights of
    |v|, the largest scale * sum |q| |k| of a row's visible keys); invisible keys and values may hold anything."""
    n, heads, _ = q.shape
    length, kv_heads, _ = keys.shape
    group = heads // kv_heads
    j = torch.arange(length, device=q.device)
    p = torch.as_tensor(positions_, device=q.device)
    seen = (j[None] <= p[:, None]) if causal else (torch.ones(n, length, dtype=torch.bool, device=q.device) &
                                                   (p[:, None] >= 0))
    if window:
        seen &= (p[:, None] - j[None] < window) | (j[None] < sinks)
    out, mass, reach = (torch.zeros_like(q) for _ in range(3))
    if length == 0:
        return out, mass, reach
    for h in range(heads):
        k, v = keys[:, h // group], values[:, h // group]
        s = q[:, h] @ torch.where(torch.isfinite(k), k, 0.0).T * scale
        bad = ~torch.isfinite(k).all(dim=1)
        s = torch.where(bad[None], torch.full_like(s, math.nan), s)
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        top = s.amax(dim=1, keepdim=True)
        w = torch.where(seen, torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top)), 0.0)
        w = w / torch.where(w.sum(dim=1, keepdim=True) == 0, 1.0, w.sum(dim=1, keepdim=True))
        finite_v = torch.where(torch.isfinite(v), v, 0.0)
        out[:, h] = w @ finite_v
        mass[:, h] = w @ finite_v.abs()
        poison = seen.double() @ (~torch.isfinite(v)).double() > 0   # a visible infinity or NaN
        out[:, h] = torch.where(poison, torch.full_like(out[:, h], math.nan), out[:, h])
        r = q[:, h].abs() @ torch.where(torch.isfinite(k), k, 0.0).abs().T * abs(scale)
        reach[:, h] = torch.where(seen, r, 0.0).amax(dim=1, keepdim=True)
    return out, mass, reach


def tolerance(out, mass, reach, length, dim, dtype, codes=False):
    """What the kernel's arithmetic allows at every output. Scores: products exact to 2^-22, dim of them summed in
    fp32, so off by at most reach * (2^-22 + dim 2^-24), which is the relative error of a weight and counts twice
    (weight and sum); exp2 and its argument 2^-20; length additions of 2^-24. bf16 rows: weights rounded to half a
    step, 2^-8, and the output once more.

    8-bit caches (codes): a weight times its value's scale is an f16 number (fp32 rows: two of them), off by at most
    2^-25 below 2^-14 besides. In that unit the row's largest such product t is at least 2^14 (the maximum is taken
    over score plus the scale's exponent, the scale's fraction is at least 1, the factor is 2^14); in tiles of 256
    columns, bf16 rows only, at least 2^-6 (factor 2^6, and 2^12 lost where one exponent stands for a block's). So
    every key's product is off by at most 2^-39 t or 2^-19 t, and its code times t at most that share of the row's
    largest mass (the largest code of a row of values is the type's largest)."""
    rel = 2 * reach * (2.0 ** -22 + dim * 2.0 ** -24) + 2.0 ** -20 + length * 2.0 ** -24
    tol = mass * rel + 2.0 ** -126
    if codes:
        tol = tol + length * 2.0 ** (-19 if dtype == torch.bfloat16 else -39) * mass.amax(dim=-1, keepdim=True)
    if dtype == torch.bfloat16:
        tol = tol + mass * 2.0 ** -8 + out.abs() * 2.0 ** -8 + tol * 2.0 ** -8
    return tol
