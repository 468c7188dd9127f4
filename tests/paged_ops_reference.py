"""The operators on a paged cache in 64 bits, one request and one head at a time (numpy), and the
error bounds their 32-bit kernels stay within.

Bounds: a rounding to a type of eps is off by at most eps / 2 of the value. A sum of n products in
fp32 is off by at most n 2^-24 of the sum of the products' magnitudes (the order does not matter).
"""

import math

import numpy as np
import torch

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float8_e4m3fn: 2.0**-4}
# half of the smallest step near zero
TINY = {torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25, torch.float8_e4m3fn: 2.0**-10}
E4M3_MAX = 448.0


def f64(t):
    return t.detach().cpu().to(torch.float64).numpy() if t.dtype != torch.float8_e4m3fn else t.cpu().float().numpy().astype(np.float64)


def token_page(table, b, t, size, num_blocks):
    """Page of request b's token t, or None (no page: nothing there, or out of range)."""
    vb = t // size
    if vb >= table.shape[1]:
        return None
    p = int(table[b, vb])
    return p if 0 < p < num_blocks else None


def attend(q, ck, cv, table, lens, scale, window=0, k_scale=1.0, v_scale=1.0, dtype=torch.bfloat16, fp8=False):
    """out, lse, per-token weights (sum over a KV head's query heads) and the bounds of each.
    q [B, Hq, D], ck / cv [blocks, H, size, D] as float64 arrays."""
    batch, hq, dim = q.shape
    blocks, heads, size, _ = ck.shape
    group = hq // heads
    cover = table.shape[1] * size
    out, lse = np.zeros((batch, hq, dim)), np.full((batch, hq), -math.inf)
    w = np.zeros((batch, heads, cover))
    b_out, b_lse, b_w = np.zeros(out.shape), np.zeros(lse.shape), np.zeros(w.shape)
    half = HALF_STEP[dtype]
    p_half = HALF_STEP[torch.float16] if fp8 else half
    p_tiny = TINY[torch.float16] if fp8 or dtype == torch.float16 else 0.0
    for b in range(batch):
        n = max(0, int(lens[b]))
        low = max(0, n - window) if window else 0
        toks = [(t, token_page(table, b, t, size, blocks)) for t in range(low, min(n, cover))]
        toks = [(t, p) for t, p in toks if p is not None]
        if not toks:
            continue
        ts, ps = np.array([t for t, _ in toks]), np.array([p for _, p in toks])
        for h in range(heads):
            k, v = ck[ps, h, ts % size] * k_scale, cv[ps, h, ts % size] * v_scale
            for g in range(h * group, (h + 1) * group):
                s = k @ q[b, g] * scale
                top = s.max()
                e = np.exp(s - top)
                p = e / e.sum()
                lse[b, g] = top + math.log(e.sum())
                out[b, g] = p @ v
                # scores: fp32 sums of dim products; an fp8 cache's queries lose up to 2^-25 of the
                # largest element each. Scaling, exponent and logarithm: a few 2^-23 of the magnitudes
                mags = np.abs(k) @ np.abs(q[b, g]) * abs(scale)
                ds = (dim + 4) * 2.0**-24 * mags + 2.0**-22 * np.abs(s)
                if fp8:
                    ds = ds + 2.0**-24 * np.abs(q[b, g]).max() * np.abs(k).sum(1) * abs(scale)
                d = ds.max() + 2.0**-21
                b_lse[b, g] = d + 2.0**-21 * (1 + abs(lse[b, g]))
                spread = p @ np.abs(v)
                # every probability is rounded once, then the output
                b_out[b, g] = half * np.abs(out[b, g]) * 1.01 + (p_half * 1.01 + 2 * d + 2.0**-16) * spread \
                    + len(ts) * p_tiny * np.abs(v).max() + TINY[dtype]
                w[b, h, ts] += p
                b_w[b, h, ts] += p * (2 * d + 2.0**-20) + 2.0**-22
    return out, lse, w, b_out, b_lse, b_w


def rows_of(x, weight, eps, table_rows, positions, rotary, interleaved):
    """One token's heads [H, D]: normed and rotated, and the magnitude that bounds the fp32 error.
    positions: per frequency; None: not rotated."""
    y = x.copy()
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * weight
    mag = np.abs(y)
    if positions is not None:
        half = rotary // 2
        i = np.arange(half)
        c, s = table_rows[positions, i], table_rows[positions, half + i]
        one, two = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, half), slice(half, rotary))
        a, b = y[:, one].copy(), y[:, two].copy()
        y[:, one], y[:, two] = a * c - b * s, a * s + b * c
        both = np.abs(a) + np.abs(b)
        mag[:, one], mag[:, two] = both, both
    return y, mag


def evict(weights, table, lens, keep, first, recent, size, num_blocks):
    """kept [B, H, keep] (-1 behind the kept ones) and new lengths."""
    batch, heads, _ = weights.shape
    kept = np.full((batch, heads, keep), -1, np.int32)
    new = np.zeros(batch, np.int32)
    for b in range(batch):
        n = max(0, min(int(lens[b]), table.shape[1] * size))
        there = [t for t in range(n) if token_page(table, b, t, size, num_blocks) is not None]
        m = min(len(there), keep)
        new[b] = m
        for h in range(heads):
            def key(t):
                x = weights[b, h, t]
                stays = t < first or t >= n - recent
                return (0 if stays else 1, 0 if stays else (-math.inf if x != x else 0), 0 if stays or x != x else -float(x), t)
            kept[b, h, :m] = sorted(sorted(there, key=key)[:m])
    return kept, new
