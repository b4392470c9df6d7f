"""Attention over the paged 8-bit cache in 64 bits, and how far a kernel's may be
from it: a bound that follows the weights, so that rows whose weight lies mostly in
a few tokens are held to the same share of what the others add as flat ones are.

Per query row, with p = exp(score - largest), P = sum p, out = p v / P:

- A score that is off by d moves its weight by p d and the output by p d (v - out) / P.
  d: half a step of the query's fixed point, 2^(e - 23) for a head whose largest
  magnitude is below 2^e, times the key's absolute sum (tiled prompts hold queries to
  2^(e - 39) and add head_dim products in fp32); and of numbers in log2 the roundings
  of the three factors, of the score and of its difference from the reference, half a
  step (2^-24) each, with 2^-22 for the exponential and the scale's factor.
- A weight is rounded in fixed point, half a step of 1 / 8350000 of the largest p 2^ex
  (ex: the V scale's exponent, or 60 below the sequence's largest) of its own page,
  times its code.  Tiled prompts round it to fp16: 2^-11 of itself, or half a
  subnormal step where it is less than 2^-21 of the largest.
- Sums in fp32: a wave adds a fourth of the pages, seven roundings each at most
  (tiled prompts: every product).
- The output is rounded to its type.
"""
import numpy as np

from kv8_reference import BLOCK, HALF_STEP, PAGE

U = 2.0 ** -24


def tiled(dtype, q, offsets, group):
    """Whether the call goes to the kernel of prompts (lmx_kv8.hip, plan)."""
    return dtype != "float32" and q.shape[0] * group >= 64 * (len(offsets) - 1)


def attend(ref, q, offsets, lengths, pages, scale, dtype):
    """(out, most) for q [rows, heads, head_dim] over a kv8_reference.Cache; rows that
    see a value that is not finite are NaN, rows of no sequence too."""
    out, most = np.full(q.shape, np.nan), np.zeros(q.shape)
    n_kv, hd = ref.k.shape[1], q.shape[2]
    group = q.shape[1] // n_kv
    prompts = tiled(dtype, q, offsets, group)
    for s, length in enumerate(lengths):
        r0, r1 = int(offsets[s]), int(offsets[s + 1])
        if r0 == r1:
            continue
        n = min(max(int(length), 0), pages.shape[1] * PAGE)
        page = pages[s, :-(-n // PAGE)]
        ok = np.repeat((page >= 0) & (page < len(ref.k)), PAGE)[:n]
        page = np.where((page >= 0) & (page < len(ref.k)), page, 0)
        for h in range(n_kv):
            ks = np.repeat(ref.k_scale[page, h], BLOCK, -1).reshape(-1)[:n].astype(np.float64)
            vs = np.repeat(ref.v_scale[page, h], BLOCK, -1).reshape(-1)[:n].astype(np.float64)
            k = ref.k[page, h].reshape(-1, hd)[:n] * ks[:, None]
            codes = ref.v[page, h].transpose(0, 2, 1).reshape(-1, hd)[:n].astype(np.float64)
            for r in range(r0, r1):
                see = np.flatnonzero(ok[:max(0, min(int(length) - (r1 - r0) + r - r0 + 1, n))])
                for g in range(h * group, (h + 1) * group):
                    if not see.size:
                        out[r, g] = 0.0
                        continue
                    x, kk, c, w = q[r, g], k[see], codes[see], vs[see]
                    v = c * w[:, None]
                    if not (np.isfinite(x).all() and np.isfinite(kk).all() and np.isfinite(v).all()):
                        continue
                    sc = kk @ x * scale
                    p = np.exp(sc - sc.max())
                    total = p.sum()
                    out[r, g] = o = p @ v / total
                    ex = np.frexp(w)[1]
                    ex = np.where(w > 0, np.maximum(ex, ex[w > 0].max(initial=-40) - 60), -100)
                    y = sc * np.log2(np.e) + ex
                    e = np.frexp(max(np.abs(x).max(), 2.0 ** -97))[1]
                    d = scale * np.abs(kk).sum(1) * 2.0 ** (e - (39 if prompts else 23))
                    if prompts:
                        d += U * hd * scale * (np.abs(kk) @ np.abs(x))
                    d += U * (np.log(2) * (3 * np.abs(sc * np.log2(np.e)) + np.abs(y) + y.max() - y) + 4)
                    m = 1.01 * (p * d) @ np.abs(v - o)
                    of_page = see // PAGE
                    if prompts:
                        m = m + 2.0 ** -11 * (p @ np.abs(v)) + 2.0 ** -32 * (p * w).max() * np.abs(c).sum(0)
                        sums = see.size / 4 + 60
                    else:
                        first = np.flatnonzero(np.r_[True, of_page[1:] != of_page[:-1]])
                        top = np.maximum.reduceat(p * 2.0 ** ex, first)
                        m = m + (0.5 / 8350000) * top @ np.add.reduceat(np.abs(c), first)
                        sums = 7 * (-(-length // PAGE) / 4 + 1) + 40
                    m = m / total + U * sums * (p @ np.abs(v) / total + np.abs(o))
                    most[r, g] = m + (np.abs(o) + m) * HALF_STEP[dtype] + (2.0 ** -25 if dtype == "float16" else 2.0 ** -126)
    return out, most
