"""Attention over the paged 8-bit cache in 64 bits, and how far a kernel's may be
from it: a bound that follows the weights, so that rows whose weight lies mostly in
a few tokens are held to the same share of what the others add as flat ones are.

Per query row, with p = exp(score - largest), P = sum p, out = p v / P:

- A score that is off by d moves its weight by p d and the output by p d (v - out) / P,
  at most p d (|v| + |out|) / P.
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


def tiled(dtype, rows, n_seqs, group, n_kv):
    """Whether a call goes to the kernel of prompts (lmx_kv8.hip, plan)."""
    each = -(-rows // n_seqs) * group
    return dtype != "float32" and each >= 96 and n_seqs * -(-each // 16) * n_kv >= 1024


def attend(ref, q, offsets, lengths, pages, scale, dtype):
    """(out, most) for q [rows, heads, head_dim] over a kv8_reference.Cache; rows that
    see a value that is not finite are NaN, rows of no sequence too."""
    out, most = np.full(q.shape, np.nan), np.zeros(q.shape)
    n_kv, hd = ref.k.shape[1], q.shape[2]
    group = q.shape[1] // n_kv
    prompts = tiled(dtype, q.shape[0], len(lengths), group, n_kv)
    for s, length in enumerate(lengths):
        r0, r1 = int(offsets[s]), int(offsets[s + 1])
        if r0 == r1:
            continue
        n = min(max(int(length), 0), pages.shape[1] * PAGE)
        page = pages[s, :-(-n // PAGE)]
        ok = np.repeat((page >= 0) & (page < len(ref.k)), PAGE)[:n]
        page = np.where((page >= 0) & (page < len(ref.k)), page, 0)
        of_page = np.arange(n) // PAGE
        first = np.flatnonzero(np.diff(of_page, prepend=-1))
        at = np.arange(r1 - r0) + int(length) - (r1 - r0)   # positions
        see = ok & (np.arange(n) <= at[:, None])
        for h in range(n_kv):
            x = q[r0:r1, h * group:(h + 1) * group]
            ks = np.repeat(ref.k_scale[page, h], BLOCK, -1).reshape(-1)[:n].astype(np.float64)
            w = np.repeat(ref.v_scale[page, h], BLOCK, -1).reshape(-1)[:n].astype(np.float64)
            # whatever is not finite makes NaN of the rows that see it, and of no other
            bad = (~np.isfinite(ks * w) & see).any(1)[:, None] | ~np.isfinite(x).all(-1)
            ks, w = np.nan_to_num(ks, nan=0.0, posinf=0.0), np.nan_to_num(w, nan=0.0, posinf=0.0)
            k = ref.k[page, h].reshape(-1, hd)[:n] * ks[:, None]
            c = np.abs(ref.v[page, h].transpose(0, 2, 1).reshape(-1, hd)[:n].astype(np.float64))
            v = ref.v[page, h].transpose(0, 2, 1).reshape(-1, hd)[:n] * w[:, None]
            x = np.where(bad[..., None], 0.0, x)
            ex = np.where(w > 0, np.maximum(np.frexp(w)[1], np.frexp(w[ok])[1].max(initial=-40) - 60), -100)
            for g in range(group):
                xg = x[:, g]
                sc = xg @ k.T * scale
                seen = np.where(see, sc, -np.inf)
                top = np.maximum(seen.max(1, initial=-1e300), -1e300)[:, None]
                p = np.exp(seen - top)
                total = np.maximum(p.sum(1), 1e-300)[:, None]
                o = p @ v / total
                s2 = np.where(see, sc * np.log2(np.e), 0.0)
                y = s2 + ex
                e = np.frexp(np.maximum(np.abs(xg).max(1), 2.0 ** -97))[1][:, None]
                d = scale * np.abs(k).sum(1) * 2.0 ** (e - (39 if prompts else 23))
                if prompts:
                    d = d + U * hd * scale * (np.abs(xg) @ np.abs(k).T)
                most_y = np.where(see, y, -1e300).max(1, initial=-1e300)[:, None]
                d = np.where(see, d + U * (np.log(2) * (3 * np.abs(s2) + np.abs(y) + most_y - y) + 4), 0.0)
                m = 1.01 * ((p * d) @ np.abs(v) + (p * d).sum(1)[:, None] * np.abs(o))
                if prompts:
                    m = m + 2.0 ** -11 * (p @ np.abs(v)) + 2.0 ** -32 * (p * w).max(1, initial=0.0)[:, None] * (see @ c)
                    sums = see.sum(1)[:, None] / 4 + 60
                elif n:
                    page_top = np.maximum.reduceat(p * 2.0 ** ex, first, axis=1)
                    m = m + (0.5 / 8350000) * (np.repeat(page_top, np.diff(np.r_[first, n]), axis=1) * see) @ c
                    sums = 7 * (-(-n // PAGE) / 4 + 1) + 40
                else:
                    sums = 0
                m = m / total + U * sums * (p @ np.abs(v) / total + np.abs(o))
                m = m + (np.abs(o) + m) * HALF_STEP[dtype] + (2.0 ** -25 if dtype == "float16" else 2.0 ** -126)
                some = see.any(1)[:, None]
                out[r0:r1, h * group + g] = np.where(bad[:, g][:, None] & some, np.nan, np.where(some, o, 0.0))
                most[r0:r1, h * group + g] = np.where(some, m, 0.0)
    return out, most
