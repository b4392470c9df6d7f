"""Plain 64-bit restatement of the 8-bit paged cache (lutmac_kv8.h): append,
attention, and how far a kernel's attention may be from it."""
import math

import numpy as np

PAGE, BLOCK = 64, 16
# half a rounding step of the types' values, relative
HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def check_rotated(got, want, q, dtype):
    """got (float64) against the rotation `want` in 64 bits of q: rounded once (fp32),
    or to 16 bits after fp32's products and sum, off by at most 2^-22 of the pair's
    larger magnitude."""
    if dtype == "float32":
        np.testing.assert_array_equal(got, want.astype(np.float32).astype(np.float64))
        return
    h = q.shape[-1] // 2
    pair = np.maximum(np.abs(q[..., :h]), np.abs(q[..., h:]))
    most = np.abs(want) * HALF_STEP[dtype] * (1 + 2.0 ** -10) + 2.0 ** -22 * np.concatenate([pair, pair], -1)
    most += 2.0 ** -24 if dtype == "float16" else 0.0
    ok = np.isfinite(want)
    assert (np.abs(got - want)[ok] <= most[ok]).all() and not np.isfinite(got[~ok]).any()


def rotate(x, rope, pos):
    """x [heads, hd] at position pos; pairs (d, d + hd / 2)."""
    if rope is None:
        return x
    h = x.shape[-1] // 2
    c, s = rope[pos, :, 0].astype(np.float64), rope[pos, :, 1].astype(np.float64)
    a, b = x[..., :h], x[..., h:]
    return np.concatenate([a * c - b * s, a * s + b * c], -1)


class Cache:
    """Host copy of a cache: dict of k, v (int8), k_scale, v_scale (fp32) arrays."""

    def __init__(self, k, v, k_scale, v_scale):
        self.k, self.v, self.k_scale, self.v_scale = (np.array(a) for a in (k, v, k_scale, v_scale))

    def round(self, x):
        return np.round(x).astype(np.int8)

    def append(self, k, v, q, offsets, lengths, pages, rope):
        """float64 row arrays; returns the rotated q (rows without a place: NaN)."""
        out = np.full(q.shape, np.nan) if q is not None else None
        for s, length in enumerate(lengths):
            r0, r1 = offsets[s], offsets[s + 1]
            start = length - (r1 - r0)
            blocks = {}
            for r in range(r0, r1):
                pos = start + r - r0
                if pos < 0 or (rope is not None and pos >= len(rope)):
                    continue
                if q is not None:
                    out[r] = rotate(q[r], rope, pos)
                if pos // PAGE >= pages.shape[1]:
                    continue
                blocks.setdefault(pos // BLOCK, []).append((r, pos))
            for block, rows in blocks.items():
                page, sub = pages[s, block // 4], block % 4
                if not 0 <= page < len(self.k):
                    continue
                kept = max(start - block * BLOCK, 0)
                xs = [rotate(k[r], rope, p) for r, p in rows], [v[r] for r, _ in rows]
                for h in range(self.k.shape[1]):
                    for codes, scale, x in ((self.k[page, h], self.k_scale, xs[0]), (self.v[page, h].T, self.v_scale, xs[1])):
                        x = np.stack([y[h] for y in x])
                        was = scale[page, h, sub]
                        with np.errstate(all="ignore"):
                            now = max(np.float32(np.abs(x).max() / 127.0), np.float32(2.0 ** -100))
                            if kept:
                                now = max(now, was) if was == was else was
                        if not np.isfinite(x).all() or not now < np.inf:
                            now = np.float32(np.nan)
                        scale[page, h, sub] = now
                        at = sub * BLOCK
                        if now == now and kept and now != was:
                            old = codes[at:at + kept].astype(np.float64) * np.float64(was)
                            codes[at:at + kept] = self.round(old / np.float64(now))
                        for (r, p), y in zip(rows, x):
                            codes[p % PAGE] = self.round(y / np.float64(now)) if now == now else 0
        return out

    def tokens(self, pages, h, n):
        """Values, scale exponents and which of a sequence's first n tokens have a page."""
        k, v, ex, ok = [], [], [], []
        for j in range(n):
            page = pages[j // PAGE] if j // PAGE < len(pages) else -1
            if not 0 <= page < len(self.k):
                page = -1
            t = j % PAGE
            ok.append(page >= 0)
            k.append(self.k[page, h, t] * np.float64(self.k_scale[page, h, t // BLOCK]))
            v.append(self.v[page, h, :, t] * np.float64(self.v_scale[page, h, t // BLOCK]))
            ex.append(np.float64(self.v_scale[page, h, t // BLOCK]))
        return np.array(k), np.array(v), np.array(ex), np.array(ok, bool)

    def attend(self, q, offsets, lengths, pages, scale, dtype):
        """(out, most): the attention of q [rows, heads, hd] and the largest error a
        kernel may have, element by element.  NaN rows stay NaN.

        The bound, per row, with n tokens seen, weights p = exp(score - max), L = sum
        p: a score is off by at most d = scale * ||k||_1 * (half a step of the query's
        fixed point) plus fp32's rounding of it, which moves the output by at most
        2 d max|v|; a weight p 2^e (e the exponent of its V scale, at most 60 below the
        largest of the sequence) by half a step of
        the largest such product, 2^-(p_exp + 1), times a code of at most 127, or (16-bit
        types) by half a step of fp16, 2^-11 of itself; fp32 sums of
        one term a page (16 a page for L), joined over waves and parts; and the last
        rounding to the type."""
        f32 = dtype == "float32"
        q_bits, p_exp = 22 if f32 else 14, np.log2(32560 if dtype == "bfloat16" else 8350000)
        out, most = np.full(q.shape, np.nan), np.zeros(q.shape)
        n_kv = self.k.shape[1]
        group = q.shape[1] // n_kv
        for s, length in enumerate(lengths):
            r0, r1 = offsets[s], offsets[s + 1]
            if r0 == r1:
                continue
            start = length - (r1 - r0)
            for h in range(n_kv):
                k, v, vs, ok = self.tokens(pages[s], h, min(max(length, 0), pages.shape[1] * PAGE))
                for r in range(r0, r1):
                    see = max(0, min(start + r - r0 + 1, len(k)))
                    keep = ok[:see]
                    for g in range(h * group, (h + 1) * group):
                        if not keep.any():
                            out[r, g] = 0.0
                            continue
                        kk, vv, ex = k[:see][keep], v[:see][keep], vs[:see][keep]
                        if not (np.isfinite(q[r, g]).all() and np.isfinite(kk).all() and np.isfinite(vv).all()):
                            continue
                        sc = kk @ q[r, g] * scale
                        p = np.exp(sc - sc.max())
                        out[r, g] = (p / p.sum()) @ vv
                        top = np.abs(q[r, g]).max()
                        e = math.frexp(max(top, 2.0 ** -97))[1]
                        d = scale * np.abs(kk).sum(1).max() * 2.0 ** (e - q_bits - 1)
                        # (join, scale, exponent and difference each round once, of values up to |score| + 200 in log2)
                        d += 6 * 2.0 ** -24 * (np.abs(sc).max() + 140)
                        a = np.abs(vv).max()
                        e2 = np.maximum(np.frexp(ex)[1], max(-100, np.frexp(vs[ok])[1].max() - 60))
                        step = 127 * 0.5 * (p * 2.0 ** e2).max() * 2.0 ** -p_exp * len(p) / p.sum()
                        step += 0.0 if f32 else 2.0 ** -11 * (p @ np.abs(vv)).max() / p.sum()
                        sums = (2 * (see / PAGE + 1) + 40) * 2.0 ** -24
                        most[r, g] = 2 * d * a + step + 2 * sums * a + np.abs(out[r, g]) * HALF_STEP[dtype] + \
                            (2.0 ** -24 if dtype == "float16" else 0.0)
        return out, most
