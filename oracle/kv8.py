"""The 8-bit KV cache in 64 bits (TEST INFRASTRUCTURE ONLY; see oracle/__init__.py).

From the format's definition: a block (the tokens of one page, one kv head) has the smallest
power-of-two scale s with amax <= 448 s (0 for a block of zeros, at least 2^-126, NaN for a
block with a value that is not finite); a code is the e4m3 value nearest to x / s, ties to
the even one. No reference counterpart: the reference's pool has the activation type."""
import math

import numpy as np


def scale_of(amax):
    if not math.isfinite(amax):
        return math.nan
    if amax == 0.0:
        return 0.0
    e = math.frexp(amax)[1] - 9                       # 448 = 0.875 * 2^9
    if amax > math.ldexp(448.0, e):
        e += 1
    return math.ldexp(1.0, max(e, -126))


def e4m3(y):
    """Nearest e4m3 values of an array with |y| <= 448 (NaN stays NaN)."""
    y = np.asarray(y, dtype=np.float64)
    _, e = np.frexp(np.where(np.isfinite(y) & (y != 0), y, 1.0))
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.where(np.isnan(y), np.nan, np.rint(y / step) * step)


def rotate(x, cos, sin):
    """Rotate-half RoPE of x [n, H, D] with table rows cos, sin [n, D]; float32, every
    product and the sum rounded once (the kernel's arithmetic), or float64 for the exact one."""
    half = x.shape[-1] // 2
    other = np.concatenate([-x[..., half:], x[..., :half]], -1)
    return x * cos[:, None] + other * sin[:, None]


class Cache:
    """One layer: values and scales, [pages, hkv, page_size, d] and [pages, hkv]."""

    def __init__(self, pages, hkv, page_size, d):
        self.v = {n: np.zeros((pages, hkv, page_size, d)) for n in "kv"}
        self.s = {n: np.zeros((pages, hkv)) for n in "kv"}
        self.ps = page_size

    def append(self, table, start, k, v):
        """Tokens k, v [n, hkv, d] at positions start.. of the sequence with pages ``table``."""
        n = k.shape[0]
        for pi in range(start // self.ps, (start + n - 1) // self.ps + 1 if n else 0):
            lo, hi = max(start, pi * self.ps), min(start + n, (pi + 1) * self.ps)
            a, b, page = lo - pi * self.ps, hi - pi * self.ps, table[pi]
            for name, x in (("k", k), ("v", v)):
                vals, scales = self.v[name][page], self.s[name][page]
                for h in range(vals.shape[0]):
                    new = np.asarray(x[lo - start:hi - start, h], dtype=np.float64)
                    s = scale_of(float(np.abs(new).max()) if np.isfinite(new).all() else math.inf)
                    was = scales[h] if a > 0 else 0.0
                    s = math.nan if math.isnan(s) or math.isnan(was) else max(s, was)
                    if math.isnan(s):
                        vals[h, :b] = math.nan
                    else:
                        safe = s if s > 0 else 1.0
                        vals[h, :a] = e4m3(vals[h, :a] / safe) * s
                        vals[h, a:b] = e4m3(new / safe) * s
                    scales[h] = s

    def read(self, table, length, name):
        """[length, hkv, d] of a sequence."""
        x = self.v[name][list(table)].transpose(0, 2, 1, 3)
        return x.reshape(-1, x.shape[2], x.shape[3])[:length]


def attention(q, k, v, sm_scale, causal=True):
    """q [n, hq, d] at the last n positions of k, v [L, hkv, d]: [n, hq, d] in 64 bits; a row
    that sees nothing is zeros."""
    q, k, v = (np.asarray(t, dtype=np.float64) for t in (q, k, v))
    n, hq, _ = q.shape
    length, hkv = k.shape[0], k.shape[1]
    out = np.zeros((n, hq, v.shape[2]))
    if not length:
        return out
    seen = np.arange(length)[None] <= np.arange(length - n, length)[:, None] if causal else \
        np.ones((n, length), bool)
    for h in range(hq):
        kh, vh = k[:, h * hkv // hq], v[:, h * hkv // hq]
        w = np.where(seen, q[:, h] @ kh.T * sm_scale, -np.inf)
        m = w.max(1, keepdims=True)
        p = np.exp(w - np.where(m == -np.inf, 0.0, m))
        out[:, h] = p / np.where(m == -np.inf, 1.0, p.sum(1, keepdims=True)) @ np.where(np.isnan(vh), 0.0, vh)
        # a value that is not a number reaches the rows that see it
        out[:, h][(seen @ np.isnan(vh).any(1)) > 0] = np.nan
    return out
