"""Caches held in 8 bits, from their definition: numpy in 64 bits, one row at a time.

A row is its codes' values (slots, KVH, 64) and scales (slots / 16, KVH), whatever
its pages are.  Pinned in ``tests/test_oracle_kv8.py`` by brute force over every
code and by torch's own e4m3 conversion.
"""

import numpy as np

BLOCK = 16
MOST = 65504.0                       # fp16's largest
LARGEST = {"int8": 127.0, "e4m3": 448.0}


def levels(code):
    """Magnitudes of the codes, ascending; a code's place is its low 7 bits."""
    if code == "int8":
        return np.arange(128, dtype=np.float64)
    return np.array([c / 8 * 2.0 ** -6 if c < 8 else (1 + c % 8 / 8) * 2.0 ** (c // 8 - 7)
                     for c in range(127)])


def least_scale(top, code):
    """Least 2^e, e >= -24, with top <= Q 2^e; NaN where top is not finite."""
    top = np.asarray(top, dtype=np.float64)
    steps = 2.0 ** np.arange(-24, 18)
    i = np.searchsorted(steps * LARGEST[code], np.where(np.isfinite(top), top, 0.0))
    return np.where(np.isfinite(top), steps[np.minimum(i, len(steps) - 1)], np.nan)


def nearest(x, s, code):
    """Value of the code nearest to x / s (ties to the even code), held within fp16."""
    lv = levels(code)
    mag = np.abs(x) / s
    i = np.searchsorted((lv[1:] + lv[:-1]) / 2, mag)
    up = np.minimum(i + 1, len(lv) - 1)
    i = np.where((mag == (lv[i] + lv[up]) / 2) & (i % 2 == 1), up, i)
    i = np.minimum(i, np.searchsorted(lv, MOST / s, side="right") - 1)
    return np.copysign(lv[i], x)


def append(values, scales, first, new, code):
    """Tokens ``new`` (n, KVH, 64) at slot ``first`` of a row, in place."""
    for lo in range(first // BLOCK * BLOCK, first + len(new), BLOCK):
        a, b = max(lo, first), min(lo + BLOCK, first + len(new))
        for h in range(new.shape[1]):
            x = new[a - first:b - first, h]
            s = least_scale(np.abs(x).max() if np.isfinite(x).all() else np.inf, code)
            if a > lo:
                old = scales[lo // BLOCK, h]
                s = old if np.isnan(old) else s if np.isnan(s) else max(s, old)
                if s > old:
                    values[lo:a, h] = nearest(values[lo:a, h] * old, s, code)
            scales[lo // BLOCK, h] = s
            values[a:b, h] = 0.0 if np.isnan(s) else nearest(x, s, code)


def dense(values, scales):
    """What the slots stand for, (slots, KVH, 64)."""
    return values * np.repeat(scales, BLOCK, axis=0)[:len(values), :, None]


def attend(q, k, v, scale=0.125):
    """q (QH, 64) over k, v (n, KVH, 64): (QH, 64); zeros over nothing, NaN where it is undefined."""
    if len(k) == 0:
        return np.zeros_like(q)
    g = len(q) // k.shape[1]
    out = np.empty_like(q)
    with np.errstate(invalid="ignore", over="ignore"):
        for i in range(len(q)):
            s = k[:, i // g] @ q[i] * scale
            p = np.exp(s - s.max())
            out[i] = p @ v[:, i // g] / p.sum()
    return out
