"""The 8-bit key and value cache restated on the CPU (no counterpart in the reference): what a cache
holds after its tokens were written, a page's order in memory, and attention over it in float64."""

import numpy as np

BLOCK = 64


def nearest_code(x):
    """The nearest e4m3 numbers to float64 x, ties to the even one: 3 bits behind the point from 2^-6
    on, steps of 2^-9 below. Magnitudes up to 448 only; NaN stays."""
    x = np.asarray(x, np.float64)
    _, power = np.frexp(np.where(np.isfinite(x), x, 0.0))
    step = np.ldexp(1.0, np.maximum(power - 1, -6) - 3)
    return np.round(x / step) * step  # numpy rounds halves to even


def block_scale(x):
    """The power of two that a block's codes are taken in."""
    finite = np.abs(x[np.isfinite(x)])
    top = float(finite.max()) if finite.size else 0.0
    if top == 0.0:
        return 1.0
    e = -100
    while top > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def quantize(x):
    """One head's block [64, D] -> (codes as float64 values, scale). Non-finite values become NaN."""
    x = np.asarray(x, np.float64)
    scale = block_scale(x)
    return nearest_code(np.where(np.isfinite(x), x, np.nan) / scale), scale


def held(x, top=None):
    """What a cache holds of one head's tokens [T, D]: the complete blocks as code * scale (magnitudes
    at most `top`, if there is one), the others as they are."""
    x = np.asarray(x, np.float64).copy()
    for lo in range(0, len(x) // BLOCK * BLOCK, BLOCK):
        codes, scale = quantize(x[lo:lo + BLOCK])
        x[lo:lo + BLOCK] = codes * scale if top is None else np.clip(codes * scale, -top, top)
    return x


def key_order(x):
    """[64, D] keys as a page's 64 D numbers."""
    out = []
    for tile in range(4):
        for c in range(x.shape[1] // 64):
            for quarter in range(4):
                for token in range(16):
                    lo = c * 64 + quarter * 16
                    out.append(x[tile * 16 + token, lo:lo + 16])
    return np.concatenate(out)


def value_order(x):
    """[64, D] values as a page's 64 D numbers."""
    out = []
    for tile in range(x.shape[1] // 16):
        for g in range(4):
            for column in range(16):
                for t in range(4):
                    out.append(x[16 * t + 4 * g:16 * t + 4 * g + 4, 16 * tile + column])
    return np.concatenate(out)


def attention(q, k, v, past, scale, window=None, sinks=0):
    """One head: rows q [n, D] of the tokens past, past + 1, .. over k, v [T, D], all float64. Returns the
    output, P |V| and the largest sum of a score's magnitudes, the parts of an error bound."""
    place, key = past + np.arange(len(q))[:, None], np.arange(len(k))[None]
    seen = key <= place
    if window is not None:
        seen &= (place - key < window) | (key < sinks)
    s = np.where(seen, scale * (q @ k.T), -np.inf)
    top = s.max(1, keepdims=True, initial=-np.inf)
    p = np.exp(s - np.where(np.isfinite(top), top, 0.0))
    total = p.sum(1, keepdims=True)
    p = np.divide(p, total, out=np.zeros_like(p), where=total > 0)
    size = scale * (np.abs(q) @ np.abs(k).T)
    return p @ v, p @ np.abs(v), float(size.max(initial=0.0, where=seen))
