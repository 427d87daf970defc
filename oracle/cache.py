"""A paged key-value cache in float64: rotary positions, what an append stores, and causal attention over the cache, each with
a bound of what float32 arithmetic and the documented roundings may add to it. Loops over sequences, heads and pages as the
definitions have them; nothing here is shared with the kernels."""

import numpy as np

FLOAT = 2.0**-24  # a rounding to float32


def owners(starts, lengths, tokens):
    """(sequence, position) of every token; sequence -1 for a token that belongs to none."""
    seq, position = np.full(tokens, -1), np.zeros(tokens, np.int64)
    for i in range(len(lengths)):
        for t in range(starts[i], starts[i + 1]):
            seq[t], position[t] = i, lengths[i] - (starts[i + 1] - t)
    return seq, position


def rotate(x, position, frequencies, interleaved=False, magnitude=1.0):
    """Heads (tokens, heads, d) turned by their positions, and the bound: the angle is off by a float32 rounding of half a turn
    and the sines by 4 units in the last place, 8 * 2^-24 together; the magnitude, two products and a sum add 4. The double
    that a frequency is given as adds its own 2^-52."""
    half = len(frequencies)
    angle = position.astype(np.float64)[:, None] * np.asarray(frequencies, np.float64)
    cos, sin = magnitude * np.cos(angle)[:, None], magnitude * np.sin(angle)[:, None]
    y, size = x.copy(), np.zeros_like(x)
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    size[..., first] = size[..., second] = abs(magnitude) * (np.abs(a) + np.abs(b)) * (12 * FLOAT + np.abs(angle)[:, None] * 2.0**-51)
    return y, size


def place(pages, page, sequence, position, count):
    """(page number, row) of a key, or None where the table has no page of the cache for it."""
    if sequence < 0 or position < 0 or position // page >= pages.shape[1]:
        return None
    number = pages[sequence, position // page]
    return (number, position % page) if 0 <= number < count else None


def keys_of(cache, pages, sequence, length):
    """The first `length` keys (or values) of a sequence, (length, kv_heads, d); a page that is not there reads as zeros."""
    count, kv_heads, page, d = cache.shape
    held = min(length, pages.shape[1] * page)
    y = np.zeros((max(held, 0), kv_heads, d))
    for j in range(0, held, page):
        number = pages[sequence, j // page]
        if 0 <= number < count:
            y[j:j + page] = cache[number].transpose(1, 0, 2)[: min(page, held - j)]
    return y


def attention(q, keys, values, starts, lengths, pages, scale, window=0, weight=0.0, tiny=0.0):
    """(y, bound), (tokens, heads, d). `weight`: the rounding of a softmax weight before its product, relative, and `tiny` the
    one of weights near zero, absolute in units of the largest weight. A score's float32 sum of d exact products, in any order, is off
    by (d + 8) 2^-23 of the sum of magnitudes, its scaling, the subtraction of a maximum and the power by 2^-22 of their sizes; that
    is a weight's relative error, once above and once below the fraction. A sum of n weighted values is off by
    (n + 64) 2^-23 of its magnitudes. Tokens without a sequence are NaN in both."""
    tokens, heads, d = q.shape
    y, bound = np.full((2, tokens, heads, d), np.nan)
    group = heads // keys.shape[1]
    for i in range(len(lengths)):
        k, v = (keys_of(c, pages, i, max(lengths[i], 0)) for c in (keys, values))
        for t in range(starts[i], starts[i + 1]):
            position = max(lengths[i], 0) - (starts[i + 1] - t)
            low, high = max(0, position + 1 - window) if window else 0, min(position + 1, len(k))
            if high <= low:
                y[t], bound[t] = 0, 0
                continue
            n = high - low
            for h in range(heads):
                kk, vv = k[low:high, h // group], v[low:high, h // group]
                s = scale * (kk @ q[t, h])
                p = np.exp(s - s.max())
                w = p / p.sum()
                y[t, h] = w @ vv
                off = scale * (np.abs(kk) @ np.abs(q[t, h])) * (d + 8) * 2 * FLOAT + (np.abs(s) + abs(s.max()) + 1) * 4 * FLOAT
                bound[t, h] = (w * (off + off.max() + weight + (n + 64) * 2 * FLOAT)) @ np.abs(vv) + tiny * n * np.abs(vv).max(0)
    return y, bound
