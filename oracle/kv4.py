"""float64 oracle of the paged 4-bit KV cache: format, page tables, norm and rotation, attention (numpy only).

The format is that of include/xinfer_attention.h: blocks of 32 features share a power of two, a feature takes the
nearest of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} times it.  Everything here is written from those definitions, element by
element where that is plainest.
"""

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = 32


def block_exponents(x):
    """Exponents e of each block of x [..., D] (finite float64)."""
    top = np.abs(x).reshape(*x.shape[:-1], -1, BLOCK).max(-1)
    e = np.where(top > 0, np.frexp(np.where(top > 0, top, 1.0))[1] - 3, -125)  # floor(log2 top) - 2
    e = e + ((top > 0) & (top > 7 * np.exp2(e.astype(np.float64))))
    return np.clip(e, -125, 125)


def nearest_codes(y):
    """Magnitude codes 0..7 of |y|: the nearest grid value, ties to the even code, 6 for all above it."""
    distance = np.abs(np.abs(y)[..., None] - GRID)
    low = distance.argmin(-1)
    high = 7 - distance[..., ::-1].argmin(-1)
    return np.where((low != high) & (low % 2 == 1), high, low)


def store(key, value):
    """(codes, scale bytes) of keys and of values [..., D]: codes are 0..7, plus 8 for negative features."""
    finite = np.isfinite(key).all(-1) & np.isfinite(value).all(-1)
    held = []
    for x, nan_scale in ((key, 255), (value, 2)):
        x = np.where(finite[..., None], x, 0.0)
        e = block_exponents(x)
        y = x / np.exp2(np.repeat(e, BLOCK, axis=-1).astype(np.float64))
        codes = nearest_codes(y) + 8 * (np.signbit(x) & finite[..., None])
        held.append((codes, np.where(finite[..., None], e + 127, nan_scale)))
    return held


def values(codes, scales, key=True):
    """What codes and scale bytes stand for; a key's scale of 255 is NaN, a value's above 252 reads as 252."""
    scales = scales.astype(np.float64)
    unit = np.where(scales == 255, np.nan, np.exp2(scales - 127)) if key else np.exp2(np.minimum(scales, 252) - 127)
    x = GRID[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    with np.errstate(invalid="ignore"):
        return x * np.repeat(unit, BLOCK, axis=-1)


def unpack(cache):
    """(keys, values) [N, Hkv, P, D] of a cache's four uint8 arrays."""
    out = []
    for codes, scales, key in ((cache[0], cache[1], True), (cache[2], cache[3], False)):
        pairs = np.stack((codes & 15, codes >> 4), axis=-1).reshape(*codes.shape[:-1], -1)
        out.append(values(pairs, np.swapaxes(scales, -1, -2), key))
    return out


def append(cache, key, value, slots):
    """Store key/value [B, Hkv, T, D] at slots [B, T] in the cache's arrays, in place."""
    pages, _, size, _ = cache[0].shape
    held = store(key, value)
    for b, t in np.ndindex(*slots.shape):
        slot = slots[b, t]
        if not 0 <= slot < pages * size:
            continue
        for (codes, scales), at in zip(held, (0, 2)):
            c = codes[b, :, t]
            cache[at][slot // size, :, slot % size] = c[..., 0::2] + 16 * c[..., 1::2]
            cache[at + 1][slot // size, :, :, slot % size] = scales[b, :, t]


def reserve(before, after, counts, tokens, size, counters, table, ring):
    """(lengths, positions, slots, counters, table, ring): one row after another."""
    rows, width = table.shape
    table, ring = table.copy(), ring.copy()
    old_ring, old_table = ring.copy(), table.copy()
    head, tail = counters
    lengths = np.zeros((2, rows), np.int64)
    positions = np.zeros((rows, tokens), np.int64)
    slots = np.full((rows, tokens), -1, np.int64)
    asked = given = taken = 0
    for r in range(rows):
        held, need = -(-before[r] // size), -(-after[r] // size)
        fits = after[r] <= width * size
        grow = max(need - held, 0) if fits else 0
        start, asked = asked, asked + grow
        if not fits or (grow > 0 and asked > tail - head):
            lengths[:, r] = 0, before[r]
            continue
        taken += grow
        for i in range(grow):
            table[r, held + i] = old_ring[(head + start + i) % len(ring)]
        for i in range(need, held):
            ring[(tail + given) % len(ring)] = old_table[r, i]
            given += 1
        lengths[:, r] = counts[r], after[r]
        for t in range(counts[r]):
            p = after[r] - counts[r] + t
            positions[r, t] = p
            slots[r, t] = table[r, p // size] * size + p % size
    return lengths, positions, slots, np.array([head + taken, tail + given]), table, ring


def norm_rope(x, weight, offset, eps, cos, sin):
    """x [..., H, D] normalised per head and its first R features rotated by cos/sin [..., R]."""
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (weight + offset)
    half = cos.shape[-1] // 2
    cos, sin = cos[..., None, :], sin[..., None, :]
    out = y.copy()
    out[..., :half] = y[..., :half] * cos[..., :half] - y[..., half:2 * half] * sin[..., :half]
    out[..., half:2 * half] = y[..., half:2 * half] * cos[..., half:] + y[..., :half] * sin[..., half:]
    return out


def attention(q, cache, table, lengths, scale, max_length=None, magnitudes=False):
    """[B, T, Hq, D]: each query over the keys it sees, pages outside the cache absent; zero where it sees none.

    ``magnitudes``: the same weights over the values' magnitudes.
    """
    keys, vals = unpack(cache)
    if magnitudes:
        vals = np.abs(vals)
    pages, kv_heads, size, _ = keys.shape
    rows, heads, tokens, dim = q.shape
    group = heads // kv_heads
    out = np.zeros((rows, tokens, heads, dim))
    for r in range(rows):
        bound = min(table.shape[1] * size, max_length or 1 << 40)
        n = min(max(lengths[0, r], 0), tokens, bound)
        length = min(max(lengths[1, r], n), bound)
        at = np.arange(length)
        page = table[r, at // size]
        at = at[(page >= 0) & (page < pages)]
        page = table[r, at // size]
        for h in range(kv_heads):
            k, v = keys[page, h, at % size], vals[page, h, at % size]
            for t in range(n):
                seen = int(np.searchsorted(at, length - n + t, side="right"))
                if not seen:
                    continue
                s = q[r, h * group: (h + 1) * group, t] @ k[:seen].T * scale
                w = np.exp(s - s.max(-1, keepdims=True))
                out[r, t, h * group: (h + 1) * group] = w / w.sum(-1, keepdims=True) @ v[:seen]
    return out
