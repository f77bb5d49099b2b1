"""Plain restatement of the compact latent cache and of eviction in numpy, 64 bits: the layout by byte address, the rounding
by search over the representable values, attention and accounts in float64, eviction by sorting."""
from __future__ import annotations

import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
E_MIN, E_MAX = -120, 125


def addresses(w, x):
    """Byte offsets in a tile of row x: K value bytes, V value bytes [w / 2], K scales, V scales [w / 32]."""
    b, byte = np.arange(w // 32), np.arange(w // 2)
    k = (byte // 16 // 4) * 1024 + x * 64 + (byte // 16 % 4) * 16 + byte % 16
    v = 8 * w + (x % 4 * 4 + x // 4) * (w // 2) + byte
    return k, v, 16 * w + x * (w // 32) + b % 4 * (w // 128) + b // 4, 16 * w + w // 2 + b * 16 + x


def quantise(rows):
    """(bytes [T, w / 2], scale bytes [T, w / 32]) of float rows [T, w]."""
    x = np.asarray(rows, np.float64).reshape(len(rows), rows.shape[1] // 32, 32)
    fine = np.isfinite(x).all(-1)
    x = np.where(fine[..., None], x, 0)
    most = np.abs(x).max(-1)
    e = np.full(most.shape, E_MIN)
    for up in range(E_MIN, E_MAX):
        e += most > 7 * 2.0 ** up
    off = np.abs(np.abs(x)[..., None] / (2.0 ** e)[..., None, None] - GRID) + np.arange(8) % 2 * 1e-9   # ties to even
    code = off.argmin(-1) + 8 * np.signbit(x)
    code = np.where(fine[..., None], code, 0).reshape(len(rows), rows.shape[1] // 2, 2).astype(np.uint8)
    return code[..., 0] | code[..., 1] << 4, np.where(fine, e + 127, 255).astype(np.uint8)


def values(code, scale):
    """Float64 values of quantise's bytes; blocks of scale 255 are NaN."""
    code = np.stack((code & 15, code >> 4), -1).reshape(len(code), 2 * code.shape[1])
    x = np.where(code & 8, -1, 1) * GRID[code & 7]
    s = np.where(scale == 255, np.nan, 2.0 ** (scale.astype(np.float64) - 127))
    return x * np.repeat(s, 32, axis=-1)


def tile_of(cache, slot):
    """The tile (a view) and the row in it of a slot of a cache [pages, block / 16, 17 w]."""
    block = cache.shape[1] * 16
    return cache[slot // block, slot % block // 16], slot % 16


def store(cache, key, value, slots):
    w = cache.shape[2] // 17
    (kc, ks), (vc, vs) = quantise(key), quantise(value)
    for t, slot in enumerate(slots):
        if 0 <= slot < cache.shape[0] * cache.shape[1] * 16:
            tile, x = tile_of(cache, int(slot))
            for at, data in zip(addresses(w, x), (kc[t], vc[t], ks[t], vs[t])):
                tile[at] = data


def load(cache, slots):
    """Rows [K | V] of slots, float64 [n, 2 w]."""
    w = cache.shape[2] // 17
    parts = [[], [], [], []]
    for slot in slots:
        tile, x = tile_of(cache, int(slot))
        for part, at in zip(parts, addresses(w, x)):
            part.append(tile[at])
    if not len(slots):
        return np.zeros((0, 2 * w))
    kc, vc, ks, vs = (np.stack(p) for p in parts)
    return np.concatenate((values(kc, ks), values(vc, vs)), 1)


def slots_of(table_row, block, n):
    j = np.arange(n)
    return table_row[j // block].astype(np.int64) * block + j % block


def attention(q, rows, scale):
    """o, lse of q [16, w] over rows [n, 2 w], and sum p |v| (what a relative error of the weights is worth)."""
    w = q.shape[1]
    if len(rows) == 0:
        return np.zeros_like(q), np.full(16, -np.inf), np.zeros_like(q)
    s = q @ rows[:, :w].T * scale
    m = s.max(1, keepdims=True)
    p = np.exp(s - m)
    total = p.sum(1, keepdims=True)
    p /= total
    return p @ rows[:, w:], (m + np.log(total))[:, 0], p @ np.abs(rows[:, w:])


def select(weights, positions, lengths, budgets, protect_from):
    """Lists per request: (length, weights, positions, source, target), padded as the operator pads them."""
    R, M = weights.shape
    out_w, out_p = np.zeros((R, M), np.float32), np.full((R, M), -1, np.int32)
    source, target = np.full((R, M // 2), -1, np.int32), np.full((R, M // 2), -1, np.int32)
    left = np.zeros(R, np.int32)
    for r in range(R):
        n = min(max(int(lengths[r]), 0), M)
        b = min(n, max(int(budgets[r]), 0))
        order = lambda j: (positions[r, j] < protect_from[r], np.isnan(weights[r, j]),
                           0 if np.isnan(weights[r, j]) else -weights[r, j], j)
        stay = set(sorted(range(n), key=order)[:b])
        holes, extra = [j for j in range(b) if j not in stay], sorted(j for j in stay if j >= b)
        assert len(holes) == len(extra)
        at = np.arange(b)
        at[holes] = extra
        left[r], out_w[r, :b], out_p[r, :b] = b, weights[r, at], positions[r, at]
        source[r, :len(extra)], target[r, :len(holes)] = extra, holes
    return left, out_w, out_p, source, target
