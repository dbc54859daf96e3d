"""The 4-bit key / value cache and the operators around it, restated in numpy for the tests: byte addresses one by one, quantisation
in the single roundings of its definition, attention, accounts, eviction, norms and rotation in 64 bits.  Test infrastructure only."""
from __future__ import annotations

import numpy as np

LARGEST = 65408.0


def _addresses(D: int, values: bool):
    """(byte, nibble, scale byte) in a tile of every (token, value): arrays [32, D]."""
    t, x = np.meshgrid(np.arange(32), np.arange(D), indexing="ij")
    G = D // 32
    if values:
        w, lane, e = x // 16, 16 * (t // 8) + x % 16, t % 8
        code, scale = 16 * D, 34 * D + 2 * (32 * (x // 32) + t)
    else:
        w, lane, e = (t // 4 % 2) * G + x // 32, 16 * (x // 8 % 4) + 4 * (t // 8) + t % 4, x % 8
        code, scale = 0, 32 * D + 2 * (G * t + x // 32)
    nibble = e // 2 + 4 * (e % 2)
    return code + ((w // 4 * 64 + lane) * 4 + w % 4) * 4 + nibble // 2, nibble % 2, scale


def decode_tile(tile: np.ndarray, values: bool) -> np.ndarray:
    """uint8 [36 D] -> float64 [32, D]."""
    byte, high, scale = _addresses(tile.size // 36, values)
    codes = (tile[byte] >> (4 * high)) & 15
    d = (tile[scale].astype(np.uint16) | (tile[scale + 1].astype(np.uint16) << 8)).view(np.float16)
    with np.errstate(invalid="ignore"):  # (scales that no token has may be anything)
        return (codes.astype(np.float64) - 8.0) * d.astype(np.float64)


def decode(cache: np.ndarray, table: np.ndarray, length: int, head: int):
    """(keys, values) float64 [length, D] of one sequence (its row of the page table) and key head."""
    pages, _, tiles, size = cache.shape
    k, v = np.zeros((length, size // 36)), np.zeros((length, size // 36))
    for t0 in range(0, length, 32):
        page = table[t0 // (32 * tiles)]
        n = min(32, length - t0)
        tile = cache[page, head, t0 % (32 * tiles) // 32]
        k[t0:t0 + n], v[t0:t0 + n] = decode_tile(tile, False)[:n], decode_tile(tile, True)[:n]
    return k, v


def _bf16(x: np.ndarray) -> np.ndarray:
    u = x.astype(np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)


def quantise(k: np.ndarray, v: np.ndarray):
    """float32 [..., D] -> what the cache stands for (float64), by its definition."""
    with np.errstate(all="ignore"):
        good = np.all((np.abs(k) < LARGEST) & (np.abs(v) < LARGEST), -1, keepdims=True)
        out = []
        for x in (k, v):
            g = np.where(good, x, 0).astype(np.float32).reshape(*x.shape[:-1], -1, 32)
            m = np.take_along_axis(g, np.argmax(np.abs(g), -1)[..., None], -1)
            d = _bf16(m * np.float32(-0.125)).astype(np.float16).astype(np.float32)
            c = np.clip(np.floor(g / d + np.float32(8.5)), 0, 15)
            c = np.where(d == 0, 8, c)
            out.append(((c.astype(np.float64) - 8) * d.astype(np.float64)).reshape(x.shape))
        return np.where(good, out[0], np.nan), np.where(good, out[1], 0.0)


def attention(q: np.ndarray, keys, values, scale: float, window: int):
    """q [new, group, D] of one key head over its [length, D] keys and values, all float64 -> (out, weights [new, group, length],
    scores, seen [new, length])."""
    n, length = q.shape[0], keys.shape[0]
    place = np.arange(length - n, length)[:, None]
    token = np.arange(length)[None]
    seen = token <= place
    if window:
        seen &= token > place - window
    with np.errstate(all="ignore"):
        s = np.einsum("ngd,td->ngt", q, keys) * scale
        s = np.where(seen[:, None], s, -np.inf)
        top = np.max(s, -1, keepdims=True, initial=-np.inf)
        e = np.where(seen[:, None], np.exp(s - np.where(np.isfinite(top), top, 0)), 0)
        total = e.sum(-1, keepdims=True)
        p = np.where(total == 0, 0, e / np.where(total == 0, 1, total))
        # a value that a row does not see is no part of its sum, whatever it is
        out = np.zeros(q.shape)
        for i in range(n):
            out[i] = p[i][:, seen[i]] @ values[seen[i]]
    return out, p, s, seen


def evict(accounts: np.ndarray, keep: int, recent: int) -> np.ndarray:
    """Places of the kept tokens of one sequence and key head; accounts [length]."""
    n = accounts.size
    if n <= keep:
        return np.arange(n)
    old = n - recent
    key = [(0 if np.isnan(a) else 1, -a if not np.isnan(a) else 0.0, t) for t, a in enumerate(accounts[:old].astype(np.float64))]
    best = sorted(t for _, _, t in sorted(key)[:keep - recent])
    return np.array(best + list(range(old, n)), dtype=np.int64)


def norm_rope(x: np.ndarray, positions, cos, sin, gain, eps: float, offset: float, norm: bool, interleaved: bool):
    """float64 [rows, heads, D] -> (result, sum of magnitudes behind each value)."""
    x = x.astype(np.float64)
    if norm:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        if gain is not None:
            x = x * (gain.astype(np.float64) + offset)
    half = cos.shape[1]
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y, size = x.copy(), np.abs(x)
    for r, p in enumerate(positions):
        if not 0 <= p < cos.shape[0]:
            y[r] = np.nan
            continue
        c, s = cos[p].astype(np.float64), sin[p].astype(np.float64)
        xa, xb = x[r][:, a], x[r][:, b]
        y[r][:, a], y[r][:, b] = xa * c - xb * s, xa * s + xb * c
        size[r][:, a] = size[r][:, b] = np.abs(xa) + np.abs(xb)
    return y, size
