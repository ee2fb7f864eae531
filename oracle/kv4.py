"""Oracle of the 4-bit paged KV cache and of what reads its logits' end: numpy, float64.

Written from the definitions alone: E2M1 elements with one power-of-two scale for 32
dims (OCP microscaling), attention over the values the cache stands for, the log
softmax of a row with its entropy and top values.
"""
from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantise(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """``x [..., 128]`` -> (codes ``[..., 128]`` 0..15, scale bytes ``[..., 4]``)."""
    x = np.asarray(x, np.float64).reshape(*x.shape[:-1], 4, 32)
    a = np.abs(x).max(-1)
    bad = ~np.isfinite(a)
    m, e = np.frexp(np.where(bad, 0.0, a))            # a = m 2^e with 0.5 <= m < 1
    e = np.clip(np.where(a == 0, -200, e - 1 + (m >= 0.875)) - 2, -125, 125).astype(int)
    y = np.where(bad[..., None], 0.0, np.abs(x) / np.ldexp(1.0, e)[..., None])
    mids = (GRID[1:] + GRID[:-1]) / 2
    # code i is reached past midpoint i - 1, or on it where i is even
    code = sum(((y >= mid) if i % 2 else (y > mid)).astype(int) for i, mid in enumerate(mids))
    code = code + 8 * np.signbit(x)
    code = np.where(bad[..., None], 0, code)
    return code.reshape(*code.shape[:-2], 128), np.where(bad, 255, e + 127)


def values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """float64 ``[..., 128]`` of codes and scale bytes."""
    x = np.where(codes & 8, -1.0, 1.0) * GRID[codes & 7]
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(int) - 127))
    return (x.reshape(*x.shape[:-1], 4, 32) * s[..., None]).reshape(x.shape)


def pack(codes: np.ndarray) -> np.ndarray:
    return (codes[..., ::2] | codes[..., 1::2] << 4).astype(np.uint8)


def rows(cache: np.ndarray, block_size: int) -> tuple[np.ndarray, np.ndarray, np.ndarray, np.ndarray]:
    """(K codes bytes, K scales, V codes bytes, V scales): views ``[blocks, Hkv, block, 64 | 4]``."""
    nb, hkv = cache.shape[:2]
    out = []
    for i in range(2):
        page = cache[:, :, i]
        out += [page[..., :block_size * 64].reshape(nb, hkv, block_size, 64),
                page[..., block_size * 64:].reshape(nb, hkv, block_size, 4)]
    return tuple(out)


def unpack_rows(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    both = np.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], 128)
    return values(both, scales)


def store(cache: np.ndarray, block_size: int, k: np.ndarray, v: np.ndarray, slots) -> None:
    """In place: row ``slots[t]`` of the cache gets ``k[t]``, ``v[t]``; slots outside are skipped."""
    nb, hkv = cache.shape[:2]
    half = block_size * 64
    for i, x in enumerate((k, v)):
        codes, scales = quantise(x)
        codes = pack(codes)
        for t, s in enumerate(slots):
            if 0 <= s < nb * block_size:
                b, r = divmod(int(s), block_size)
                cache[b, :, i, r * 64:r * 64 + 64] = codes[t]
                cache[b, :, i, half + r * 4:half + r * 4 + 4] = scales[t]


def load(cache: np.ndarray, block_size: int, slots) -> tuple[np.ndarray, np.ndarray]:
    kc, ks, vc, vs = rows(cache, block_size)
    nb, hkv = cache.shape[:2]
    out = np.zeros((2, len(slots), hkv, 128))
    for t, s in enumerate(slots):
        if 0 <= s < nb * block_size:
            b, r = divmod(int(s), block_size)
            out[0, t] = unpack_rows(kc[b, :, r], ks[b, :, r])
            out[1, t] = unpack_rows(vc[b, :, r], vs[b, :, r])
    return out[0], out[1]


def decode(q: np.ndarray, cache: np.ndarray, block_size: int, tables: np.ndarray, lens, scale: float):
    """(out, sum_t p_t |v_t|, max_t sum |q| |k_t| scale) of ``q [B, Hq, 128]``; a block outside
    the pool reads block 0, a context of none gives zeros."""
    kc, ks, vc, vs = rows(cache, block_size)
    nb, hkv = cache.shape[:2]
    n, hq, d = q.shape
    out, absv, size = np.zeros(q.shape), np.zeros(q.shape), np.zeros((n, hq, 1))
    g = hq // hkv
    for b in range(n):
        L = min(max(0, int(lens[b])), tables.shape[1] * block_size)
        if L == 0:
            continue
        t = tables[b, :-(-L // block_size)].astype(int)
        t = np.where((t < 0) | (t >= nb), 0, t)
        for h in range(hkv):
            k = unpack_rows(kc[t, h], ks[t, h]).reshape(-1, d)[:L]
            v = unpack_rows(vc[t, h], vs[t, h]).reshape(-1, d)[:L]
            for i in range(h * g, h * g + g):
                s = k @ q[b, i] * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                out[b, i], absv[b, i] = p @ v, p @ np.abs(v)
                size[b, i] = (np.abs(k) @ np.abs(q[b, i])).max() * abs(scale)
    return out, absv, size


def log_softmax(x: np.ndarray) -> np.ndarray:
    x = np.asarray(x, np.float64)
    with np.errstate(all="ignore"):
        m = x.max(-1, keepdims=True)
        d = x - m
        return d - np.log(np.exp(d).sum(-1, keepdims=True))


def entropy(x: np.ndarray) -> np.ndarray:
    lp = log_softmax(x)
    with np.errstate(all="ignore"):
        p = np.exp(lp)
        return -np.where(p == 0, 0.0, p * lp).sum(-1)


def top(x: np.ndarray, k: int) -> np.ndarray:
    """Indices of the k largest of each row: the lowest index first among equals, NaN largest."""
    x = np.asarray(x, np.float64) + 0.0
    key = np.where(np.isnan(x), np.inf, x)
    return np.stack([np.lexsort((np.arange(r.size), -r, ~np.isnan(o)))[:k]
                     for r, o in zip(key, x)]) if len(x) else np.zeros((0, k), int)
