"""Binary64 oracle of the token-by-token serving operators (test infrastructure only).

Restates from their definitions, in numpy: the head norm and rotation, the 4-bit
cache format (quantise, pack, unpack) and the attention over cached rows.
"""
from __future__ import annotations

import numpy as np

GROUP, TILE = 32, 16
F16_MAX = 65504.0


# ---- head norm + rotation
def axis_of_pair(axis_pairs) -> np.ndarray:
    return np.repeat(np.arange(len(axis_pairs)), axis_pairs)


def norm(x: np.ndarray, weight, eps: float) -> np.ndarray:
    y = x / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + eps)
    return y if weight is None else y * weight


def pair_channels(rotary: int, interleaved: bool) -> tuple:
    j = np.arange(rotary // 2)
    return (2 * j, 2 * j + 1) if interleaved else (j, j + rotary // 2)


def qk_norm_rope(x, positions, frequencies, axis_pairs, interleaved=False, weight=None, eps=1e-6, normalize=True):
    """x [tokens][heads][dim] float64, positions [tokens][axes] -> float64."""
    y = norm(x, weight, float(np.float32(eps))) if normalize else x.copy()
    angle = positions[:, axis_of_pair(axis_pairs)].astype(np.float64) * frequencies
    cos, sin = np.cos(angle)[:, None], np.sin(angle)[:, None]
    ca, cb = pair_channels(2 * len(frequencies), interleaved)
    out = y.copy()
    out[..., ca] = y[..., ca] * cos - y[..., cb] * sin
    out[..., cb] = y[..., cb] * cos + y[..., ca] * sin
    return out


# ---- the cache format
_POSITIVE = np.arange(0x7C00, dtype=np.uint16).view(np.float16).astype(np.float64)
_FINITE = np.concatenate([-_POSITIVE[:0:-1], _POSITIVE])


def quantise(x: np.ndarray) -> tuple:
    """x [..., dim] float64 -> codes [..., dim] uint8, s, z [..., dim / 32] float64 (z NaN for a NaN group)."""
    y = np.clip(x, -F16_MAX, F16_MAX).reshape(*x.shape[:-1], -1, GROUP)
    bad = np.isnan(y).any(-1)
    y = np.where(bad[..., None], 0.0, y)
    lo, hi = y.min(-1), y.max(-1)
    z = _FINITE[np.searchsorted(_FINITE, lo, side="right") - 1]
    s = _POSITIVE[np.searchsorted(15.0 * _POSITIVE, hi - z, side="left")]
    s, z = np.where(bad, 0.0, s), np.where(bad, np.nan, z)
    with np.errstate(divide="ignore", invalid="ignore"):
        code = np.where(s[..., None] > 0, np.rint((y - z[..., None]) / s[..., None]), 0.0)
    return code.astype(np.uint8).reshape(x.shape), s, z


def values(codes: np.ndarray, s: np.ndarray, z: np.ndarray) -> np.ndarray:
    c = codes.reshape(*codes.shape[:-1], -1, GROUP).astype(np.float64)
    return (z[..., None] + s[..., None] * c).reshape(codes.shape)


def tile_bytes(dim: int) -> int:
    return 2 * TILE * (dim // 2 + dim // GROUP * 4)


def _places(dim: int) -> tuple:
    c = np.arange(dim)
    halfword = (c % 32) // 4 * (dim // 32) + c // 32
    return 2 * halfword + (c % 4) // 2, c % 2


class Cache:
    """A cache in host memory: bytes as the library lays them out."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, dim: int, fill: int = 0):
        self.page_size, self.kv_heads, self.dim, self.pages = page_size, kv_heads, dim, pages
        self.data = np.full((pages, kv_heads, page_size // TILE, tile_bytes(dim)), fill, dtype=np.uint8)

    def _at(self, page: int, head: int, slot: int, which: int) -> tuple:
        tile = self.data[page, head, slot // TILE]
        half = tile[which * (tile_bytes(self.dim) // 2):][: tile_bytes(self.dim) // 2]
        codes = half[: TILE * self.dim // 2].reshape(TILE, -1)[slot % TILE]
        params = half[TILE * self.dim // 2:].reshape(TILE, -1)[slot % TILE]
        return codes, params

    def write(self, page: int, slot: int, head: int, which: int, x: np.ndarray) -> None:
        c, s, z = quantise(x)
        codes, params = self._at(page, head, slot, which)
        byte, high = _places(self.dim)
        codes[:] = 0
        np.bitwise_or.at(codes, byte, (c << (4 * high)).astype(np.uint8))
        params.view(np.float16)[0::2] = s
        params.view(np.float16)[1::2] = z

    def parts(self, page: int, slot: int, head: int, which: int) -> tuple:
        codes, params = self._at(page, head, slot, which)
        byte, high = _places(self.dim)
        p = params.view(np.float16).astype(np.float64)
        return ((codes[byte] >> (4 * high)) & 15).astype(np.uint8), p[0::2], p[1::2]

    def rows(self, table_row: np.ndarray, first: int, last: int, head: int, which: int) -> tuple:
        """(values, |z| + 15 s per channel) of positions first..last-1 of a sequence."""
        out, size = np.zeros((last - first, self.dim)), np.zeros((last - first, self.dim))
        for i, p in enumerate(range(first, last)):
            c, s, z = self.parts(int(table_row[p // self.page_size]), p % self.page_size, head, which)
            out[i] = values(c, s, z)
            size[i] = np.repeat(np.abs(z) + 15.0 * s, GROUP)
        return out, size


def attention(cache: Cache, table_row, length: int, q: np.ndarray, scale: float, causal=True, window=0) -> tuple:
    """q [n][heads][dim] of one sequence that holds `length` tokens, the n of q the last of them.
    -> out [n][heads][dim], lse [n][heads], weight [n][heads][dim] (the mean of |z| + 15 s of the
    values under the softmax), reach [n][heads] (the largest scale * sum |q| (|z| + 15 s) of the keys)
    and the largest |z| + 15 s of a value."""
    n, heads, dim = q.shape
    share = heads // cache.kv_heads
    out, weight = np.zeros(q.shape), np.zeros(q.shape)
    lse, reach, largest = np.full((n, heads), -np.inf), np.zeros((n, heads)), 0.0
    for kvh in range(cache.kv_heads):
        k, ks = cache.rows(table_row, 0, length, kvh, 0)
        v, vs = cache.rows(table_row, 0, length, kvh, 1)
        largest = max(largest, np.nanmax(vs, initial=0.0))
        for t in range(n):
            last = length - n + t if causal else length - 1
            first = max(0, last - window + 1) if window else 0
            if last < first:
                continue
            sl = slice(first, last + 1)
            for h in range(kvh * share, (kvh + 1) * share):
                x = k[sl] @ q[t, h] * scale
                top = x.max() if not np.isnan(x).any() else np.nan
                e = np.exp(x - top)
                total = e.sum()
                out[t, h], lse[t, h] = e @ v[sl] / total, top + np.log(total)
                weight[t, h] = e @ vs[sl] / total
                reach[t, h] = (ks[sl] @ np.abs(q[t, h])).max() * abs(scale)
    return out, lse, weight, reach, largest
