"""The 8-bit KV pool in 64 bits: a row's scale byte, its e4m3 codes, and the
values codes and bytes stand for.  Written from the definition: e is the
smallest integer >= 1 with max |x| <= 448 * 2^(e - 127); a code is the row over
that scale rounded to the nearest e4m3 value, ties to the even code."""

from __future__ import annotations

import numpy as np


def _e4m3_values() -> np.ndarray:
    """The 127 non-negative finite e4m3 values, by code."""
    code = np.arange(127)
    exp, man = code >> 3, code & 7
    return np.where(exp == 0, man * 2.0 ** -9, (8 + man) * 2.0 ** (exp - 10.0))


VALUES = _e4m3_values()


def encode(x: np.ndarray) -> np.ndarray:
    """Nearest e4m3 code of every finite x with |x| <= 448."""
    a = np.abs(x)
    hi = np.clip(np.searchsorted(VALUES, a), 1, 126)
    lo = hi - 1
    down, up = a - VALUES[lo], VALUES[hi] - a
    code = np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    return (code | (np.signbit(x) * 0x80)).astype(np.uint8)


def decode(codes: np.ndarray) -> np.ndarray:
    mag = codes & 0x7F
    v = np.where(mag == 127, np.nan, VALUES[np.minimum(mag, 126)])
    return np.where(codes & 0x80, -v, v)


def quantise(rows: np.ndarray, is_v: bool) -> tuple[np.ndarray, np.ndarray]:
    """(codes, scale bytes) of rows (..., D)."""
    rows = rows.astype(np.float64)
    bad = ~(np.abs(rows) < 248 * 2.0 ** 120).all(-1)
    x = np.where(bad[..., None], 0.0, rows)
    top = np.abs(x).max(-1)
    e = np.ones(top.shape, np.int64)
    for b in range(254, 1, -1):       # the smallest byte that holds the row
        e = np.where(top > 448.0 * 2.0 ** (b - 128), np.maximum(e, b), e)
    codes = encode(x / 2.0 ** (e[..., None] - 127.0))
    codes[bad] = 0 if is_v else 0x7F
    return codes, np.where(bad, 255, e).astype(np.uint8)


def dequantise(codes: np.ndarray, e: np.ndarray) -> np.ndarray:
    v = decode(codes) * 2.0 ** (e[..., None].astype(np.float64) - 127.0)
    return np.where(e[..., None] == 255, np.nan, v)
