"""The 8-bit cache's entries, scales and appends from their definitions (test infrastructure).

An entry is a byte of OCP e4m3 (bias 7, no infinities, 0x7F and 0xFF NaN), a scale a byte b that stands for 2^(b - 127).
"""
from __future__ import annotations

import numpy as np

BLOCK = 16


def _values() -> np.ndarray:
    b = np.arange(256)
    e, m = b >> 3 & 15, b & 7
    x = np.where(e > 0, (8 + m) * 2.0 ** (e - 10.0), m * 2.0**-9)
    x[(b & 127) == 127] = np.nan
    return np.where(b & 128, -x, x)


VALUES = _values()


def encode(x: np.ndarray) -> np.ndarray:
    """The nearest entries, ties to the even byte; what is not finite is NaN. Nothing may pass 464 (448 and half a step)."""
    x = np.asarray(x, np.float64)
    size = np.where(np.isfinite(x), np.abs(x), 0.0)
    assert size.max(initial=0.0) <= 464.0
    table = VALUES[:127]
    above = np.minimum(np.searchsorted(table, size), 126)
    below = np.maximum(above - 1, 0)
    lo, hi = size - table[below], table[above] - size
    code = np.where((hi < lo) | ((hi == lo) & (above % 2 == 0)), above, below)
    code = np.where(np.isfinite(x), code, 127)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def byte_for(top) -> np.ndarray:
    """The least scale, from byte 1, at which `top` >= 0 is at most 448."""
    m, e = np.frexp(np.asarray(top, np.float64))  # top = m 2^e, m from 1/2; 448 = 7/8 2^9
    return np.where(m > 0, np.maximum(e - 9 + (m > 0.875) + 127, 1), 1).astype(np.int64)


def power(byte) -> np.ndarray:
    return 2.0 ** (np.asarray(byte, np.float64) - 127)


def append(entries, scales, places, x, err=0.0):
    """One call's tokens of one head: entries [pages, page, dim] and scales [pages, page / 16] in bytes, places [(page, inside)]
    of tokens x [tokens, dim] (the value of each in 64 bits, off by at most err [tokens, dim] in the computation checked).
    Returns, for each block that the call touches, {(page, block): (low, high, rows)}: the scale's bytes that `err` allows, and
    for each of the block's places the token whose value it gets, or -1."""
    x, err = np.asarray(x, np.float64), np.broadcast_to(err, np.shape(x))
    blocks = {}
    for t, (p, i) in enumerate(places):
        blocks.setdefault((p, i // BLOCK), np.full(BLOCK, -1))[i % BLOCK] = t
    found = {}
    for (p, b), rows in blocks.items():
        at = rows[rows >= 0]
        size = np.where(np.isfinite(x[at]), np.abs(x[at]), 0.0)
        old = 1 if rows[0] >= 0 else int(scales[p, b])
        slack = np.where(np.isfinite(x[at]), err[at], 0.0)
        low, high = (max(int(byte_for((np.maximum(size + s, 0.0)).max())), old) for s in (-slack, slack))
        found[p, b] = (low, high, rows)
    return found
