"""The paged cache's operators in 64 bits, from their definitions (test infrastructure).

Arrays are numpy; 16-bit entries come as uint16 (bf16) or float16 and are widened exactly.
"""
from __future__ import annotations

import numpy as np

UNIT = {"bf16": 2.0**-8, "f16": 2.0**-11, "f32": 2.0**-24}  # half an ulp over the least value that has it


def to_bf16(x: np.ndarray) -> np.ndarray:
    """fp32 to bf16 bits, to nearest even; a NaN stays one."""
    b = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32)
    r = ((b + np.uint32(0x7FFF) + ((b >> np.uint32(16)) & np.uint32(1))) >> np.uint32(16)).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def pack(x: np.ndarray, dtype: str) -> np.ndarray:
    if dtype == "bf16":
        return to_bf16(np.asarray(x, np.float32))
    return np.asarray(x, np.float16 if dtype == "f16" else np.float32)


def widen(x: np.ndarray) -> np.ndarray:
    if x.dtype == np.uint16:
        return (x.astype(np.uint32) << np.uint32(16)).view(np.float32).astype(np.float64)
    return x.astype(np.float64)


def prep_heads(x, weight, eps, pos, inv_freq, rot, interleaved, rope_scale=1.0):
    """x [tokens, heads, dim] fp64: the norm of each head, then its rotation; and the magnitude that the
    rotation's errors scale with (|a| + |b| of each pair)."""
    x = np.array(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    mag = np.zeros_like(x)
    if rot:
        a, b = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if interleaved else (np.arange(rot // 2), np.arange(rot // 2, rot))
        # whole turns leave the angle before the cosine sees it, in extended precision
        angle = np.fmod(np.asarray(pos, np.longdouble)[:, None] * np.asarray(inv_freq, np.longdouble)[None],
                        2 * np.arctan2(np.longdouble(0), np.longdouble(-1)))
        c, s = np.cos(angle).astype(np.float64)[:, None] * rope_scale, np.sin(angle).astype(np.float64)[:, None] * rope_scale
        xa, xb = x[..., a].copy(), x[..., b].copy()
        x[..., a], x[..., b] = xa * c - xb * s, xa * s + xb * c
        mag[..., a] = mag[..., b] = (np.abs(xa) + np.abs(xb)) * abs(rope_scale)
    return x, mag


def gather(cache: np.ndarray, table_row, n: int, page: int, head: int) -> np.ndarray:
    """The first n entries of one slot and head of cache [pages, heads, page, dim], widened."""
    if n == 0:
        return np.zeros((0, cache.shape[-1]))
    t = np.arange(n)
    return widen(cache[np.asarray(table_row)[t // page], head, t % page])


def attend(q, k, v, limit, scale):
    """softmax(scale q k^T) v, row i over the first limit[i] keys, zeros for none; and for the error bound of each
    row: the mean of |v| under its weights, the largest |q| . |k| and the largest |score|."""
    q = np.asarray(q, np.float64)
    out = np.zeros((len(q), v.shape[1]))
    mean, reach, top = np.zeros_like(out), np.zeros(len(q)), np.zeros(len(q))
    for i, n in enumerate(limit):
        if n <= 0:
            continue
        s = k[:n] @ q[i] * scale
        w = np.exp(s - s.max())
        w /= w.sum()
        out[i] = w @ v[:n]
        mean[i] = w @ np.abs(v[:n])
        reach[i] = (np.abs(k[:n]) @ np.abs(q[i])).max() * scale
        top[i] = np.abs(s).max()
    return out, mean, reach, top


def bound(out, mean, reach, top, limit, dim, dtype, out_dtype):
    """The largest error of an fp32 computation whose weights are rounded to `dtype` (to twice its bits or more for
    fp32 outputs). A score is off by (dim + 2) 2^-24 |q|.|k| from its sum and by |score| 2^-22 in the exponent's argument, an
    exponential by 2^-20 of itself; a weight's rounding is half an ulp, and for fp16 at least 2^-25 of the largest weight (the kernels
    keep more: closed forms hold them to that, this is for entries at random);
    sums of n terms are off by n 2^-24. Numerator and denominator may err in opposite directions."""
    n = np.maximum(np.asarray(limit, np.float64), 0)
    e = (dim + 2) * 2.0**-24 * reach + top * 2.0**-22 + 2.0**-20
    unit = UNIT[dtype] if out_dtype != "f32" else UNIT[dtype] ** 2 * 2
    unit = unit + (n * 2.0**-25 if dtype == "f16" else 0.0)
    weight = 2 * e + unit + 2 * n * 2.0**-24
    least = {"bf16": 2.0**-133, "f16": 2.0**-24, "f32": 2.0**-149}[out_dtype]
    return (2 * weight)[:, None] * mean + UNIT[out_dtype] * np.abs(out) + least
