"""Host side of the paged cache and the attention that reads it (include/vxs_sampler.h: vxs_kv_cache and after).

``KvCache``, ``KvPrep`` and ``SharedPrefix`` describe device memory of the caller's (torch tensors, ``hip.DeviceArray``
or addresses) and keep it alive; ``Context.kv_append_device``, ``attn_prompt_device`` and ``attn_step_device`` take
them. ``rope_frequencies`` gives the rotation's frequencies for long contexts too.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import numpy as np

from . import _lib
from ._lib import ptr

DTYPES = {"f32": _lib.VXS_F32, "bf16": _lib.VXS_BF16, "f16": _lib.VXS_F16}


class KvCache:
    """One layer's cache (vxs_kv_cache). `k`, `v`: pages * kv_heads * page_size * head_dim entries of `dtype`
    ("bf16" or "f16"), as [pages, kv_heads, page_size, head_dim] or with the given strides in entries; `table`: int32
    [slots, ld_table] page numbers."""

    def __init__(self, k, v, dtype: str, kv_heads: int, head_dim: int, pages: int, page_size: int, table, slots: int,
                 ld_table: int, page_stride: Optional[int] = None, head_stride: Optional[int] = None,
                 token_stride: Optional[int] = None):
        self._keep = (k, v, table)
        token = head_dim if token_stride is None else token_stride
        head = page_size * head_dim if head_stride is None else head_stride
        page = kv_heads * page_size * head_dim if page_stride is None else page_stride
        self.dtype, self.kv_heads, self.head_dim, self.page_size, self.slots = dtype, kv_heads, head_dim, page_size, slots
        self.struct = _lib.VxsKvCache(ptr(k), ptr(v), ptr(table), ld_table, page, head, token, slots, pages, page_size,
                                      kv_heads, head_dim, DTYPES[dtype])
        self.ref = ctypes.byref(self.struct)


class KvPrep:
    """What happens to query and key heads before attention (vxs_kv_prep): RMS norms with fp32 weights [head_dim]
    (None: none), then the rotation of the first `rot_dim` entries by position * inv_freq (fp32 [rot_dim / 2]),
    in pairs (i, i + rot_dim / 2), or (2i, 2i + 1) if `interleaved`; cosine and sine times `rope_scale`."""

    def __init__(self, q_norm=None, k_norm=None, eps: float = 1e-6, inv_freq=None, rot_dim: int = 0,
                 interleaved: bool = False, rope_scale: float = 1.0):
        self._keep = (q_norm, k_norm, inv_freq)
        self.struct = _lib.VxsKvPrep(ptr(q_norm), ptr(k_norm), ptr(inv_freq), eps, rope_scale, rot_dim, 1 if interleaved else 0)
        self.ref = ctypes.byref(self.struct)


class SharedPrefix:
    """Groups of rows whose first tokens are the same (vxs_shared_prefix): rows [off[g], off[g + 1]) share their
    first len[g] <= max_len tokens; `off` int32 [groups + 1], `length` int32 [groups], device memory. They are read once for
    a group where that is faster, with `always` in any case."""

    def __init__(self, groups: int, off, length, max_len: int, always: bool = False):
        self._keep = (off, length)
        self.struct = _lib.VxsSharedPrefix(ptr(off), ptr(length), groups, max_len, _lib.VXS_FLAG_SHARE_ALWAYS if always else 0)
        self.ref = ctypes.byref(self.struct)


def rope_frequencies(rot_dim: int, theta: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                     original_length: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0):
    """(inv_freq, rope_scale) of a rotation: float32 [rot_dim / 2] radians per position, theta^(-2i / rot_dim), and the
    magnitude of cosine and sine. For contexts `factor` times longer than the trained `original_length`:

    ``"linear"``  every frequency over `factor` (positions squeezed into the trained range);
    ``"ntk"``     (NTK-aware scaling) theta raised by factor^(rot_dim / (rot_dim - 2)): the lowest frequency over `factor`, the
                  highest kept;
    ``"yarn"``    (YaRN, Peng et al. 2023) frequencies that turn more than `beta_fast` times over `original_length` kept, those
                  under `beta_slow` turns over `factor`, a linear ramp over the index between; magnitude 0.1 ln(factor) + 1."""
    if rot_dim <= 0 or rot_dim % 2:
        raise ValueError("rot_dim must be positive and even")
    if not (theta > 0 and factor > 0):
        raise ValueError("theta and factor must be positive")
    i = np.arange(0, rot_dim, 2, dtype=np.float64)
    freq, scale = theta ** (-i / rot_dim), 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "ntk":
        if rot_dim < 4:
            raise ValueError("ntk scaling needs rot_dim >= 4")
        freq = (theta * factor ** (rot_dim / (rot_dim - 2))) ** (-i / rot_dim)
    elif scaling == "yarn":
        if original_length <= 0:
            raise ValueError("yarn scaling needs original_length")

        def index_of(turns: float) -> float:  # where a frequency makes so many turns over original_length
            return rot_dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(theta))

        low = max(math.floor(index_of(beta_fast)), 0)
        high = min(math.ceil(index_of(beta_slow)), rot_dim - 1)
        ramp = np.clip((i / 2 - low) / max(high - low, 1e-3), 0.0, 1.0)
        freq = freq / factor * ramp + freq * (1.0 - ramp)
        scale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    elif scaling is not None:
        raise ValueError(f"unknown scaling {scaling!r}")
    return freq.astype(np.float32), scale
