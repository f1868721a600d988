"""The 8-bit cache's oracle, pinned: e4m3 against torch's, scales against their definition, blocks that grow."""
from __future__ import annotations

import numpy as np
import torch

from oracle import attention8_np as o8


def test_values_and_rounding_match_torch():
    bytes_ = torch.arange(256, dtype=torch.uint8)
    assert np.array_equal(o8.VALUES, bytes_.view(torch.float8_e4m3fn).double().numpy(), equal_nan=True)
    mid = (o8.VALUES[:126] + o8.VALUES[1:127]) / 2
    near = np.concatenate([mid, np.nextafter(mid, 1e9), np.nextafter(mid, 0), o8.VALUES[:127], np.geomspace(1e-6, 448, 5000)]).astype(np.float32)
    x = np.concatenate([near, -near])
    x = x[np.abs(x) <= 448]
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(o8.encode(x), want)
    assert (o8.encode([np.nan, np.inf]) == 0x7F).all()


def test_scales_are_the_least():
    top = np.concatenate([np.geomspace(1e-30, 1e30, 4000), 448 * 2.0 ** np.arange(-100, 100), np.nextafter(448 * 2.0 ** np.arange(-100, 100), np.inf)])
    b = o8.byte_for(top)
    assert (top <= 448 * o8.power(b)).all() and (top > 448 * o8.power(b - 1)).all()
    assert (o8.byte_for([0.0, 1e-40]) == 1).all()


def test_a_larger_scale_changes_only_small_entries():
    """Divided by a power of two, an entry keeps its bits unless it falls below 2^-6, where the steps are 2^-9."""
    for by in range(1, 12):
        x = o8.VALUES[:127]
        y = o8.VALUES[o8.encode(x * 2.0**-by)]
        assert (y[x * 2.0**-by >= 2.0**-6] == (x * 2.0**-by)[x * 2.0**-by >= 2.0**-6]).all()
        assert (np.abs(y - x * 2.0**-by) <= 2.0**-10).all()


def test_append_finds_blocks():
    scales = np.full((3, 2), 120)
    x = np.array([[1.0, -3.0], [500.0, 2.0], [np.inf, 7.0]])
    got = o8.append(None, scales, [(1, 15), (1, 16), (2, 3)], x)
    assert set(got) == {(1, 0), (1, 1), (2, 0)}
    assert got[1, 0][:2] == (120, 120) and got[1, 1][:2] == (128, 128)  # (16 begins a block: its old scale counts for nothing)
    assert got[2, 0][0] == 121 or got[2, 0][:2] == (121, 121)
    assert got[1, 1][2].tolist() == [1] + [-1] * 15


def test_append_takes_infinite_entries_for_none():
    """A block's scale is that of its finite entries: an infinite one beside 7 asks for 7's, which is larger than the old one."""
    got = o8.append(None, np.full((3, 2), 120), [(2, 3)], np.array([[np.inf, 7.0]]))
    assert set(got) == {(2, 0)} and got[2, 0][:2] == (121, 121) and got[2, 0][2].tolist() == [-1] * 3 + [0] + [-1] * 12
