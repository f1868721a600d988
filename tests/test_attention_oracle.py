"""CPU checks of the attention oracle and of the host side of the paged cache."""
from __future__ import annotations

import ctypes
import math
import os
import subprocess
import textwrap

import numpy as np
import pytest

from oracle import attention_np as on
from voxwerk_amd import _lib
from voxwerk_amd.attention import rope_frequencies

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_bf16_rounds_to_nearest_even():
    x = np.array([1.0, 1.00390625, 1.01171875, 1.00391, -1.00391, 3.3895314e38, np.inf, -0.0, 1e-40], np.float32)
    got = on.widen(on.to_bf16(x))
    assert got[:5].tolist() == [1.0, 1.0, 1.015625, 1.0078125, -1.0078125]
    assert got[6] == np.inf and math.copysign(1, got[7]) == -1 and np.isnan(on.widen(on.to_bf16(np.array([np.nan]))))[0]


def test_attend_against_a_plain_sum():
    r = np.random.default_rng(0)
    q, k, v = r.standard_normal((3, 8)), r.standard_normal((5, 8)), r.standard_normal((5, 8))
    out, mean, *_ = on.attend(q, k, v, [0, 1, 5], 0.5)
    assert not out[0].any() and np.allclose(out[1], v[0])
    w = [math.exp(0.5 * sum(a * b for a, b in zip(q[2], kk))) for kk in k]
    assert np.allclose(out[2], sum(a * b for a, b in zip(w, v)) / sum(w))
    assert (np.abs(out) <= mean + 1e-12).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_keeps_lengths_and_relative_angles(interleaved):
    """A rotation keeps a pair's length, and products of rotated heads depend on the distance of their positions alone."""
    r = np.random.default_rng(1)
    freq, _ = rope_frequencies(16)
    x = r.standard_normal((2, 1, 24))
    a, _ = on.prep_heads(x, None, 0.0, [7, 19], freq, 16, interleaved)
    b, _ = on.prep_heads(x, None, 0.0, [1007, 1019], freq, 16, interleaved)
    assert np.allclose((a * a).sum(), (x * x).sum()) and np.array_equal(a[..., 16:], x[..., 16:])
    assert np.allclose(a[0, 0] @ a[1, 0], b[0, 0] @ b[1, 0])


def test_rope_frequencies():
    plain, one = rope_frequencies(128, 1e6)
    assert plain.dtype == np.float32 and one == 1.0 and plain[0] == 1.0
    assert np.allclose(plain, 1e6 ** (-np.arange(0, 128, 2) / 128), rtol=1e-6)
    linear, _ = rope_frequencies(128, 1e6, "linear", 4.0)
    assert np.allclose(linear, plain / 4, rtol=1e-6)
    ntk, _ = rope_frequencies(128, 1e6, "ntk", 4.0)
    assert ntk[0] == 1.0 and np.isclose(ntk[-1], plain[-1] / 4, rtol=1e-5)
    yarn, mag = rope_frequencies(128, 1e4, "yarn", 4.0, 4096)
    base, _ = rope_frequencies(128, 1e4)
    turns = 4096 * base / (2 * np.pi)
    assert np.allclose(yarn[turns > 40], base[turns > 40], rtol=1e-6) and np.allclose(yarn[turns < 0.8], base[turns < 0.8] / 4, rtol=1e-6)
    assert (np.diff(yarn) < 0).all() and np.isclose(mag, 0.1 * math.log(4) + 1)
    for bad in ({"rot_dim": 7}, {"rot_dim": 0}, {"rot_dim": 8, "theta": -1.0}, {"rot_dim": 8, "scaling": "other"},
                {"rot_dim": 8, "scaling": "yarn"}, {"rot_dim": 2, "scaling": "ntk"}):
        with pytest.raises(ValueError):
            rope_frequencies(**bad)


def test_attention_struct_layouts(tmp_path):
    """The cache's structures as a C compiler lays them out == what the bindings pass."""
    structs = {"vxs_kv_cache": _lib.VxsKvCache, "vxs_kv_prep": _lib.VxsKvPrep, "vxs_shared_prefix": _lib.VxsSharedPrefix}
    lines = []
    for name, s in structs.items():
        lines.append(f'printf("{name} %zu", sizeof({name}));')
        lines += [f'printf(" {f[0]}=%zu", offsetof({name}, {f[0]}));' for f in s._fields_]
        lines.append('printf("\\n");')
    src = tmp_path / "layout.c"
    src.write_text(textwrap.dedent("""
        #include <stdio.h>
        #include "vxs_sampler.h"
        int main(void) { %s return 0; }
    """) % "\n".join(lines))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, size, *fields = line.split()
        assert int(size) == ctypes.sizeof(structs[name])
        for f in fields:
            field, off = f.split("=")
            assert getattr(structs[name], field).offset == int(off)
