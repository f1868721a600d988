"""Host checks, without a GPU: what the C entry points of the paged caches refuse (and that nothing is launched then), and the
axes of frequencies."""
from __future__ import annotations

import ctypes
import os
import subprocess

import numpy as np
import pytest

from voxwerk_amd import _lib, build
from voxwerk_amd.attention import Kv8Cache, KvCache, KvPrep, RopeAxes, SharedPrefix, rope_axes

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BAD, UNSUPPORTED = _lib.VXS_ERR_INVALID_ARG, _lib.VXS_ERR_UNSUPPORTED
X = 1 << 20  # an address that nobody follows
ENTRIES = ("vxs_attn_prompt_device", "vxs_attn_cross_device", "vxs_attn8_prompt_device", "vxs_attn8_cross_device",
           "vxs_attn_step_device", "vxs_attn8_step_device")
APPENDS = ("vxs_kv_append_device", "vxs_kv_append_axes_device", "vxs_kv8_append_device")


@pytest.fixture(scope="module")
def api(tmp_path_factory):
    here = tmp_path_factory.mktemp("api")
    so, first = here / "api.so", here / "first.h"
    first.write_text("#include <algorithm>\nusing std::max;\nusing std::min;\n")  # (device functions in the headers name the compiler's)
    subprocess.run(["g++", "-std=c++17", "-O1", "-include", str(first), "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(build.ROCM, "include"),
                    "-I", build.INCLUDE, "-Wl,-z,defs", "-o", str(so), os.path.join(build.CSRC, "vxs_attn_api.cpp"),
                    os.path.join(REPO, "tests", "attention_refusals.cpp")], check=True)
    lib = ctypes.CDLL(str(so))
    for name, (res, args) in _lib._SIGNATURES.items():
        if name.startswith(("vxs_attn", "vxs_kv")):
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = res, args
    lib.test_context.restype = ctypes.c_void_p
    lib.vxs_last_error.restype, lib.vxs_last_error.argtypes = ctypes.c_char_p, [ctypes.c_void_p]
    return lib


def cache_for(name, **change):
    c = Kv8Cache(X, X, X, X, "bf16", 2, 64, 9, 16, X, 2, 5) if "8" in name else KvCache(X, X, "bf16", 2, 64, 9, 16, X, 2, 5)
    for field, value in change.items():
        setattr(c.struct, "q_dtype" if field == "dtype" and "8" in name else field, value)
    return c


def attend(api, name, cache=None, n=2, tokens=4, q_heads=4, q=X, ldq=256, off=X, lens=X, scale=0.1, out=X, ldo=256, out_dtype=1,
           max_len=40, prefix=None, work=None, work_bytes=0):
    c = cache or cache_for(name)
    head, fn = (api.test_context(), n), getattr(api, name)
    if "step" in name:
        return fn(*head, q_heads, q, ldq, c.ref, None, lens, max_len, prefix.ref if prefix else None, scale, out, ldo, out_dtype, work, work_bytes)
    return fn(*head, tokens, q_heads, q, ldq, c.ref, None, off, lens, scale, out, ldo, out_dtype)


def append(api, name, cache=None, tokens=2, q_heads=4, q=X, ldq=512, k=X, ldk=512, v=X, ldv=512, kind=0, pos=X, slots=X, index=X,
           out=X, ldo=256, prep="default", axes=None):
    c = cache or cache_for(name)
    prep = KvPrep(None, None, 0.0, X, 64) if prep == "default" else prep
    more = () if name == "vxs_kv_append_device" else (axes.ref if axes is not None else None,)
    return getattr(api, name)(api.test_context(), tokens, q_heads, q, ldq, k, ldk, v, ldv, kind, prep.ref if prep else None, *more,
                              pos, slots, index, c.ref, out, ldo, None)


@pytest.fixture()
def refused(api):
    before = api.test_launches()

    def check(code, fn, *args, **kw):
        assert fn(api, *args, **kw) == code, (args, kw)
        assert api.vxs_last_error(api.test_context()), "no text"
        assert api.test_launches() == before, "launched"

    return check


@pytest.mark.parametrize("name", ENTRIES + APPENDS)
def test_caches_that_are_refused(refused, name):
    fn = attend if "attn" in name else append
    for change in ({"pages": 0}, {"slots": -1}, {"page_size": 0}, {"kv_heads": 0}, {"ld_table": 0}, {"dtype": 0}, {"dtype": 9},
                   {"k": None}, {"v": None}, {"table": None}, {"token_stride": 63}, {"head_stride": 0}, {"page_stride": -8}, {"kv_heads": 3}):
        refused(BAD, fn, name, cache=cache_for(name, **change))
    for change in ({"head_dim": 32}, {"head_dim": 60, "token_stride": 64}, {"page_size": 24}, {"page_size": 8}, {"page_size": 1 << 17},
                   {"token_stride": 68}, {"head_stride": 1028}, {"page_stride": 2052}, {"k": X + 2}, {"v": X + 8}, {"ld_table": 1 << 27},
                   {"token_stride": 1 << 26}, {"page_stride": 1 << 31}):
        refused(UNSUPPORTED, fn, name, cache=cache_for(name, **change))
    if "8" in name:
        for change in ({"k_scale": None}, {"v_scale": None}):
            refused(BAD, fn, name, cache=cache_for(name, **change))
        for change in ({"k_scale": X + 2}, {"v_scale": X + 1}, {"token_stride": 72}, {"head_stride": 1032}, {"page_stride": 2056}):
            refused(UNSUPPORTED, fn, name, cache=cache_for(name, **change))


@pytest.mark.parametrize("name", ENTRIES)
def test_attention_that_is_refused(refused, name):
    for kw in ({"q_heads": 3}, {"q_heads": 0}, {"ldq": 248}, {"ldo": 248}, {"scale": 0.0}, {"scale": -1.0}, {"scale": float("nan")},
               {"scale": float("inf")}, {"out_dtype": 2}, {"out_dtype": 7}, {"q": None}, {"out": None}, {"lens": None}, {"n": -1}):
        refused(BAD, attend, name, **kw)
    for kw in ({"ldq": 260}, {"ldo": 260}, {"q": X + 8}, {"out": X + 4}):
        refused(UNSUPPORTED, attend, name, **kw)
    if "step" not in name:
        refused(BAD, attend, name, tokens=-1)
        refused(BAD, attend, name, off=None)
        refused(UNSUPPORTED, attend, name, tokens=1 << 30)
        return
    odd = SharedPrefix(1, X, X, 4)
    odd.struct.flags = 1
    for kw in ({"max_len": -1}, {"prefix": SharedPrefix(-1, X, X, 4)}, {"prefix": SharedPrefix(1, None, X, 4)},
               {"prefix": SharedPrefix(1, X, None, 4)}, {"prefix": SharedPrefix(1, X, X, -4)}, {"prefix": odd},
               {"work": X + 4, "work_bytes": 1 << 16}, {"n": 1, "max_len": 1 << 20, "cache": cache_for(name, ld_table=1 << 16), "work": X, "work_bytes": 16}):
        refused(BAD, attend, name, **kw)


@pytest.mark.parametrize("name", APPENDS)
def test_appends_that_are_refused(refused, name):
    prep = lambda *a: {"prep": KvPrep(*a)}  # noqa: E731
    for kw in ({"tokens": -1}, {"q_heads": 3}, {"q_heads": 0}, {"q": None, "k": None, "v": None}, {"v": None}, {"out": None}, {"pos": None},
               {"ldq": 252}, {"ldk": 124}, {"ldv": 124}, {"ldo": 252}, {"kind": 3}, {"kind": -1}, prep(None, None, 0.0, None, 64),
               prep(None, None, 0.0, X, 66), prep(None, None, 0.0, X, -8), prep(None, None, 0.0, X, 7), prep(X, None, -1.0), prep(None, X, float("nan"))):
        refused(BAD, append, name, **kw)
    for kw in ({"ldq": 514}, {"ldk": 514}, {"ldv": 513}, {"ldo": 258}, {"q": X + 4}, {"k": X + 8}, {"out": X + 4},
               prep(None, None, 0.0, X, 12), prep(None, None, 0.0, X + 4, 64), {"tokens": 1 << 24}):
        refused(UNSUPPORTED, append, name, **kw)
    if name == "vxs_kv_append_device":
        return
    for axes, kw in ((RopeAxes(X, 0, 64), {}), (RopeAxes(X, -1, 64), {}), (RopeAxes(None, 3, 64), {}), (RopeAxes(X, 3, 1), {}), (RopeAxes(X, 3, 64), {"index": None})):
        refused(BAD, append, name, axes=axes, **kw)
    refused(UNSUPPORTED, append, name, axes=RopeAxes(X + 4, 3, 64))


def test_what_is_not_refused(api):
    for name in ENTRIES:
        before = api.test_launches()
        assert attend(api, name) == 0 and attend(api, name, out_dtype=0) == 0
        assert api.test_launches() == before + 2
        assert attend(api, name, n=0) == 0 and ("step" in name or attend(api, name, tokens=0) == 0)
        assert api.test_launches() == before + 2, "nothing to do is no launch"
    for name in APPENDS:
        before = api.test_launches()
        assert append(api, name) == 0 and append(api, name, k=None, v=None, index=None) == 0 and append(api, name, q=None, out=None) == 0
        assert append(api, name, prep=None, pos=None) == 0
        if name != "vxs_kv_append_device":
            assert append(api, name, axes=RopeAxes(X, 3, 2)) == 0 and append(api, name, k=None, v=None, index=None, axes=RopeAxes(X, 3, 2)) == 0
        assert append(api, name, tokens=0) == 0
        assert api.test_launches() == before + (4 if name == "vxs_kv_append_device" else 6)
    for name in ("vxs_attn_step_workspace", "vxs_attn8_step_workspace"):
        c = cache_for(name, ld_table=1000)
        assert getattr(api, name)(api.test_context(), 1, 4, c.ref, 4000, None) > 0
        assert getattr(api, name)(api.test_context(), -1, 4, c.ref, 4000, None) == BAD
        assert getattr(api, name)(None, 1, 4, c.ref, 4000, None) == BAD


def test_rope_axes():
    assert rope_axes([2, 1, 1]).tolist() == [0, 0, 1, 2] and rope_axes([3]).tolist() == [0, 0, 0]
    mixed = rope_axes([24, 20, 20], interleaved=True)
    assert mixed.dtype == np.int32 and [int((mixed == a).sum()) for a in range(3)] == [24, 20, 20]
    assert mixed[:7].tolist() == [0, 1, 2, 0, 1, 2, 0] and mixed[57:].tolist() == [0, 1, 2, 0, 0, 0, 0]
    assert rope_axes([0, 2]).tolist() == [1, 1]
    for bad in ([], [0, 0], [-1, 3]):
        with pytest.raises(ValueError):
            rope_axes(bad)
    with pytest.raises(ValueError):
        rope_axes([1, 1, 9], interleaved=True)


def test_structures_match_the_header(tmp_path):
    """The sizes and places of the fields that Python fills are the compiler's."""
    structs = {"vxs_kv_cache": _lib.VxsKvCache, "vxs_kv8_cache": _lib.VxsKv8Cache, "vxs_rope_axes": _lib.VxsRopeAxes,
               "vxs_kv_prep": _lib.VxsKvPrep, "vxs_shared_prefix": _lib.VxsSharedPrefix}
    lines = [f'printf("{name} %zu", sizeof({name}));' + "".join(f'printf(" %zu", offsetof({name}, {f}));' for f, _ in cls._fields_) + 'printf("\\n");'
             for name, cls in structs.items()]
    src, exe = tmp_path / "s.c", tmp_path / "s"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "vxs_sampler.h"\nint main(void) {' + "\n".join(lines) + "return 0; }\n")
    subprocess.run(["gcc", "-I", build.INCLUDE, str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        name, *numbers = line.split()
        cls = structs[name]
        assert [int(n) for n in numbers] == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_], name
