"""GPU checks of vxs_kv_append_device against the 64-bit oracle: norms, both rotation layouts, parts of a head, types,
pages and layouts, tokens outside the cache, refusals."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import attention_np as on
from voxwerk_amd import _lib, hip
from voxwerk_amd.attention import KvCache, KvPrep, rope_frequencies
from voxwerk_amd.sampler import SamplerError

from attention_cases import Paged, device, out_array, as_out, rows_of

pytestmark = pytest.mark.gpu

# (q_heads, kv_heads, dim, rot, interleaved, norm, in, dtype, page, order)
SHAPES = [
    (16, 8, 128, 128, False, True, "f32", "bf16", 16, "heads"),
    (16, 8, 128, 128, True, True, "bf16", "bf16", 16, "tokens"),
    (5, 1, 64, 64, False, False, "f32", "f16", 32, "heads"),
    (4, 4, 64, 32, False, True, "f16", "f16", 64, "tokens"),
    (4, 2, 64, 8, True, True, "bf16", "f16", 16, "heads"),
    (2, 2, 256, 256, False, True, "f32", "bf16", 16, "heads"),
    (6, 3, 256, 96, False, False, "bf16", "bf16", 128, "tokens"),
    (3, 1, 256, 64, True, True, "f16", "bf16", 16, "heads"),
    (2, 1, 128, 0, False, True, "f32", "f16", 16, "heads"),
    (2, 1, 128, 0, False, False, "f32", "bf16", 16, "heads"),
    (40, 8, 128, 64, True, False, "f32", "bf16", 16, "heads"),
]


def tolerance(y, mag, dim, normed, dtype):
    """An angle is off by 2^-24 of a turn and the fp32 sine and cosine by 2^-18, so a rotated entry by 2^-17 of |a| + |b|;
    the norm's sum of dim squares, root, division and products by (dim + 8) 2^-24; then half an ulp."""
    rel = (dim + 8) * 2.0**-24 if normed else 2.0**-23
    least = 2.0**-24 if dtype == "f16" else 2.0**-133
    return np.abs(y) * (on.UNIT[dtype] + rel) + mag * (2.0**-17 + rel) + least


def run(ctx, paged, q_heads, x, in_dtype, tokens, pos, slots, index=None, prep=None, parts="qkv", status=True):
    """x [tokens, (q + 2 kv) heads * dim + pad]; returns q_out and the status."""
    d, kh, ld = paged.dim, paged.kv_heads, x.shape[1]
    dx = device(x)
    size = x.itemsize
    q = dx.ptr if "q" in parts else None
    k, v = (dx.ptr + size * q_heads * d, dx.ptr + size * (q_heads + kh) * d) if "k" in parts else (None, None)
    out, st = out_array(tokens, q_heads * d + 4, paged.dtype), device(np.full(tokens, 9, np.int32)) if status else None
    keep = [None if a is None else device(np.array(a, np.int32)) for a in (pos, slots, index)]
    hip.synchronize()
    ctx.kv_append_device(tokens, q_heads, q, ld, k, ld, v, ld, in_dtype, paged.cache, keep[0], keep[1], out, q_heads * d + 4,
                         prep=prep, index=keep[2], status=st)
    ctx.synchronize()
    raw = out.numpy()
    assert (raw[:, q_heads * d:] == 7).all(), "the pad was written"
    return raw, st.numpy() if status else None


@pytest.mark.parametrize("tokens", [1, 3, 300])
@pytest.mark.parametrize("q_heads,kv_heads,dim,rot,interleaved,norm,in_dtype,dtype,page,order", SHAPES)
def test_append(ctx, q_heads, kv_heads, dim, rot, interleaved, norm, in_dtype, dtype, page, order, tokens):
    r = np.random.default_rng(dim + rot + tokens)
    lens = [max(1, tokens // 3), tokens - 2 * (tokens // 3) + 40, tokens + 2000]
    paged = Paged(lens, kv_heads, dim, page, dtype, order, seed=tokens)
    before = paged.download()
    heads = q_heads + 2 * kv_heads
    x = rows_of(tokens, heads, dim, in_dtype, r, pad=4, scale=1.5)
    slots = r.integers(0, 3, tokens)
    index = np.array([r.permutation(lens[s])[0] for s in slots])
    # each place once: of tokens that drew the same place, only the first is appended
    first = np.array([not any(slots[j] == slots[i] and index[j] == index[i] for j in range(i)) for i in range(tokens)])
    index[~first] = -1
    pos = r.integers(0, 1 << 20, tokens)
    pos[0] = (1 << 31) - 1
    freq, scale = rope_frequencies(rot, 1e6, "yarn", 4.0, 32768) if rot else (None, 1.0)
    qn, kn = ((1 + 0.3 * r.standard_normal((2, dim))).astype(np.float32) if norm else (None, None))
    prep = KvPrep(device(qn), device(kn), 1e-6, device(freq), rot, interleaved, scale)
    raw, status = run(ctx, paged, q_heads, x, in_dtype, tokens, pos, slots, index, prep)
    assert (status == np.where(first, 0, _lib.VXS_ERR_ID_OUT_OF_RANGE)).all()

    w = on.widen(x)[:, :heads * dim].reshape(tokens, heads, dim)
    scale = float(np.float32(scale))
    y, mag = on.prep_heads(w[:, :q_heads], qn, float(np.float32(1e-6)), pos, freq, rot, interleaved, scale)
    got = on.widen(as_out(raw, dtype))[:, :q_heads * dim].reshape(y.shape)
    assert (np.abs(got - y) <= tolerance(y, mag, dim, norm, dtype)).all()
    y, mag = on.prep_heads(w[:, q_heads:q_heads + kv_heads], kn, float(np.float32(1e-6)), pos, freq, rot, interleaved, scale)
    k, v = paged.download()
    touched = np.zeros((paged.pages, page), bool)
    for t in np.nonzero(first)[0]:
        p, i = paged.table[slots[t], index[t] // page], index[t] % page
        touched[p, i] = True
        assert (np.abs(on.widen(np.ascontiguousarray(k[p, :, i])) - y[t]) <= tolerance(y[t], mag[t], dim, norm, dtype)).all()
        want = on.pack(w[t, q_heads + kv_heads:], dtype)
        assert np.array_equal(v[p, :, i].view(np.uint16), want.view(np.uint16))
    for now, then in ((k, before[0]), (v, before[1])):
        same = (now.view(np.uint16) == then.view(np.uint16)).all(axis=(1, 3))
        assert (same | touched).all(), "an entry outside the tokens' places changed"


def test_parts_and_defaults(ctx):
    """Queries alone, keys and values alone; slots by default the tokens' own, places by default the positions."""
    r = np.random.default_rng(0)
    paged = Paged([20, 40, 33], 2, 64, 16, "bf16", seed=1)
    x = rows_of(3, 8, 64, "f32", r)
    freq, _ = rope_frequencies(64)
    prep = KvPrep(None, None, 0.0, device(freq), 64)
    pos = [19, 0, 32]
    before = paged.download()
    whole, status = run(ctx, paged, 4, x, "f32", 3, pos, None, prep=prep)
    assert not status.any()
    k, v = paged.download()
    for t, p in enumerate(pos):
        assert np.array_equal(v[paged.table[t, p // 16], :, p % 16], on.pack(x[t, 384:512].reshape(2, 64), "bf16"))
    paged.upload()
    only_q, status = run(ctx, paged, 4, x, "f32", 3, pos, None, prep=prep, parts="q")
    assert np.array_equal(only_q, whole) and not status.any()
    assert all(np.array_equal(a, b) for a, b in zip(paged.download(), before))
    only_kv, _ = run(ctx, paged, 4, x, "f32", 3, pos, None, prep=prep, parts="kv", status=False)
    assert (only_kv == 7).all() and all(np.array_equal(a, b) for a, b in zip(paged.download(), (k, v)))
    # one norm alone, and no rotation without a prep
    norm = np.full(64, 2.0, np.float32)
    got, _ = run(ctx, paged, 4, x, "f32", 3, pos, None, prep=KvPrep(None, device(norm), 1e-6), parts="qkv")
    assert np.array_equal(got[:, :256], on.pack(x[:, :256], "bf16"))
    got, _ = run(ctx, paged, 4, x, "f32", 3, None, None, index=pos, parts="qkv")
    assert np.array_equal(got[:, :256], on.pack(x[:, :256], "bf16"))


def test_tokens_outside_the_cache(ctx):
    """A slot, place or page outside the cache: the status says so, nothing is written, the query is there."""
    r = np.random.default_rng(0)
    paged = Paged([20, 40, 33], 2, 64, 16, "bf16", seed=1, width=5)
    x = rows_of(7, 8, 64, "f32", r)
    slots, index = [0, 1, 3, -1, 0, 1, 2], [16, 80, 0, 0, -1, 60, 1 << 30]
    before = paged.download()
    q, status = run(ctx, paged, 4, x, "f32", 7, index, slots)
    assert status.tolist() == [0] + [_lib.VXS_ERR_ID_OUT_OF_RANGE] * 6
    k, v = paged.download()
    changed = (v.view(np.uint16) != before[1].view(np.uint16)).any(axis=(1, 3))
    assert changed.sum() == 1 and changed[paged.table[0, 1], 0]
    assert np.array_equal(q[:, :256], on.pack(x[:, :256], "bf16"))


def test_extreme_heads(ctx):
    """An all-zero head, a tiny one, one whose squares pass the fp16 range, and NaN, which stays its own."""
    paged = Paged([8], 1, 128, 16, "bf16", seed=1)
    x = np.zeros((4, 3 * 128), np.float32)
    x[1] = 1e-18
    x[2] = 1e4
    x[3, :128] = np.nan
    x[3, 128:] = 1.0
    w = device(np.ones(128, np.float32))
    raw, _ = run(ctx, paged, 1, x, "f32", 4, None, [0] * 4, index=[0, 1, 2, 3], prep=KvPrep(w, w, 1e-6))
    got = on.widen(raw)[:, :128]
    assert not got[0].any() and np.isnan(got[3]).all()
    assert np.allclose(got[1], 1e-15, rtol=2.0**-8) and np.allclose(got[2], 1.0, rtol=2.0**-8)
    k, _ = paged.download()
    assert np.allclose(on.widen(k[paged.table[0, 0], 0, 3:4]), 1.0, rtol=2.0**-8)


def test_refusals(ctx):
    paged = Paged([40, 20], 2, 64, 16, "bf16", seed=1)
    x = device(np.zeros(1 << 14, np.float32))
    i32 = device(np.zeros(64, np.int32))
    good = KvPrep(None, None, 0.0, x, 64)

    def call(tokens=2, q_heads=4, q=x, ldq=512, k=x, ldk=512, v=x, ldv=512, kind="f32", cache=None, pos=i32, out=x, ldo=256,
             prep=good, index=None):
        ctx.kv_append_device(tokens, q_heads, q, ldq, k, ldk, v, ldv, kind, cache or paged.cache, pos, i32, out, ldo, prep=prep, index=index)

    def refused(code, **kw):
        with pytest.raises(SamplerError) as e:
            call(**kw)
        assert e.value.code == code and ctx.last_error()

    bad, unsupported = _lib.VXS_ERR_INVALID_ARG, _lib.VXS_ERR_UNSUPPORTED
    for kw in ({"tokens": -1}, {"q_heads": 3}, {"q_heads": 0}, {"q": None, "k": None, "v": None}, {"v": None}, {"out": None}, {"pos": None},
               {"ldq": 252}, {"ldk": 124}, {"ldv": 124}, {"ldo": 252}, {"prep": KvPrep(None, None, 0.0, None, 64)},
               {"prep": KvPrep(None, None, 0.0, x, 66)}, {"prep": KvPrep(None, None, 0.0, x, -8)}, {"prep": KvPrep(None, None, 0.0, x, 7)},
               {"prep": KvPrep(x, None, -1.0)}, {"prep": KvPrep(None, x, float("nan"))}):
        refused(bad, **kw)
    for kw in ({"ldq": 514}, {"ldk": 514}, {"ldv": 513}, {"ldo": 258}, {"q": x.ptr + 4}, {"k": x.ptr + 8}, {"out": x.ptr + 4},
               {"prep": KvPrep(None, None, 0.0, x, 12)}, {"prep": KvPrep(None, None, 0.0, x.ptr + 4, 64)},
               {"cache": KvCache(paged.dk, paged.dv, "bf16", 2, 32, paged.pages, 16, paged.dtable, 2, paged.width)}):
        refused(unsupported, **kw)
    call(tokens=0)
    ctx.synchronize()


def test_too_many_tokens_are_refused(ctx):
    """A launch's threads are counted in 32 bits."""
    paged = Paged([40, 20], 2, 64, 16, "bf16", seed=1)
    x, i32 = device(np.zeros(1 << 14, np.float32)), device(np.zeros(64, np.int32))
    with pytest.raises(SamplerError) as e:
        ctx.kv_append_device(1 << 24, 4, x, 256, None, 0, None, 0, "f32", paged.cache, i32, i32, x, 256)
    assert e.value.code == _lib.VXS_ERR_UNSUPPORTED and ctx.last_error()
