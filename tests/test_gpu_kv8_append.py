"""GPU checks of vxs_kv8_append_device and of positions of several axes against the 64-bit oracle: blocks that begin, go on and grow,
norms, rotations, types, pages and layouts, tokens outside the cache, rows in any order within a block, refusals."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import attention8_np as o8
from oracle import attention_np as on
from voxwerk_amd import _lib, hip
from voxwerk_amd.attention import KvPrep, RopeAxes, rope_axes, rope_frequencies
from voxwerk_amd.sampler import SamplerError

from attention_cases import Paged, as_out, device, out_array, rows_of
from attention8_cases import Paged8

pytestmark = pytest.mark.gpu

# (q_heads, kv_heads, dim, rot, interleaved, norm, axes, in, dtype, page, order)
SHAPES = [
    (16, 8, 128, 128, False, True, 1, "f32", "bf16", 16, "heads"),
    (16, 8, 128, 128, True, True, 3, "bf16", "bf16", 16, "tokens"),
    (5, 1, 64, 64, False, False, 2, "f32", "f16", 32, "heads"),
    (4, 4, 64, 32, False, True, 1, "f16", "f16", 64, "tokens"),
    (4, 2, 64, 8, True, True, 3, "bf16", "f16", 16, "heads"),
    (2, 2, 256, 256, False, True, 3, "f32", "bf16", 16, "heads"),
    (6, 3, 256, 96, False, False, 1, "bf16", "bf16", 128, "tokens"),
    (3, 1, 256, 64, True, True, 4, "f16", "bf16", 16, "heads"),
    (2, 1, 128, 0, False, True, 1, "f32", "f16", 16, "heads"),
    (2, 1, 128, 0, False, False, 1, "f32", "bf16", 32, "heads"),
    (40, 8, 128, 64, True, False, 3, "f32", "bf16", 16, "heads"),
]


def computed_within(y, mag, dim, normed):
    """An angle is off by 2^-24 of a turn and the fp32 sine and cosine by 2^-18, so a rotated entry by 2^-17 of |a| + |b|; the
    norm's sum of dim squares, root, division and products by (dim + 8) 2^-24."""
    rel = (dim + 8) * 2.0**-24 if normed else 2.0**-23
    return np.abs(y) * rel + mag * (2.0**-17 + rel)


def run(ctx, paged, q_heads, x, in_dtype, tokens, pos, slots, index=None, prep=None, parts="qkv", status=True, axis=None):
    """x [tokens, (q + 2 kv) heads * dim + pad]; returns q_out and the status."""
    d, kh, ld = paged.dim, paged.kv_heads, x.shape[1]
    dx = device(x)
    size = x.itemsize
    q = dx.ptr if "q" in parts else None
    k, v = (dx.ptr + size * q_heads * d, dx.ptr + size * (q_heads + kh) * d) if "k" in parts else (None, None)
    out, st = out_array(tokens, q_heads * d + 4, paged.dtype), device(np.full(tokens, 9, np.int32)) if status else None
    keep = [None if a is None else device(np.array(a, np.int32)) for a in (pos, slots, index)]
    axes = None if axis is None else RopeAxes(device(axis), len(pos), np.shape(pos)[1])
    hip.synchronize()
    ctx.kv_append_device(tokens, q_heads, q, ld, k, ld, v, ld, in_dtype, paged.cache, keep[0], keep[1], out, q_heads * d + 4,
                         prep=prep, index=keep[2], status=st, axes=axes)
    ctx.synchronize()
    raw = out.numpy()
    assert (raw[:, q_heads * d:] == 7).all(), "the pad was written"
    return raw, st.numpy() if status else None


def turned(x, weight, eps, pos, axis, freq, rot, interleaved, scale):
    """on.prep_heads with a position for each frequency: pos [axes, tokens]."""
    if axis is None or not rot:
        return on.prep_heads(x, weight, eps, pos if pos is None or np.ndim(pos) == 1 else pos[0], freq, rot, interleaved, scale)
    y = mag = None
    for a in range(len(pos)):  # the pairs of one axis from a rotation by its positions
        z, m = on.prep_heads(x, weight, eps, pos[a], freq, rot, interleaved, scale)
        mine = np.zeros(x.shape[-1], bool)
        i = np.nonzero(axis == a)[0]
        mine[2 * i if interleaved else i] = True
        mine[2 * i + 1 if interleaved else i + rot // 2] = True
        if y is None:
            y, mag = z, m
        y[..., mine], mag[..., mine] = z[..., mine], m[..., mine]
    return y, mag


def check_store(paged, before, pages, inside, x, err, h, which):
    """Keys (which 0) or values (1) of head h after tokens x went to (pages, inside); `before`: download() then."""
    now, now_s = paged.after[which][:, h], paged.after[2 + which][:, h].astype(int)
    then, then_s = before[which][:, h], before[2 + which][:, h].astype(int)
    found = o8.append(then, then_s, list(zip(pages, inside)), x, err)
    touched = np.zeros(now_s.shape, bool)
    for (p, b), (low, high, rows) in found.items():
        touched[p, b] = True
        byte = now_s[p, b]
        assert low <= byte <= high, f"scale {byte} of page {p}, block {b}: {low} to {high}"
        at = slice(b * o8.BLOCK, (b + 1) * o8.BLOCK)
        new = rows >= 0
        y, e = np.asarray(x)[rows[new]], np.broadcast_to(err, np.shape(x))[rows[new]]
        got = o8.VALUES[now[p, at][new]] * o8.power(byte)
        odd = ~np.isfinite(y)
        assert np.isnan(got[odd]).all()
        with np.errstate(invalid="ignore"):
            half = np.maximum(2.0**-4 * (np.abs(y) + e), 2.0**-10 * o8.power(byte))
            assert (np.abs(got - y) <= half + e)[~odd].all()
        if not np.any(err):
            assert np.array_equal(now[p, at][new] & np.where(odd, 0x7F, 0xFF), np.where(odd, 0x7F, o8.encode(y / o8.power(byte))))
        old, want = then[p, at][~new], then[p, at][~new]
        if rows[0] < 0 and byte != then_s[p, b]:
            want = o8.encode(o8.VALUES[old] * 2.0 ** (then_s[p, b] - byte))
            want = np.where(np.isnan(o8.VALUES[old]), now[p, at][~new], want)  # (one NaN or the other)
            assert (np.isnan(o8.VALUES[want]) == np.isnan(o8.VALUES[old])).all()
        assert np.array_equal(now[p, at][~new], want), "an entry beside the call's tokens"
    assert np.array_equal(now_s[~touched], then_s[~touched]), "a scale of another block changed"
    same = (now == then).all(-1).reshape(now.shape[0], -1, o8.BLOCK).all(-1)
    assert (same | touched).all(), "another block changed"
    return len(found)


def packed_tokens(paged, new, r, order=None):
    """Rows of new[s] tokens that end at paged.lens[s], sequence after sequence."""
    slots = np.repeat(np.arange(len(new)), new)
    index = np.concatenate([np.arange(paged.lens[s] - n, paged.lens[s]) for s, n in enumerate(new)]).astype(int)
    return slots, index


def check_call(ctx, paged, q_heads, slots, index, in_dtype, rot=0, interleaved=False, norm=False, axes=1, scale=1.5, x=None, valid=None):
    r, d, kh, tokens = paged.rng, paged.dim, paged.kv_heads, len(slots)
    heads = q_heads + 2 * kh
    if x is None:
        x = rows_of(tokens, heads, d, in_dtype, r, pad=4, scale=scale)
    valid = np.ones(tokens, bool) if valid is None else valid
    pos = r.integers(0, 1 << 20, (axes, tokens))
    pos[0, 0] = (1 << 31) - 1
    axis = None if axes == 1 else r.integers(0, axes, max(rot // 2, 1)).astype(np.int32)
    freq, rs = rope_frequencies(rot, 1e6, "yarn", 4.0, 32768) if rot else (None, 1.0)
    qn, kn = ((1 + 0.3 * r.standard_normal((2, d))).astype(np.float32) if norm else (None, None))
    prep = KvPrep(device(qn), device(kn), 1e-6, device(freq), rot, interleaved, rs)
    before = paged.download()
    raw, status = run(ctx, paged, q_heads, x, in_dtype, tokens, pos if axes > 1 else pos[0], slots, index, prep, axis=axis)
    assert (status == np.where(valid, 0, _lib.VXS_ERR_ID_OUT_OF_RANGE)).all()
    w = on.widen(x)[:, :heads * d].reshape(tokens, heads, d)
    rs, eps = float(np.float32(rs)), float(np.float32(1e-6))
    y, mag = turned(w[:, :q_heads], qn, eps, pos, axis, freq, rot, interleaved, rs)
    got = on.widen(as_out(raw, paged.dtype))[:, :q_heads * d].reshape(y.shape)
    tol = computed_within(y, mag, d, norm) + np.abs(y) * on.UNIT[paged.dtype] + (2.0**-24 if paged.dtype == "f16" else 2.0**-133)
    with np.errstate(invalid="ignore"):
        assert (np.abs(got - y) <= tol)[np.isfinite(y)].all()
    y, mag = turned(w[:, q_heads:q_heads + kh], kn, eps, pos, axis, freq, rot, interleaved, rs)
    paged.after = paged.download()
    at = np.nonzero(valid)[0]
    pages, inside = paged.table[np.array(slots)[at], np.array(index)[at] // paged.page], np.array(index)[at] % paged.page
    plain = not norm and not rot
    for h in range(kh):
        err = 0.0 if plain else computed_within(y[at, h], mag[at, h], d, norm)
        check_store(paged, before, pages, inside, y[at, h], err, h, 0)
        check_store(paged, before, pages, inside, w[at, q_heads + kh + h], 0.0, h, 1)


@pytest.mark.parametrize("lens,new", [([37], [1]), ([16, 17, 300, 1], [1, 1, 1, 1]), ([5, 40, 333], [3, 33, 300]), ([1200, 70], [1150, 20])])
@pytest.mark.parametrize("q_heads,kv_heads,dim,rot,interleaved,norm,axes,in_dtype,dtype,page,order", SHAPES)
def test_append(ctx, q_heads, kv_heads, dim, rot, interleaved, norm, axes, in_dtype, dtype, page, order, lens, new):
    """One token, one of each sequence, pieces that begin and end within blocks, and enough rows that waves share 16 of them."""
    paged = Paged8(lens, kv_heads, dim, page, dtype, order, seed=dim + rot + len(new))
    slots, index = packed_tokens(paged, new, paged.rng)
    check_call(ctx, paged, q_heads, slots, index, in_dtype, rot, interleaved, norm, axes)


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 1.0, 300.0, 1e30])
def test_scales_of_all_sizes(ctx, scale):
    """Blocks that stay, grow by a little and by far; what was there falls below the new steps in the end."""
    paged = Paged8([40, 23, 300], 2, 64, 16, "bf16", seed=3)
    slots, index = packed_tokens(paged, [10, 1, 30], paged.rng)
    check_call(ctx, paged, 4, slots, index, "f32", scale=scale)


def test_token_by_token(ctx):
    """A sequence that comes token by token ends with the scales of one that comes whole, and entries that differ where they were
    rounded below the scales' steps on the way only; each step of the way is checked."""
    n, d = 50, 64
    whole, steps = Paged8([n], 2, d, 16, "bf16", seed=1), Paged8([n], 2, d, 16, "bf16", seed=1)
    x = rows_of(n, 6, d, "f32", np.random.default_rng(2), pad=4)
    x[:, :6 * d] *= np.geomspace(0.01, 100, n, dtype=np.float32)[:, None]  # (each token needs a larger scale)
    run(ctx, whole, 2, x, "f32", n, None, [0] * n, np.arange(n))
    for t in range(n):
        check_call(ctx, steps, 2, [0], [t], "f32", x=x[t:t + 1])
    a, b = whole.download(), steps.download()
    used = whole.table[0, :4]
    for i in (2, 3):
        assert np.array_equal(a[i][used], b[i][used])
        scale = o8.power(a[i][used])  # [pages, heads, 1]
        k, s = (o8.VALUES[z[i - 2][used]] * scale[..., None] for z in (a, b))
        there = np.arange(4)[:, None] * 16 + np.arange(16) < n
        off = np.abs(k - s).transpose(0, 2, 1, 3)[there]
        # An entry that ends below 2^-6 of the scale S is a multiple of 2^-9 S. Coming whole it is rounded once, by 2^-10 S; on the way by
        # 2^-11 S first (4 bits of less than 2^-6 S), by 2^-10 of each smaller scale, together 2^-10 S, and by 2^-10 S in the end: less than two
        # steps apart, so at most one. Others are the same.
        assert (off <= (2.0**-9 * scale)[:, None].repeat(16, 1)[there]).all()


def test_rows_in_any_order_within_a_block(ctx):
    """Rows of one block in any order, some places twice (the later row stays), more rows than a wave has lanes."""
    for tokens in (40, 150, 1100):
        paged = Paged8([64, 64, 64], 2, 64, 16, "bf16", seed=tokens)
        r = paged.rng
        slots, index = [], []
        for i, n in enumerate(np.diff(np.concatenate([[0], np.sort(r.choice(tokens - 1, 10, replace=False)) + 1, [tokens]]))):
            slots += [i % 3] * n
            index += (16 * (i // 3) + r.integers(0, 16, n)).tolist()
        check_call(ctx, paged, 2, slots, index, "f32", 64, norm=True)


def test_tokens_outside_the_cache(ctx):
    """A slot, place or page outside the cache: the status says so, nothing is written, the query is there."""
    paged = Paged8([20, 40, 33], 2, 64, 16, "bf16", seed=1, width=5)
    slots, index = [0, 1, 3, -1, 0, 1, 2, 2], [16, 80, 0, 0, -1, 60, 1 << 30, 5]
    valid = np.array([True] + [False] * 6 + [True])
    check_call(ctx, paged, 4, slots, index, "f32", valid=valid)


def test_parts_and_defaults(ctx):
    """Queries alone, keys and values alone; slots by default the tokens' own, places by default the positions."""
    paged = Paged8([20, 40, 33], 2, 64, 16, "bf16", seed=1)
    x = rows_of(3, 8, 64, "f32", paged.rng)
    freq, _ = rope_frequencies(64)
    prep = KvPrep(None, None, 0.0, device(freq), 64)
    pos = [19, 0, 32]
    before = paged.download()
    whole, status = run(ctx, paged, 4, x, "f32", 3, pos, None, prep=prep)
    assert not status.any()
    after = paged.download()
    assert not all(np.array_equal(a, b) for a, b in zip(after, before))
    paged.upload()
    only_q, status = run(ctx, paged, 4, x, "f32", 3, pos, None, prep=prep, parts="q")
    assert np.array_equal(only_q, whole) and not status.any()
    assert all(np.array_equal(a, b) for a, b in zip(paged.download(), before))
    only_kv, _ = run(ctx, paged, 4, x, "f32", 3, pos, None, prep=prep, parts="kv", status=False)
    assert (only_kv == 7).all() and all(np.array_equal(a, b) for a, b in zip(paged.download(), after))


def test_infinite_and_nan(ctx):
    """They are NaN entries, and the scale is that of the finite ones; a block of nothing else has the least scale."""
    paged = Paged8([48], 1, 64, 16, "bf16", seed=1)
    x = rows_of(33, 3, 64, "f32", paged.rng, pad=4)
    x[5, 70:90], x[6, 140] = np.inf, -np.inf
    x[7, 100], x[8, 130] = np.nan, 3e38
    x[16:32, :192] = np.nan
    x[32, :192] = 0.0
    check_call(ctx, paged, 1, [0] * 33, np.arange(33), "f32", x=x)
    p = paged.table[0]
    assert paged.after[2][p[1], 0, 0] == 1 and paged.after[2][p[2], 0, 0] == 1 and paged.after[3][p[0], 0, 0] == o8.byte_for(float(np.float32(3e38)))


# ---- axes over a 16-bit cache -----------------------------------------------------------------------


@pytest.mark.parametrize("tokens", [1, 3, 300, 2051])
@pytest.mark.parametrize("q_heads,kv_heads,dim,rot,interleaved,norm,axes,in_dtype,dtype,page,order", [s for s in SHAPES if s[6] > 1])
def test_axes_16(ctx, q_heads, kv_heads, dim, rot, interleaved, norm, axes, in_dtype, dtype, page, order, tokens):
    r = np.random.default_rng(dim + tokens)
    paged = Paged([tokens + 40], kv_heads, dim, page, dtype, order, seed=tokens)
    heads = q_heads + 2 * kv_heads
    x = rows_of(tokens, heads, dim, in_dtype, r, pad=4, scale=1.5)
    index = 40 + np.arange(tokens)
    pos = r.integers(-5, 1 << 20, (axes, tokens + 7))  # (rows of positions longer than the call)
    axis = r.integers(0, axes, rot // 2).astype(np.int32)
    freq, rs = rope_frequencies(rot, 1e4)
    qn, kn = ((1 + 0.3 * r.standard_normal((2, dim))).astype(np.float32) if norm else (None, None))
    raw, status = run(ctx, paged, q_heads, x, in_dtype, tokens, pos, [0] * tokens, index, KvPrep(device(qn), device(kn), 1e-6, device(freq), rot, interleaved), axis=axis)
    assert not status.any()
    w = on.widen(x)[:, :heads * dim].reshape(tokens, heads, dim)
    eps, least = float(np.float32(1e-6)), 2.0**-24 if dtype == "f16" else 2.0**-133
    k, v = paged.download()
    for got, part, weight in ((on.widen(as_out(raw, dtype))[:, :q_heads * dim].reshape(tokens, q_heads, dim), w[:, :q_heads], qn),
                              (on.widen(np.ascontiguousarray(k[paged.table[0, index // page], :, index % page])), w[:, q_heads:q_heads + kv_heads], kn)):
        y, mag = turned(part, weight, eps, pos[:, :tokens], axis, freq, rot, interleaved, rs)
        assert (np.abs(got - y) <= computed_within(y, mag, dim, norm) + np.abs(y) * on.UNIT[dtype] + least).all()
    assert np.array_equal(v[paged.table[0, index // page], :, index % page].view(np.uint16), on.pack(w[:, q_heads + kv_heads:], dtype).view(np.uint16))


def test_axes_that_agree_are_one(ctx):
    """The same position on every axis is a position, bit for bit; an axis outside counts as the nearest."""
    paged = Paged([40], 2, 64, 16, "bf16", seed=1)
    x = rows_of(9, 8, 64, "f32", paged.rng)
    freq, _ = rope_frequencies(64)
    prep = KvPrep(None, None, 0.0, device(freq), 64)
    pos = paged.rng.integers(0, 5000, 9)
    one, _ = run(ctx, paged, 4, x, "f32", 9, pos, [0] * 9, np.arange(9), prep)
    k = paged.download()
    for axis in (rope_axes([12, 10, 10]), rope_axes([12, 10, 10], True), np.full(32, -3, np.int32), np.full(32, 99, np.int32)):
        paged.upload()
        many, _ = run(ctx, paged, 4, x, "f32", 9, np.stack([pos] * 3), [0] * 9, np.arange(9), prep, axis=axis)
        assert np.array_equal(one, many) and all(np.array_equal(a.view(np.uint16), b.view(np.uint16)) for a, b in zip(k, paged.download()))
    a, _ = run(ctx, paged, 4, x, "f32", 9, np.stack([pos, pos + 9, pos + 5]), [0] * 9, np.arange(9), prep, axis=np.full(32, 99, np.int32))
    b, _ = run(ctx, paged, 4, x, "f32", 9, pos + 5, [0] * 9, np.arange(9), prep)
    assert np.array_equal(a, b)


def test_refused_calls_launch_nothing(ctx):
    """(tests/test_attention8_host.py has the whole list, without a GPU.)"""
    paged = Paged8([40, 20], 2, 64, 16, "bf16", seed=1)
    x, i32 = device(np.zeros(1 << 14, np.float32)), device(np.zeros(64, np.int32))
    before = paged.download()
    for kw in ({"axes": RopeAxes(i32, 0, 64), "index": i32}, {"axes": RopeAxes(i32, 3, 64)}, {"axes": RopeAxes(i32, 3, 1), "index": i32}):
        with pytest.raises(SamplerError) as e:
            ctx.kv_append_device(2, 4, x, 512, x, 512, x, 512, "f32", paged.cache, i32, i32, x, 256, prep=KvPrep(None, None, 0.0, x, 64), **kw)
        assert e.value.code == _lib.VXS_ERR_INVALID_ARG and ctx.last_error()
    ctx.synchronize()
    assert all(np.array_equal(a, b) for a, b in zip(before, paged.download()))
