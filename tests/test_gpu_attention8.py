"""GPU checks of attention over an 8-bit paged cache against the 64-bit oracle: lengths around every tile edge, head groups,
types, page sizes, layouts, shared prefixes, scales, what unseen places hold; and of cross attention over both kinds of cache.

Every entry that no row may read is NaN or the largest, every scale of a block outside the sequences 0, 254 or 255."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from oracle import attention8_np as o8
from oracle import attention_np as on
from voxwerk_amd import _lib, hip
from voxwerk_amd.attention import Kv8Cache, SharedPrefix
from voxwerk_amd.sampler import Context, SamplerError

import attention_cases
from attention_cases import Paged, device, out_array, rows_of, run_prompt, run_step
from attention8_cases import Paged8, check, run_cross

pytestmark = pytest.mark.gpu

EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 700, 1025]
# (q_heads, kv_heads, dim, page, dtype, out, order)
SHAPES = [
    (16, 8, 128, 16, "bf16", "bf16", "heads"),
    (16, 8, 128, 64, "f16", "f32", "tokens"),
    (4, 4, 64, 32, "bf16", "f32", "heads"),
    (6, 2, 128, 16, "f16", "f16", "tokens"),
    (14, 2, 64, 128, "f16", "f16", "heads"),
    (16, 1, 256, 16, "bf16", "bf16", "heads"),
    (20, 1, 64, 16, "bf16", "f32", "tokens"),
    (33, 1, 128, 32, "bf16", "bf16", "heads"),
    (80, 1, 64, 16, "f16", "f32", "heads"),
    (2, 2, 256, 256, "f16", "f32", "tokens"),
    (8, 1, 128, 16, "bf16", "f32", "heads"),
    (3, 3, 256, 64, "f16", "f16", "heads"),
]


def checked(paged, *args, **kw):
    """check() of attention8_cases for an 8-bit cache, of attention_cases for a 16-bit one."""
    if isinstance(paged, Paged8):
        return check(*args, **kw)
    *head, out_dtype, what = args
    return attention_cases.check(*head, paged.dtype, out_dtype, what)


def step_and_check(ctx, paged, q_heads, out, share=(), scale=None, q_scale=2.0, what="step", kv_len=None, slots=None, **kw):
    lens = paged.lens if kv_len is None else kv_len
    rows = len(lens)
    scale = scale or paged.dim**-0.5
    q = rows_of(rows, q_heads, paged.dim, paged.dtype, paged.rng, pad=8, scale=q_scale)
    got = run_step(ctx, paged, q, q_heads, scale, out, share=share, kv_len=kv_len, slots=slots, ldo_pad=8, **kw)
    slot = lambda r: r if slots is None else slots[r]  # noqa: E731
    cap = paged.width * paged.page
    seen = [min(n, cap) if 0 <= slot(r) < len(paged.lens) else 0 for r, n in enumerate(lens)]
    checked(paged, got, q, seen, lambda r, h: paged.entries(slot(r) if seen[r] > 0 else 0, max(seen[r], 0), h), q_heads, paged.kv_heads,
            paged.dim, scale, out, what)
    assert (got.view(np.uint16 if out != "f32" else np.float32)[:, q_heads * paged.dim:] == 7).all(), "the pad was written"
    return q, got


@pytest.mark.parametrize("q_heads,kv_heads,dim,page,dtype,out,order", SHAPES)
def test_step_lengths(ctx, q_heads, kv_heads, dim, page, dtype, out, order):
    paged = Paged8(EDGES, kv_heads, dim, page, dtype, order, seed=dim + q_heads)
    step_and_check(ctx, paged, q_heads, out)


@pytest.mark.parametrize("q_heads,kv_heads,dim,page,dtype,out,order", SHAPES)
def test_step_one_long_row(ctx, q_heads, kv_heads, dim, page, dtype, out, order):
    """Few rows: a row's keys are divided among many workgroups, with and without the workspace for it."""
    paged = Paged8([3001], kv_heads, dim, page, dtype, order, seed=dim + q_heads)
    step_and_check(ctx, paged, q_heads, out)
    step_and_check(ctx, paged, q_heads, out, work=None, what="no workspace")


@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("page,prefix", [(16, 16), (16, 500), (64, 70), (32, 1), (16, 1030)])
def test_step_shared_prefix(ctx, rows, page, prefix):
    r = np.random.default_rng(rows + prefix)
    for q_heads, kv_heads, dim, dtype, out in ((16, 8, 128, "bf16", "bf16"), (7, 1, 64, "f16", "f32"), (4, 4, 256, "bf16", "f32")):
        lens = (prefix + r.integers(1, 200, rows)).tolist()
        share = [(0, rows, prefix)]
        paged = Paged8(lens, kv_heads, dim, page, dtype, "heads", seed=rows, share=share)
        step_and_check(ctx, paged, q_heads, out, share=share, what=f"prefix {prefix}")


def test_step_groups(ctx):
    """Several groups of different prefixes, rows outside every group, groups of one row and of none."""
    share = [(2, 7, 130), (7, 8, 64), (8, 8, 40), (8, 45, 333)]
    lens = [9, 200] + [130 + 11 * i for i in range(1, 6)] + [100] + [334 + 7 * i for i in range(37)] + [0, 77]
    for q_heads, kv_heads, dim, dtype, out in ((16, 8, 128, "bf16", "f32"), (32, 4, 64, "f16", "f16"), (40, 1, 128, "bf16", "bf16")):
        paged = Paged8(lens, kv_heads, dim, 16, dtype, "tokens", seed=3, share=share)
        step_and_check(ctx, paged, q_heads, out, share=share)


@pytest.mark.parametrize("rows,prefix", [(6, 90), (100, 2000)])
def test_step_shares_where_it_is_faster(ctx, rows, prefix):
    """Without the flag a prefix is shared from some size on; either way the outputs are the rows' own."""
    share = [(0, rows, prefix)]
    paged = Paged8([prefix + 1 + i % 37 for i in range(rows)], 2, 128, 16, "bf16", seed=rows, share=share)
    step_and_check(ctx, paged, 4, "f32", share=share, always=False)


def test_step_shorter_than_the_prefix(ctx):
    """A row that ends inside its group's prefix sees its own length only; keys past it may hold anything."""
    share = [(0, 6, 100)]
    paged = Paged8([160, 300, 101, 100, 140, 120], 2, 128, 16, "bf16", seed=5, share=share)
    lens = [160, 33, 101, 100, 0, 64]
    step_and_check(ctx, paged, 8, "f32", share=share, kv_len=lens)
    p = paged.table[0, 70 // 16]
    paged.v[p, :, 70 % 16, 5] = 0x7F
    paged.upload()
    q = rows_of(6, 8, 128, "bf16", paged.rng)
    got = run_step(ctx, paged, q, 8, 128**-0.5, "f32", kv_len=lens, share=share).reshape(6, 8, 128)
    assert np.isnan(got[[0, 2, 3], :, 5]).all() and np.isfinite(got[[1, 4, 5]]).all()
    assert np.isfinite(np.delete(got, 5, axis=2)).all()
    keep = [1, 4, 5]
    check(got.reshape(6, -1)[keep], q[keep], [lens[i] for i in keep], lambda r, h: paged.entries(keep[r], lens[keep[r]], h), 8, 2,
          128, 128**-0.5, "f32", "rows that do not see it")


def test_step_slots_and_lengths_outside(ctx):
    """Slots in any order; a slot outside the cache has no keys, a length above the table's is cut to it."""
    paged = Paged8([64, 50, 128, 20], 4, 64, 16, "bf16", seed=1)
    step_and_check(ctx, paged, 8, "f32", kv_len=[50, 20, 128, 10, 30, 5], slots=[1, 3, 2, -1, 4, 0], max_len=128)
    step_and_check(ctx, paged, 8, "f32", kv_len=[1 << 30, -5], slots=[2, 0], max_len=16)


def test_pages_outside_the_pool(ctx):
    """A page number outside the pool (a caller's mistake) reads some page of it, and that page's scales."""
    paged = Paged8([200, 40], 2, 128, 32, "bf16", seed=1)
    paged.k[:], paged.v[:], paged.ks[:], paged.vs[:] = 0x38, 0x38, 127, 127  # (ones everywhere)
    for bad in (-1, paged.pages, 1 << 30, -(1 << 31)):
        paged.table[0, 3] = bad
        paged.upload()
        q = rows_of(2, 4, 128, "bf16", paged.rng)
        assert np.allclose(run_step(ctx, paged, q, 4, 0.1, "f32"), 1.0, rtol=1e-5)
        q = rows_of(60, 4, 128, "bf16", paged.rng)
        assert np.allclose(run_prompt(ctx, paged, q, [0, 30, 60], 4, 0.1, "f32"), 1.0, rtol=1e-5)


@pytest.mark.parametrize("max_len", [0, 1, 100, 5000])
def test_step_longer_than_announced(ctx, max_len):
    """max_len only divides the work."""
    paged = Paged8([700, 3, 0, 260], 2, 128, 16, "bf16", seed=2)
    step_and_check(ctx, paged, 4, "f32", max_len=max_len)


def test_step_many_short_rows(ctx):
    """More (row, key head)s than fit at once, a wave each."""
    r = np.random.default_rng(1)
    for dim, dtype, out in ((128, "bf16", "bf16"), (64, "f16", "f32"), (256, "bf16", "f32")):
        paged = Paged8(r.integers(0, 257, 140).tolist(), 4, dim, 16, dtype, seed=dim)
        step_and_check(ctx, paged, 8, out)


def test_step_sharp_and_flat_scores(ctx):
    """One key with nearly all the weight, wherever it lies; equal scores; scores that grow along the keys, blocks' scales with them."""
    for at in (0, 31, 64, 450, 699):
        paged = Paged8([700], 1, 64, 16, "bf16", seed=at)
        p, i = paged.table[0, at // 16], at % 16
        paged.k[p, 0, i] = o8.encode(np.full(64, 3.0 / float(o8.power(paged.ks[p, 0, 0]))).clip(-448, 448))
        paged.upload()
        q = np.full((1, 4 * 64), 0x4040, np.uint16)  # 3.0
        got = run_step(ctx, paged, q, 4, 0.125, "f32")
        check(got, q, [700], lambda r, h: paged.entries(0, 700, h), 4, 1, 64, 0.125, "f32", f"sharp at {at}")
    for grow in (0, 1, -1):
        paged = Paged8([700], 1, 64, 16, "f16", seed=7)
        b = np.arange(44)
        paged.ks[paged.table[0], 0, 0] = 110 + (grow * b) // 4 + (11 if grow < 0 else 0)
        paged.upload()
        q = rows_of(1, 2, 64, "f16", paged.rng)
        got = run_step(ctx, paged, q, 2, 1.0, "f32")
        check(got, q, [700], lambda r, h: paged.entries(0, 700, h), 2, 1, 64, 1.0, "f32", f"grows by {grow}")


@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32")])
def test_scales_far_apart(ctx, dtype, out):
    """Blocks whose scales are at both ends of what the products can hold, next to each other: values from 2^-100 to 2^100, keys tiny."""
    paged = Paged8([300], 2, 64, 16, dtype, seed=3)
    b = np.arange(19)
    paged.vs[paged.table[0, b], :, 0] = np.where(b[:, None] % 3 == 0, 27, np.where(b[:, None] % 3 == 1, 121, 217))
    paged.ks[paged.table[0, b], :, 0] = np.where(b[:, None] % 2 == 0, 20, 121)
    paged.upload()
    q = rows_of(3, 4, 64, dtype, paged.rng)
    lens = [300, 16, 140]
    got = run_step(ctx, paged, q, 4, 0.125, out, kv_len=lens, slots=[0, 0, 0])
    check(got, q, lens, lambda r, h: paged.entries(0, lens[r], h), 4, 2, 64, 0.125, out, "scales far apart")
    got = run_prompt(ctx, paged, rows_of(300, 4, 64, dtype, paged.rng), [0, 300], 4, 0.125, out)
    assert np.isfinite(on.widen(got)).all()


def test_every_entry(ctx):
    """Each of the 254 numbers that a byte can be, as the only value that a row sees, at several scales. Its weight is kept to 24 bits,
    its products' sums, the reciprocal of the weight and the last product are rounded: eight times 2^-24 at most. The weight is 2^-8 when the
    maximum has just been set, so a value's products lie below fp32's normal range 2^-126 where it is below 2^-118 (byte 12): there a sum
    has no bits that it has to keep, three products and the sum are off by 2^-126 each at most, and the output by 2^8 times that."""
    numbers = [b for b in range(256) if b & 127 != 127]
    for byte in (127, 121, 12, 240):
        paged = Paged8([1] * 4, 1, 64, 16, "bf16", seed=byte)
        codes = np.array(numbers + [0] * 2, np.uint8).reshape(4, 64)
        for s in range(4):
            paged.v[paged.table[s, 0], 0, 0] = codes[s]
            paged.vs[paged.table[s, 0], 0, 0] = byte
        paged.upload()
        got = run_step(ctx, paged, rows_of(4, 1, 64, "bf16", paged.rng), 1, 0.125, "f32")
        want = o8.VALUES[codes] * o8.power(byte)
        assert (np.abs(got - want) <= 2.0**-21 * np.abs(want) + 2.0**-116).all()


def test_step_nonfinite_that_is_seen(ctx):
    """A NaN key or a NaN value that a row sees makes its outputs NaN, as the formula says; other rows are as ever."""
    paged = Paged8([100, 100, 100], 1, 64, 16, "bf16", seed=11)
    paged.k[paged.table[0, 2], 0, 3, 9] = 0x7F
    paged.v[paged.table[1, 2], 0, 3, 9] = 0xFF
    paged.upload()
    q = rows_of(3, 2, 64, "bf16", paged.rng)
    got = run_step(ctx, paged, q, 2, 0.125, "f32").reshape(3, 2, 64)
    assert np.isnan(got[0]).all() and np.isnan(got[1, :, 9]).all() and np.isfinite(np.delete(got[1], 9, axis=1)).all()
    check(got.reshape(3, -1)[2:], q[2:], [100], lambda r, h: paged.entries(2, 100, h), 2, 1, 64, 0.125, "f32", "beside NaN")


def test_workspace_serves_both_kinds_of_cache(ctx):
    """One workspace, zeroed once, between steps over 16-bit and 8-bit caches of other sizes: each is right."""
    share = [(0, 24, 500)]
    calls = [
        (Paged8([2900, 1500], 2, 128, 16, seed=1), 8, ()),
        (Paged([700] * 24, 2, 128, 16, seed=2), 8, ()),
        (Paged8([2600], 1, 64, 16, "f16", seed=3), 5, ()),
        (Paged8([700] * 24, 2, 128, 16, seed=4, share=share), 8, share),
        (Paged([900, 300, 0, 1700, 65], 2, 256, 32, "f16", seed=5), 2, ()),
        (Paged8([600] * 40, 3, 64, 16, seed=6), 12, ()),
        (Paged8([900, 300, 0, 1700, 65], 2, 256, 32, "bf16", seed=5), 2, ()),
    ]
    n = max(ctx.attn_step_workspace(len(p.lens), h, p.cache, max(p.lens), SharedPrefix(1, 16, 16, 500, True) if s else None) for p, h, s in calls)
    work = device(np.zeros(n, np.uint8))
    first = {}
    for _ in range(2):
        for i, (p, h, s) in enumerate(calls):
            p.rng = np.random.default_rng(i)
            _, got = step_and_check(ctx, p, h, "f32", share=s, work=work, what=f"call {i}")
            assert np.array_equal(first.setdefault(i, got).view(np.uint32), got.view(np.uint32)), "not the same bits again"


def test_workspace_of_larger_sizes_is_enough(ctx):
    paged = Paged8([1800] * 24, 2, 128, 16, seed=7)
    for prefix in (None, SharedPrefix(1, 16, 16, 900, True)):
        n = ctx.attn_step_workspace(24, 8, paged.cache, 1800, prefix)
        for rows in range(25):
            for most in (0, 1, 256, 257, 700, 1800):
                assert ctx.attn_step_workspace(rows, 8, paged.cache, most, prefix) <= n
                assert ctx.attn_step_workspace(rows, 8, paged.cache, most) <= n
    work = device(np.zeros(ctx.attn_step_workspace(24, 8, paged.cache, 1800), np.uint8))
    for rows in (24, 1, 5, 24, 13):
        few = Paged8([1800] * rows, 2, 128, 16, seed=rows)
        step_and_check(ctx, few, 8, "f32", work=work, what=f"{rows} rows")


# ---- prompts ---------------------------------------------------------------------------------------


def packed_and_check(ctx, paged, new, q_heads, out, kv_len=None, slots=None, q_scale=2.0, lead=0, tail=0, cross=False, what="packed"):
    """new[i] tokens of sequence i; `lead` and `tail` rows of the queries belong to no sequence."""
    lens = paged.lens if kv_len is None else kv_len
    off = lead + np.concatenate([[0], np.cumsum(new)])
    q = rows_of(int(off[-1]) + tail, q_heads, paged.dim, paged.dtype, paged.rng, pad=8, scale=q_scale)
    got = (run_cross if cross else run_prompt)(ctx, paged, q, off, q_heads, paged.dim**-0.5, out, kv_len=kv_len, slots=slots, ldo_pad=8)
    whose = np.repeat(np.arange(len(new)), new)
    slot = [i if slots is None else slots[i] for i in range(len(new))]
    have = [max(0, min(n, paged.width * paged.page)) if 0 <= s < len(paged.lens) else 0 for n, s in zip(lens, slot)]
    limits = [have[i] if cross else max(0, have[i] - new[i] + j + 1) for i in range(len(new)) for j in range(new[i])]
    inside = slice(lead, len(q) - tail)
    checked(paged, got[inside], q[inside], limits,
            lambda r, h: paged.entries(slot[whose[r]] if limits[r] else 0, limits[r], h), q_heads, paged.kv_heads, paged.dim,
            paged.dim**-0.5, out, what)
    raw = got.view(np.uint16 if out != "f32" else np.float32)
    assert (raw[:, q_heads * paged.dim:] == 7).all() and (raw[:lead] == 7).all() and (raw[len(q) - tail:] == 7).all()
    return q, got


@pytest.mark.parametrize("q_heads,kv_heads,dim,page,dtype,out,order", SHAPES)
def test_prompt_packed(ctx, q_heads, kv_heads, dim, page, dtype, out, order):
    """Whole prompts of every edge length, an empty one among them."""
    new = [5, 0, 1, 33, 64, 65, 2, 130, 31, 16]
    paged = Paged8(new, kv_heads, dim, page, dtype, order, seed=dim + q_heads)
    packed_and_check(ctx, paged, new, q_heads, out, lead=3, tail=5)


@pytest.mark.parametrize("q_heads,kv_heads,dim,page,dtype,out,order", SHAPES[:8])
def test_prompt_resumed(ctx, q_heads, kv_heads, dim, page, dtype, out, order):
    """New tokens after cached ones, and sequences with fewer keys than new tokens: their first see nothing."""
    new, lens = [7, 40, 1, 66, 12, 70], [500, 40, 300, 130, 5, 0]
    paged = Paged8(lens, kv_heads, dim, page, dtype, order, seed=dim + q_heads)
    packed_and_check(ctx, paged, new, q_heads, out)


@pytest.mark.parametrize("q_heads,kv_heads,dim,dtype,out", [(8, 4, 128, "bf16", "bf16"), (4, 4, 64, "f16", "f32"), (6, 2, 256, "bf16", "f32"),
                                                            (4, 2, 128, "f16", "f16")])
def test_prompt_one_long(ctx, q_heads, kv_heads, dim, dtype, out):
    paged = Paged8([777], kv_heads, dim, 16, dtype, seed=1)
    packed_and_check(ctx, paged, [777], q_heads, out)


def test_prompt_many_workgroups(ctx):
    """Enough rows that each workgroup takes 128 of them."""
    for dim, dtype, out in ((128, "bf16", "bf16"), (64, "f16", "f16"), (256, "bf16", "f32")):
        paged = Paged8([300] * 20, 8, dim, 32, dtype, seed=dim)
        new = [300, 290, 1, 129, 130, 64] + [100 + 3 * i for i in range(14)]
        packed_and_check(ctx, paged, new, 16, out)


def test_prompt_slots_and_lengths_outside(ctx):
    paged = Paged8([64, 50, 128, 20], 4, 64, 16, "bf16", seed=1)
    for cross in (False, True):
        packed_and_check(ctx, paged, [10, 20, 30, 4, 6, 3], 8, "f32", kv_len=[50, 20, 1 << 30, 10, 9, -4], slots=[1, 3, 2, -1, 4, 0], cross=cross)


@pytest.mark.parametrize("dim,dtype", [(64, "f16"), (128, "bf16"), (256, "bf16")])
@pytest.mark.parametrize("n,new,at", [(150, 150, 77), (2200, 90, 2150)])
def test_prompt_nan_after(ctx, dim, dtype, n, new, at):
    """NaN keys and values at later places do not touch earlier tokens' results; later ones get what they see."""
    paged = Paged8([n], 2, dim, 16, dtype, seed=dim)
    p = paged.table[0, at // 16]
    odd = np.arange(dim) % 5 == 2
    paged.v[p, 0, at % 16, odd] = 0x7F
    paged.k[p, 1, at % 16, 3] = 0xFF
    paged.upload()
    q = rows_of(new, 4, dim, dtype, paged.rng)
    got = run_prompt(ctx, paged, q, [0, new], 4, dim**-0.5, "f32")
    first = at - (n - new)  # of the tokens that see it
    check(got[:first], q[:first], [n - new + j + 1 for j in range(first)], lambda r, h: paged.entries(0, n - new + r + 1, h), 4, 2, dim,
          dim**-0.5, "f32", "before")
    late = got[first:].reshape(new - first, 2, 2, dim)
    assert np.isnan(late[:, 0][..., odd]).all() and np.isfinite(late[:, 0][..., ~odd]).all() and np.isnan(late[:, 1]).all()


@pytest.mark.parametrize("q_heads,kv_heads,dim,page,dtype,out", [
    (8, 1, 64, 16, "f16", "f16"), (6, 2, 64, 64, "bf16", "f32"), (4, 2, 128, 16, "bf16", "bf16"), (3, 1, 256, 32, "f16", "f32")])
def test_prompt_long_contexts(ctx, q_heads, kv_heads, dim, page, dtype, out):
    """A few new tokens after contexts that end anywhere in the tiles that the waves take in turn."""
    new, lens = [5, 40, 1, 34, 3, 12, 0, 2], [2500, 2055, 2111, 300, 2, 0, 17, 2304]
    paged = Paged8(lens, kv_heads, dim, page, dtype, seed=dim + q_heads)
    packed_and_check(ctx, paged, new, q_heads, out)


def test_prompt_matches_steps(ctx):
    """The last token of a prompt is a step over the same pages, and a token of a cross call."""
    paged = Paged8([90, 200, 33], 2, 128, 16, "bf16", seed=9)
    q = rows_of(323, 8, 128, "bf16", paged.rng)
    got = run_prompt(ctx, paged, q, [0, 90, 290, 323], 8, 0.1, "f32")
    last = [89, 289, 322]
    step = run_step(ctx, paged, np.ascontiguousarray(q[last]), 8, 0.1, "f32")
    assert np.linalg.norm(got[last] - step) <= 2e-5 * np.linalg.norm(step)
    cross = run_cross(ctx, paged, np.ascontiguousarray(q[last]), [0, 1, 2, 3], 8, 0.1, "f32")
    assert np.linalg.norm(cross - step) <= 2e-5 * np.linalg.norm(step)


# ---- cross attention -------------------------------------------------------------------------------


@pytest.mark.parametrize("kind", [Paged, Paged8])
@pytest.mark.parametrize("q_heads,kv_heads,dim,page,dtype,out,order", SHAPES)
def test_cross_packed(ctx, q_heads, kv_heads, dim, page, dtype, out, order, kind):
    """Targets of every edge length over states of every edge length, none on either side among them."""
    new, lens = [5, 0, 1, 33, 64, 65, 2, 130, 31, 16, 7], [64, 9, 700, 1, 65, 16, 0, 33, 129, 300, 15]
    paged = kind(lens, kv_heads, dim, page, dtype, order, seed=dim + q_heads)
    packed_and_check(ctx, paged, new, q_heads, out, lead=2, tail=3, cross=True)


@pytest.mark.parametrize("kind", [Paged, Paged8])
def test_cross_long_and_wide(ctx, kind):
    """Few tokens over long states (groups of waves take turns), many over short ones (128 rows a workgroup)."""
    for dim, dtype, out in ((64, "f16", "f16"), (128, "bf16", "f32"), (256, "bf16", "bf16")):
        paged = kind([2500, 2055, 0, 2304], 2, dim, 16, dtype, seed=dim)
        packed_and_check(ctx, paged, [4, 30, 5, 1], 4, out, cross=True)
        paged = kind([40, 100, 3], 16, dim, 32, dtype, seed=dim)
        packed_and_check(ctx, paged, [400, 300, 390], 16, out, cross=True)


@pytest.mark.parametrize("kind", [Paged, Paged8])
def test_cross_slots_and_nan(ctx, kind):
    """Several sequences over one slot's states; a NaN value is everybody's."""
    paged = kind([90, 200], 2, 128, 16, "bf16", seed=9)
    slots, lens = [1, 1, 0, 1], [200, 77, 90, 0]
    packed_and_check(ctx, paged, [20, 3, 40, 2], 8, "f32", kv_len=lens, slots=slots, cross=True)
    paged.v[paged.table[1, 5], 0, 3, 9] = 0x7F if kind is Paged8 else 0x7FC0
    paged.upload()
    q = rows_of(65, 8, 128, "bf16", paged.rng)
    got = run_cross(ctx, paged, q, [0, 20, 23, 63, 65], 8, 0.1, "f32", kv_len=lens, slots=slots).reshape(65, 2, 4, 128)
    assert np.isnan(got[:20, 0, :, 9]).all() and np.isfinite(got[20:]).all() and not got[63:].any()
    assert np.isfinite(np.delete(got[:, 0], 9, axis=2)).all() and np.isfinite(got[:, 1]).all()


# ---- the rest --------------------------------------------------------------------------------------


def test_captured(ctx):
    """Captured calls, replayed between other work, give what eager ones give."""
    lib = hip.lib()
    paged = Paged8([1500, 900, 31], 2, 128, 16, seed=4)
    n = ctx.attn_step_workspace(3, 8, paged.cache, 1500)
    q = rows_of(3, 8, 128, "bf16", paged.rng, scale=2.0)
    work, dq, dl, do = device(np.zeros(max(n, 16), np.uint8)), device(q), device(np.array(paged.lens, np.int32)), device(np.arange(4, dtype=np.int32))
    outs = [out_array(3, 8 * 128, "f32") for _ in range(3)]
    stream, graph, run = (ctypes.c_void_p() for _ in range(3))
    hip.check(lib.hipStreamCreateWithFlags(ctypes.byref(stream), 1), "stream")
    with Context(0) as own:
        own.set_stream(stream.value)
        hip.check(lib.hipStreamBeginCapture(stream, 2), "begin")
        own.attn_step_device(3, 8, dq, 8 * 128, paged.cache, dl, 1500, 0.1, outs[0], 8 * 128, "f32", workspace=work, workspace_bytes=work.nbytes)
        own.attn_prompt_device(3, 3, 8, dq, 8 * 128, paged.cache, do, dl, 0.1, outs[1], 8 * 128, "f32")
        own.attn_cross_device(3, 3, 8, dq, 8 * 128, paged.cache, do, dl, 0.1, outs[2], 8 * 128, "f32")
        hip.check(lib.hipStreamEndCapture(stream, ctypes.byref(graph)), "end")
        hip.check(lib.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0), "instantiate")
        for i in range(4):
            q = rows_of(3, 8, 128, "bf16", paged.rng, scale=2.0)
            dq.upload(q)
            eager = [run_step(ctx, paged, q, 8, 0.1, "f32"), run_prompt(ctx, paged, q, [0, 1, 2, 3], 8, 0.1, "f32"),
                     run_cross(ctx, paged, q, [0, 1, 2, 3], 8, 0.1, "f32")]
            hip.check(lib.hipGraphLaunch(run, stream), "launch")
            hip.check(lib.hipStreamSynchronize(stream), "wait")
            for out, want in zip(outs, eager):
                assert np.array_equal(out.numpy().view(np.uint32), want.view(np.uint32)), f"replay {i}"
        own.set_stream(None)
    hip.check(lib.hipGraphExecDestroy(run), "destroy")
    hip.check(lib.hipGraphDestroy(graph), "destroy")
    hip.check(lib.hipStreamDestroy(stream), "destroy")


def test_offsets_past_32_bits(ctx):
    """Pages whose byte offsets pass 2^32: a pool of 4.5 GiB of which only the used pages are written."""
    page, kv_heads, dim = 1024, 8, 128
    size = page * kv_heads * dim
    pages = (9 << 29) // size + 1
    far = [pages - 1, 3, pages - 2]
    paged = Paged8([2500], kv_heads, dim, page, "bf16", seed=1)
    k, v = (hip.DeviceArray((pages * size,), np.uint8) for _ in range(2))
    ks, vs = (hip.DeviceArray((pages * kv_heads * (page // 16),), np.uint8) for _ in range(2))
    blocks = kv_heads * (page // 16)
    for i, p in enumerate(far):
        for d, s, n in ((k, paged.dk, size), (v, paged.dv, size), (ks, paged.dks, blocks), (vs, paged.dvs, blocks)):
            hip.check(hip.lib().hipMemcpy(d.ptr + n * p, s.ptr + n * int(paged.table[0, i]), n, hip.D2D), "copy")
    table = device(np.array([far], np.int32))
    q = rows_of(1, 16, dim, "bf16", paged.rng)
    a = run_step(ctx, paged, q, 16, 0.1, "f32")
    q2 = rows_of(40, 16, dim, "bf16", paged.rng)
    b = run_prompt(ctx, paged, q2, [0, 40], 16, 0.1, "f32")
    paged.cache = Kv8Cache(k, v, ks, vs, "bf16", kv_heads, dim, pages, page, table, 1, 3)
    assert np.array_equal(run_step(ctx, paged, q, 16, 0.1, "f32"), a)
    assert np.array_equal(run_prompt(ctx, paged, q2, [0, 40], 16, 0.1, "f32"), b)


def test_two_contexts_at_once(ctx):
    """Calls of two contexts on their own streams, each with its own workspace, at the same time."""
    paged = [Paged8([1900, 700], 2, 128, 16, seed=s) for s in (1, 2)]
    qs = [rows_of(2, 8, 128, "bf16", p.rng, scale=2.0) for p in paged]
    alone = [run_step(ctx, p, q, 8, 0.1, "f32") for p, q in zip(paged, qs)]
    with Context(0) as a, Context(0) as b:
        outs, keep = [], []
        for c, p, q in zip((a, b), paged, qs):
            n = c.attn_step_workspace(2, 8, p.cache, 1900)
            keep.append((device(np.zeros(max(n, 16), np.uint8)), device(q), device(np.array(p.lens, np.int32))))
            outs.append(out_array(2, 8 * 128, "f32"))
        hip.synchronize()
        for _ in range(20):
            for c, p, (w, dq, dl), o in zip((a, b), paged, keep, outs):
                c.attn_step_device(2, 8, dq, 8 * 128, p.cache, dl, 1900, 0.1, o, 8 * 128, "f32", workspace=w, workspace_bytes=w.nbytes)
        a.synchronize()
        b.synchronize()
        for o, want in zip(outs, alone):
            assert np.array_equal(o.numpy().view(np.uint32), want.view(np.uint32))


def test_refused_calls_launch_nothing(ctx):
    """(tests/test_attention8_host.py has the whole list, without a GPU.)"""
    paged = Paged8([40, 20], 2, 64, 16, "bf16", seed=1)
    x, i32 = device(np.zeros(1 << 14, np.uint16)), device(np.zeros(64, np.int32))
    for fn, args in ((ctx.attn_step_device, (1 << 27, 2, x, 128, paged.cache, i32, 40, 0.1, x, 128, "bf16")),
                     (ctx.attn_prompt_device, (1 << 27, 8, 2, x, 128, paged.cache, i32, i32, 0.1, x, 128, "bf16")),
                     (ctx.attn_cross_device, (2, 8, 2, x, 128, paged.cache, i32, i32, 0.1, x, 128, "f16"))):
        with pytest.raises(SamplerError):
            fn(*args)
    q = rows_of(2, 2, 64, "bf16", paged.rng)
    run_step(ctx, paged, q, 2, 0.1)
