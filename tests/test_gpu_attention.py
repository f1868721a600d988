"""GPU checks of attention over a paged cache against the 64-bit oracle: lengths around every tile edge, head groups,
types, page sizes, layouts, shared prefixes, what unseen places hold, refusals.

Every page entry that no row may read is NaN, infinity or the type's largest value throughout (attention_cases.Paged)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from oracle import attention_np as on
from voxwerk_amd import _lib, hip
from voxwerk_amd.attention import KvCache, SharedPrefix
from voxwerk_amd.sampler import Context, SamplerError

from attention_cases import Paged, check, device, out_array, poison, rows_of, run_prompt, run_step

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
]


def step_and_check(ctx, paged, q_heads, out, share=(), scale=None, q_scale=2.0, what="step", kv_len=None, slots=None, **kw):
    lens = paged.lens if kv_len is None else kv_len
    rows = len(lens)
    scale = scale or paged.dim**-0.5
    q = rows_of(rows, q_heads, paged.dim, paged.dtype, paged.rng, pad=8, scale=q_scale)
    got = run_step(ctx, paged, q, q_heads, scale, out, share=share, kv_len=kv_len, slots=slots, ldo_pad=8, **kw)
    slot = lambda r: r if slots is None else slots[r]  # noqa: E731
    cap = paged.width * paged.page
    seen = [min(n, cap) if 0 <= slot(r) < len(paged.lens) else 0 for r, n in enumerate(lens)]
    check(got, q, seen, lambda r, h: paged.entries(slot(r) if seen[r] > 0 else 0, max(seen[r], 0), h), q_heads, paged.kv_heads,
          paged.dim, scale, paged.dtype, out, what)
    assert (got.view(np.uint16 if out != "f32" else np.float32)[:, q_heads * paged.dim:] == 7).all(), "the pad was written"
    return q, got


@pytest.mark.parametrize("q_heads,kv_heads,dim,page,dtype,out,order", SHAPES)
def test_step_lengths(ctx, q_heads, kv_heads, dim, page, dtype, out, order):
    paged = Paged(EDGES, kv_heads, dim, page, dtype, order, seed=dim + q_heads)
    step_and_check(ctx, paged, q_heads, out)


@pytest.mark.parametrize("q_heads,kv_heads,dim,page,dtype,out,order", SHAPES)
def test_step_one_long_row(ctx, q_heads, kv_heads, dim, page, dtype, out, order):
    """Few rows: a row's keys are divided among many workgroups, with and without the workspace for it."""
    paged = Paged([3001], kv_heads, dim, page, dtype, order, seed=dim + q_heads)
    step_and_check(ctx, paged, q_heads, out)
    step_and_check(ctx, paged, q_heads, out, work=None, what="no workspace")


@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("page,prefix", [(16, 16), (16, 500), (64, 70), (32, 1), (16, 1030)])
def test_step_shared_prefix(ctx, rows, page, prefix):
    r = np.random.default_rng(rows + prefix)
    for q_heads, kv_heads, dim, dtype, out in ((16, 8, 128, "bf16", "bf16"), (7, 1, 64, "f16", "f32"), (4, 4, 256, "bf16", "f32")):
        lens = (prefix + r.integers(1, 200, rows)).tolist()
        share = [(0, rows, prefix)]
        paged = Paged(lens, kv_heads, dim, page, dtype, "heads", seed=rows, share=share)
        q, got = step_and_check(ctx, paged, q_heads, out, share=share, what=f"prefix {prefix}")
        alone = run_step(ctx, paged, q, q_heads, dim**-0.5, out, ldo_pad=8)
        tol = 2e-5 if out == "f32" else 4 * on.UNIT[out]
        a, b = on.widen(got)[:, :q_heads * dim], on.widen(alone)[:, :q_heads * dim]
        assert np.linalg.norm(a - b) <= tol * np.linalg.norm(b) * 64


def test_step_groups(ctx):
    """Several groups of different prefixes, rows outside every group, groups of one row and of none."""
    share = [(2, 7, 130), (7, 8, 64), (8, 8, 40), (8, 45, 333)]
    lens = [9, 200] + [130 + 11 * i for i in range(1, 6)] + [100] + [334 + 7 * i for i in range(37)] + [0, 77]
    for q_heads, kv_heads, dim, dtype, out in ((16, 8, 128, "bf16", "f32"), (32, 4, 64, "f16", "f16"), (40, 1, 128, "bf16", "bf16")):
        paged = Paged(lens, kv_heads, dim, 16, dtype, "tokens", seed=3, share=share)
        step_and_check(ctx, paged, q_heads, out, share=share)


def test_step_shorter_than_the_prefix(ctx):
    """A row that ends inside its group's prefix sees its own length only; keys past it may hold anything."""
    share = [(0, 6, 100)]
    paged = Paged([160, 300, 101, 100, 140, 120], 2, 128, 16, "bf16", seed=5, share=share)
    step_and_check(ctx, paged, 8, "f32", share=share, kv_len=[160, 33, 101, 100, 0, 64])
    # value 70 of the prefix is infinite: rows that see it are infinite or NaN there, the others as ever
    p = paged.table[0, 70 // 16]
    paged.v[p, :, 70 % 16, 5] = 0x7F80
    paged.upload()
    q = rows_of(6, 8, 128, "bf16", paged.rng)
    lens = [160, 33, 101, 100, 0, 64]
    got = run_step(ctx, paged, q, 8, 128**-0.5, "f32", kv_len=lens, share=share).reshape(6, 8, 128)
    assert not np.isfinite(got[[0, 2, 3], :, 5]).any() and np.isfinite(got[[1, 4, 5]]).all()
    assert np.isfinite(np.delete(got, 5, axis=2)).all()
    keep = [1, 4, 5]
    check(got.reshape(6, -1)[keep], q[keep], [lens[i] for i in keep], lambda r, h: paged.entries(keep[r], lens[keep[r]], h), 8, 2,
          128, 128**-0.5, "bf16", "f32", "rows that do not see it")


def test_step_slots_and_lengths_outside(ctx):
    """Slots in any order; a slot outside the cache has no keys, a length above the table's is cut to it."""
    paged = Paged([64, 50, 128, 20], 4, 64, 16, "bf16", seed=1)
    step_and_check(ctx, paged, 8, "f32", kv_len=[50, 20, 128, 10, 30, 5], slots=[1, 3, 2, -1, 4, 0], max_len=128)
    step_and_check(ctx, paged, 8, "f32", kv_len=[1 << 30, -5], slots=[2, 0], max_len=16)


@pytest.mark.parametrize("max_len", [0, 1, 100, 5000])
def test_step_longer_than_announced(ctx, max_len):
    """max_len only divides the work."""
    paged = Paged([700, 3, 0, 260], 2, 128, 16, "bf16", seed=2)
    step_and_check(ctx, paged, 4, "f32", max_len=max_len)


def test_step_sharp_and_flat_scores(ctx):
    """One key with nearly all the weight, wherever it lies; equal scores; scores that grow along the keys."""
    for at in (0, 31, 64, 450, 699):
        paged = Paged([700], 1, 64, 16, "bf16", seed=at)
        paged.k[paged.table[0, at // 16], 0, at % 16] = on.to_bf16(np.full(64, 3.0, np.float32))
        paged.upload()
        q = np.full((1, 4 * 64), 0x4040, np.uint16)  # 3.0
        got = run_step(ctx, paged, q, 4, 0.125, "f32")
        check(got, q, [700], lambda r, h: paged.entries(0, 700, h), 4, 1, 64, 0.125, "bf16", "f32", f"sharp at {at}")
    for grow in (0.0, 0.02, 0.5, -0.5):
        paged = Paged([700], 1, 64, 16, "f16", seed=7)
        t = np.arange(700)
        k = np.zeros((700, 64), np.float16)
        k[:, 0] = (t * grow).astype(np.float16)
        paged.k[paged.table[0, t // 16], 0, t % 16] = k
        paged.upload()
        q = np.zeros((1, 2 * 64), np.float16)
        q[:, ::64] = 1.0
        got = run_step(ctx, paged, q, 2, 1.0, "f32")
        check(got, q, [700], lambda r, h: paged.entries(0, 700, h), 2, 1, 64, 1.0, "f16", "f32", f"grows by {grow}")


def test_step_nonfinite_that_is_seen(ctx):
    """A NaN key or a NaN value that a row sees makes its outputs NaN, as the formula says; other rows are as ever."""
    paged = Paged([100, 100, 100], 1, 64, 16, "bf16", seed=11)
    paged.k[paged.table[0, 2], 0, 3, 9] = 0x7FC0
    paged.v[paged.table[1, 2], 0, 3, 9] = 0x7FC0
    paged.upload()
    q = rows_of(3, 2, 64, "bf16", paged.rng)
    got = run_step(ctx, paged, q, 2, 0.125, "f32").reshape(3, 2, 64)
    assert np.isnan(got[0]).all() and np.isnan(got[1, :, 9]).all() and np.isfinite(np.delete(got[1], 9, axis=1)).all()
    check(got.reshape(3, -1)[2:], q[2:], [100], lambda r, h: paged.entries(2, 100, h), 2, 1, 64, 0.125, "bf16", "f32", "beside NaN")


def test_step_workspace_is_ready_again(ctx):
    """One workspace for calls of different sizes in a row, and the same bits each time."""
    long, wide = Paged([2900, 1500], 2, 128, 16, seed=1), Paged([700] * 24, 2, 128, 16, seed=2)
    share = [(0, 24, 500)]
    shared = Paged([700] * 24, 2, 128, 16, seed=3, share=share)
    n = max(ctx.attn_step_workspace(2, 8, long.cache, 2900), ctx.attn_step_workspace(24, 8, wide.cache, 700),
            ctx.attn_step_workspace(24, 8, shared.cache, 700, SharedPrefix(1, 16, 16, 500, True)))
    work = device(np.zeros(n, np.uint8))
    qs = [rows_of(len(p.lens), 8, 128, "bf16", p.rng, scale=2.0) for p in (long, wide, shared)]
    first = None
    for _ in range(3):
        got = [run_step(ctx, p, q, 8, 0.1, "f32", work=work, share=s) for p, q, s in zip((long, wide, shared), qs, ((), (), share))]
        first = first or got
        for a, b in zip(first, got):
            assert np.array_equal(a.view(np.uint32), b.view(np.uint32))


def test_step_workspace_serves_other_sizes(ctx):
    """One workspace, zeroed once, between calls whose rows, parts, head sizes and types differ: each is right."""
    share = [(0, 24, 500)]
    # (cache, query heads, prefixes): many parts of few rows come before few parts of many
    calls = [
        (Paged([2900, 1500], 2, 128, 16, seed=1), 8, ()),
        (Paged([700] * 24, 2, 128, 16, seed=2), 8, ()),
        (Paged([2600], 1, 64, 16, "f16", seed=3), 5, ()),
        (Paged([700] * 24, 2, 128, 16, seed=4, share=share), 8, share),
        (Paged([900, 300, 0, 1700, 65], 2, 256, 32, "f16", seed=5), 2, ()),
        (Paged([600] * 40, 3, 64, 16, seed=6), 12, ()),
    ]
    n = max(ctx.attn_step_workspace(len(p.lens), h, p.cache, max(p.lens), SharedPrefix(1, 16, 16, 500, True) if s else None) for p, h, s in calls)
    work = device(np.zeros(n, np.uint8))
    for _ in range(2):
        for i, (p, h, s) in enumerate(calls):
            step_and_check(ctx, p, h, "f32", share=s, work=work, what=f"call {i}")


def test_step_workspace_of_larger_sizes_is_enough(ctx):
    """A workspace for the largest batch and length serves every smaller call: fewer rows divide their keys further."""
    paged = Paged([1800] * 24, 2, 128, 16, seed=7)
    for prefix in (None, SharedPrefix(1, 16, 16, 900, True)):
        n = ctx.attn_step_workspace(24, 8, paged.cache, 1800, prefix)
        for rows in range(25):
            for most in (0, 1, 256, 257, 700, 1800):
                assert ctx.attn_step_workspace(rows, 8, paged.cache, most, prefix) <= n
                assert ctx.attn_step_workspace(rows, 8, paged.cache, most) <= n
    work = device(np.zeros(ctx.attn_step_workspace(24, 8, paged.cache, 1800), np.uint8))
    for rows in (24, 1, 5, 24, 13):
        few = Paged([1800] * rows, 2, 128, 16, seed=rows)
        step_and_check(ctx, few, 8, "f32", work=work, what=f"{rows} rows")


def test_step_captured(ctx):
    """A captured step, replayed between other work, gives what an eager one gives."""
    lib = hip.lib()
    paged = Paged([1500, 900, 31], 2, 128, 16, seed=4)
    q = rows_of(3, 8, 128, "bf16", paged.rng, scale=2.0)
    n = ctx.attn_step_workspace(3, 8, paged.cache, 1500)
    work, dq, dl = device(np.zeros(max(n, 16), np.uint8)), device(q), device(np.array(paged.lens, np.int32))
    out = out_array(3, 8 * 128, "f32")
    stream, graph, run = (ctypes.c_void_p() for _ in range(3))
    hip.check(lib.hipStreamCreateWithFlags(ctypes.byref(stream), 1), "stream")
    with Context(0) as own:
        own.set_stream(stream.value)
        hip.check(lib.hipStreamBeginCapture(stream, 2), "begin")
        own.attn_step_device(3, 8, dq, 8 * 128, paged.cache, dl, 1500, 0.1, out, 8 * 128, "f32", workspace=work, workspace_bytes=work.nbytes)
        hip.check(lib.hipStreamEndCapture(stream, ctypes.byref(graph)), "end")
        hip.check(lib.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0), "instantiate")
        for i in range(4):
            q = rows_of(3, 8, 128, "bf16", paged.rng, scale=2.0)
            dq.upload(q)
            eager = run_step(ctx, paged, q, 8, 0.1, "f32")
            hip.check(lib.hipGraphLaunch(run, stream), "launch")
            hip.check(lib.hipStreamSynchronize(stream), "wait")
            assert np.array_equal(out.numpy().view(np.uint32), eager.view(np.uint32)), f"replay {i}"
        own.set_stream(None)
    hip.check(lib.hipGraphExecDestroy(run), "destroy")
    hip.check(lib.hipGraphDestroy(graph), "destroy")
    hip.check(lib.hipStreamDestroy(stream), "destroy")


# ---- prompts ---------------------------------------------------------------------------------------


def prompt_and_check(ctx, paged, new, q_heads, out, kv_len=None, slots=None, q_scale=2.0, lead=0, tail=0, what="prompt"):
    """new[i] tokens of sequence i; `lead` and `tail` rows of the queries belong to no sequence."""
    lens = paged.lens if kv_len is None else kv_len
    off = lead + np.concatenate([[0], np.cumsum(new)])
    q = rows_of(int(off[-1]) + tail, q_heads, paged.dim, paged.dtype, paged.rng, pad=8, scale=q_scale)
    got = run_prompt(ctx, paged, q, off, q_heads, paged.dim**-0.5, out, kv_len=kv_len, slots=slots, ldo_pad=8)
    whose = np.repeat(np.arange(len(new)), new)
    slot = [i if slots is None else slots[i] for i in range(len(new))]
    have = [min(n, paged.width * paged.page) if 0 <= s < len(paged.lens) else 0 for n, s in zip(lens, slot)]
    limits = [max(0, have[i] - new[i] + j + 1) for i in range(len(new)) for j in range(new[i])]
    inside = slice(lead, len(q) - tail)
    check(got[inside], q[inside], limits,
          lambda r, h: paged.entries(slot[whose[r]] if limits[r] else 0, limits[r], h), q_heads, paged.kv_heads, paged.dim,
          paged.dim**-0.5, paged.dtype, out, what)
    raw = got.view(np.uint16 if out != "f32" else np.float32)
    assert (raw[:, q_heads * paged.dim:] == 7).all() and (raw[:lead] == 7).all() and (raw[len(q) - tail:] == 7).all()
    return q, got


@pytest.mark.parametrize("q_heads,kv_heads,dim,page,dtype,out,order", SHAPES)
def test_prompt_packed(ctx, q_heads, kv_heads, dim, page, dtype, out, order):
    """Whole prompts of every edge length, an empty one among them."""
    new = [5, 0, 1, 33, 64, 65, 2, 130, 31, 16]
    paged = Paged(new, kv_heads, dim, page, dtype, order, seed=dim + q_heads)
    prompt_and_check(ctx, paged, new, q_heads, out, lead=3, tail=5)


@pytest.mark.parametrize("q_heads,kv_heads,dim,page,dtype,out,order", SHAPES[:8])
def test_prompt_resumed(ctx, q_heads, kv_heads, dim, page, dtype, out, order):
    """New tokens after cached ones, and sequences with fewer keys than new tokens: their first see nothing."""
    new, lens = [7, 40, 1, 66, 12, 70], [500, 40, 300, 130, 5, 0]
    paged = Paged(lens, kv_heads, dim, page, dtype, order, seed=dim + q_heads)
    prompt_and_check(ctx, paged, new, q_heads, out)


@pytest.mark.parametrize("q_heads,kv_heads,dim,dtype,out", [(8, 4, 128, "bf16", "bf16"), (4, 4, 64, "f16", "f32"), (6, 2, 256, "bf16", "f32")])
def test_prompt_one_long(ctx, q_heads, kv_heads, dim, dtype, out):
    paged = Paged([777], kv_heads, dim, 16, dtype, seed=1)
    prompt_and_check(ctx, paged, [777], q_heads, out)


def test_prompt_slots_and_lengths_outside(ctx):
    paged = Paged([64, 50, 128, 20], 4, 64, 16, "bf16", seed=1)
    prompt_and_check(ctx, paged, [10, 20, 30, 4, 6], 8, "f32", kv_len=[50, 20, 1 << 30, 10, 9], slots=[1, 3, 2, -1, 4])


@pytest.mark.parametrize("dim,dtype", [(64, "f16"), (128, "bf16"), (256, "bf16")])
def test_prompt_nonfinite_after(ctx, dim, dtype):
    """Infinite and NaN keys and values at later places do not touch earlier tokens' results."""
    n, at = 150, 77
    paged = Paged([n], 2, dim, 16, dtype, seed=dim)
    p = paged.table[0, at // 16]
    bad = poison((2, dim), dtype, paged.rng)
    paged.v[p, :, at % 16] = bad
    paged.k[p, 1, at % 16] = bad[1]
    paged.upload()
    q = rows_of(n, 4, dim, dtype, paged.rng)
    got = run_prompt(ctx, paged, q, [0, n], 4, dim**-0.5, "f32")
    check(got[:at], q[:at], list(range(1, at + 1)), lambda r, h: paged.entries(0, r + 1, h), 4, 2, dim, dim**-0.5, dtype, "f32", "before")
    nan = np.isnan(on.widen(bad)).any(1)
    late = got[at:].reshape(n - at, 2, 2, dim)
    for h in range(2):
        where = np.isnan(on.widen(bad[h]))
        assert not nan[h] or np.isnan(late[:, h][..., where]).all()
    big = ~np.isfinite(on.widen(bad[0]))
    assert np.isfinite(late[:, 0][..., ~big]).all() and not np.isfinite(late[:, 0][..., big]).any()


@pytest.mark.parametrize("q_heads,kv_heads,dim,page,dtype,out", [
    (8, 1, 64, 16, "f16", "f16"), (6, 2, 64, 64, "bf16", "f32"), (4, 2, 128, 16, "bf16", "bf16"), (3, 1, 256, 32, "f16", "f32")])
def test_prompt_long_contexts(ctx, q_heads, kv_heads, dim, page, dtype, out):
    """A few new tokens after contexts that end anywhere in the tiles that the waves take in turn."""
    new, lens = [5, 40, 1, 34, 3, 12, 0, 2], [2500, 2055, 2111, 300, 2, 0, 17, 2304]
    paged = Paged(lens, kv_heads, dim, page, dtype, seed=dim + q_heads)
    prompt_and_check(ctx, paged, new, q_heads, out)


@pytest.mark.parametrize("dim,dtype", [(64, "bf16"), (64, "f16"), (128, "f16")])
def test_prompt_nonfinite_after_long_context(ctx, dim, dtype):
    """The same behind a long context: earlier new tokens are right, later ones get what they see."""
    n, new, at = 2200, 90, 2150
    paged = Paged([n], 2, dim, 16, dtype, seed=dim)
    p = paged.table[0, at // 16]
    bad = poison((2, dim), dtype, paged.rng)
    paged.v[p, :, at % 16] = bad
    paged.upload()
    q = rows_of(new, 4, dim, dtype, paged.rng)
    got = run_prompt(ctx, paged, q, [0, new], 4, dim**-0.5, "f32")
    first = at - (n - new)  # of the tokens that see it
    check(got[:first], q[:first], [n - new + j + 1 for j in range(first)], lambda r, h: paged.entries(0, n - new + r + 1, h), 4, 2, dim,
          dim**-0.5, dtype, "f32", "before")
    late = got[first:].reshape(new - first, 2, 2, dim)
    for h in range(2):
        odd = ~np.isfinite(on.widen(bad[h]))
        assert np.isfinite(late[:, h][..., ~odd]).all() and not np.isfinite(late[:, h][..., odd]).any()


def test_prompt_matches_steps(ctx):
    """The last token of a prompt is a step over the same pages."""
    paged = Paged([90, 200, 33], 2, 128, 16, "bf16", seed=9)
    q = rows_of(323, 8, 128, "bf16", paged.rng)
    got = run_prompt(ctx, paged, q, [0, 90, 290, 323], 8, 0.1, "f32")
    last = [89, 289, 322]
    step = run_step(ctx, paged, np.ascontiguousarray(q[last]), 8, 0.1, "f32")
    assert np.linalg.norm(got[last] - step) <= 2e-5 * np.linalg.norm(step)


def test_offsets_past_32_bits(ctx):
    """Pages whose byte and entry offsets pass 2^32: a pool of 5 GiB of which only the used pages are written."""
    page, kv_heads, dim = 1024, 8, 128
    size = page * kv_heads * dim
    pages = (5 << 30) // (2 * size) + 1
    far = [pages - 1, 3, pages - 2]
    paged = Paged([2500], kv_heads, dim, page, "bf16", seed=1)
    k, v = (hip.DeviceArray((pages * size,), np.uint16) for _ in range(2))
    for i, p in enumerate(far):
        for d, s in ((k, paged.dk), (v, paged.dv)):
            hip.check(hip.lib().hipMemcpy(d.ptr + 2 * size * p, s.ptr + 2 * size * int(paged.table[0, i]), 2 * size, hip.D2D), "copy")
    table = device(np.array([far], np.int32))
    near = paged.cache
    q = rows_of(1, 16, dim, "bf16", paged.rng)
    a = run_step(ctx, paged, q, 16, 0.1, "f32")
    q2 = rows_of(40, 16, dim, "bf16", paged.rng)
    b = run_prompt(ctx, paged, q2, [0, 40], 16, 0.1, "f32")
    paged.cache = KvCache(k, v, "bf16", kv_heads, dim, pages, page, table, 1, 3)
    assert np.array_equal(run_step(ctx, paged, q, 16, 0.1, "f32"), a)
    assert np.array_equal(run_prompt(ctx, paged, q2, [0, 40], 16, 0.1, "f32"), b)
    paged.cache = near


def test_refusals(ctx):
    paged = Paged([40, 20], 2, 64, 16, "bf16", seed=1)
    x = device(np.zeros(1 << 16, np.uint16))
    i32 = device(np.zeros(64, np.int32))

    def cache(**change):
        c = KvCache(paged.dk, paged.dv, "bf16", 2, 64, paged.pages, 16, paged.dtable, 2, paged.width)
        for name, value in change.items():
            setattr(c.struct, name, value)
        return c

    def step(c=None, rows=2, q_heads=4, q=x, ldq=256, lens=i32, max_len=40, scale=0.1, out=x, ldo=256, out_dtype="bf16", **kw):
        ctx.attn_step_device(rows, q_heads, q, ldq, c or cache(), lens, max_len, scale, out, ldo, out_dtype, **kw)

    def prompt(c=None, seqs=2, tokens=4, q_heads=4, q=x, ldq=256, off=i32, lens=i32, scale=0.1, out=x, ldo=256, out_dtype="bf16"):
        ctx.attn_prompt_device(seqs, tokens, q_heads, q, ldq, c or cache(), off, lens, scale, out, ldo, out_dtype)

    def refused(code, fn, *a, **kw):
        with pytest.raises(SamplerError) as e:
            fn(*a, **kw)
        assert e.value.code == code and ctx.last_error()

    bad, unsupported = _lib.VXS_ERR_INVALID_ARG, _lib.VXS_ERR_UNSUPPORTED
    for fn in (step, prompt):
        for change in ({"pages": 0}, {"slots": -1}, {"page_size": 0}, {"kv_heads": 0}, {"ld_table": 0}, {"dtype": 0}, {"dtype": 9},
                       {"k": None}, {"v": None}, {"table": None}, {"token_stride": 63}, {"head_stride": 0}, {"page_stride": -8},
                       {"kv_heads": 3}):
            refused(bad, fn, cache(**change))
        for change in ({"head_dim": 32}, {"head_dim": 60, "token_stride": 64}, {"page_size": 24}, {"page_size": 8}, {"page_size": 1 << 17},
                       {"token_stride": 68}, {"head_stride": 1028}, {"page_stride": 2052}, {"k": paged.dk.ptr + 2}, {"v": paged.dv.ptr + 8},
                       {"ld_table": 1 << 27}):
            refused(unsupported, fn, cache(**change))
        for kw in ({"q_heads": 3}, {"q_heads": 0}, {"ldq": 248}, {"ldo": 248}, {"scale": 0.0}, {"scale": -1.0}, {"scale": float("nan")},
                   {"scale": float("inf")}, {"out_dtype": "f16"}, {"q": None}, {"out": None}, {"lens": None}):
            refused(bad, fn, **kw)
        for kw in ({"ldq": 260}, {"ldo": 260}, {"q": x.ptr + 8}, {"out": x.ptr + 4}):
            refused(unsupported, fn, **kw)
    refused(bad, step, rows=-1)
    refused(bad, step, max_len=-1)
    refused(bad, prompt, seqs=-1)
    refused(bad, prompt, tokens=-1)
    refused(bad, prompt, off=None)
    refused(unsupported, prompt, tokens=1 << 30)
    refused(bad, step, prefix=SharedPrefix(-1, i32, i32, 4))
    refused(bad, step, prefix=SharedPrefix(1, None, i32, 4))
    refused(bad, step, prefix=SharedPrefix(1, i32, None, 4))
    refused(bad, step, prefix=SharedPrefix(1, i32, i32, -4))
    odd = SharedPrefix(1, i32, i32, 4)
    odd.struct.flags = 1
    refused(bad, step, prefix=odd)
    refused(bad, step, workspace=x.ptr + 4, workspace_bytes=1 << 16)
    n = ctx.attn_step_workspace(1, 4, cache(), 1 << 20)
    assert n >= 0
    if n:
        refused(bad, step, rows=1, max_len=1 << 20, workspace=x, workspace_bytes=n - 1)
    with pytest.raises(SamplerError):
        ctx.attn_step_workspace(-1, 4, cache(), 10)
    step(rows=0)  # nothing to do is no error
    prompt(tokens=0)
    prompt(seqs=0)
    ctx.synchronize()


def test_step_rows_of_one_sequence(ctx):
    """A few new tokens of a long sequence as rows of a step: one slot, a row's own length each, their context shared."""
    n, new = 1500, 9
    paged = Paged([n, 70], 2, 128, 16, "bf16", seed=4)
    q = rows_of(new, 8, 128, "bf16", paged.rng, scale=2.0)
    lens = [n - new + 1 + i for i in range(new)]
    context = n - new
    got = run_step(ctx, paged, q, 8, 0.1, "f32", kv_len=lens, slots=[0] * new, share=[(0, new, context)])
    check(got, q, lens, lambda r, h: paged.entries(0, lens[r], h), 8, 2, 128, 0.1, "bf16", "f32", "rows of one sequence")
    whole = run_prompt(ctx, paged, q, [0, new], 8, 0.1, "f32", kv_len=[n], slots=[0])
    assert np.linalg.norm(whole - got) <= 2e-5 * np.linalg.norm(got)


@pytest.mark.parametrize("rows,prefix", [(6, 90), (70, 900)])
def test_step_shares_where_it_is_faster(ctx, rows, prefix):
    """Without the flag a prefix is shared from some size on; either way the outputs are the rows' own."""
    share = [(0, rows, prefix)]
    paged = Paged([prefix + 1 + i % 37 for i in range(rows)], 8, 128, 16, "bf16", seed=rows, share=share)
    step_and_check(ctx, paged, 16, "f32", share=share, always=False)


def test_too_many_rows_are_refused(ctx):
    """A launch's threads are counted in 32 bits: more rows or sequences than that are an error, and nothing is launched."""
    paged = Paged([40, 20], 2, 64, 16, "bf16", seed=1)
    x, i32 = device(np.zeros(1 << 14, np.uint16)), device(np.zeros(64, np.int32))
    with pytest.raises(SamplerError):
        ctx.attn_step_device(1 << 27, 2, x, 128, paged.cache, i32, 40, 0.1, x, 128, "bf16")
    with pytest.raises(SamplerError):
        ctx.attn_prompt_device(1 << 27, 8, 2, x, 128, paged.cache, i32, i32, 0.1, x, 128, "bf16")
    q = rows_of(2, 2, 64, "bf16", paged.rng)
    run_step(ctx, paged, q, 2, 0.1)
