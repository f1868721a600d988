"""GPU checks of attention over a paged cache where sizes change how the work is divided, against the 64-bit oracle."""
from __future__ import annotations

import threading

import numpy as np
import pytest

from voxwerk_amd import _lib, hip
from voxwerk_amd.attention import SharedPrefix
from voxwerk_amd.sampler import Context, SamplerError

from attention_cases import Paged, as_out, check, device, out_array, rows_of, run_prompt, run_step

pytestmark = pytest.mark.gpu


def run_announced(ctx, paged, q, q_heads, scale, out_dtype, kv_len, slots, max_len, off, prefix_len, prefix_max):
    """A step whose max_len and prefix max_len are capacities, above the real lengths."""
    rows, width = len(q), q_heads * paged.dim
    keep = [device(np.array(x, np.int32)) for x in (off, prefix_len, kv_len, slots)]
    prefix = SharedPrefix(len(prefix_len), keep[0], keep[1], prefix_max, True)
    n = ctx.attn_step_workspace(rows, q_heads, paged.cache, max_len, prefix)
    work, dq, out = device(np.zeros(n, np.uint8)), device(q), out_array(rows, width, out_dtype)
    hip.synchronize()
    ctx.attn_step_device(rows, q_heads, dq, q.shape[1], paged.cache, keep[2], max_len, scale, out, width, out_dtype, slots=keep[3],
                         prefix=prefix, workspace=work, workspace_bytes=n)
    ctx.synchronize()
    return as_out(out.numpy(), out_dtype)


@pytest.mark.parametrize("max_len", [262145, 300000])
@pytest.mark.parametrize("q_heads,dim,dtype,out", [(1, 64, "bf16", "f32"), (3, 128, "f16", "f16")])
def test_step_parts_of_a_wave_each(ctx, max_len, q_heads, dim, dtype, out):
    """More rows than workgroups at once, announced lengths far above the real ones: a long row outside the group is divided
    among waves that share nothing, at whole granules whatever max_len is."""
    rows, shared = 514, 48
    paged = Paged([60, 3500], 1, dim, 16, dtype, seed=dim, width=-(-max_len // 16))
    kv_len, slots = [60] * (rows - 1) + [3500], [0] * (rows - 1) + [1]
    q = rows_of(rows, q_heads, dim, dtype, paged.rng, scale=2.0)
    got = run_announced(ctx, paged, q, q_heads, dim**-0.5, out, kv_len, slots, max_len, [0, rows - 1], [shared], max_len - 100)
    check(got, q, kv_len, lambda r, h: paged.entries(slots[r], kv_len[r], h), q_heads, 1, dim, dim**-0.5, dtype, out, f"announced {max_len}")


@pytest.mark.parametrize("rows,q_heads,kv_heads,dim,dtype,out", [
    (600, 1, 1, 64, "f16", "f32"), (300, 40, 1, 64, "bf16", "bf16"), (70, 16, 8, 128, "bf16", "f32"), (520, 2, 1, 256, "f16", "f16")])
def test_step_many_short_rows(ctx, rows, q_heads, kv_heads, dim, dtype, out):
    """Short rows, more than fit at once, without a prefix: a wave each, lengths around every tile edge, some rows without a key."""
    lens = [(0, 1, 15, 16, 31, 33, 64, 65, 100, 255, 256)[r % 11] for r in range(rows)]
    paged = Paged(lens, kv_heads, dim, 16, dtype, seed=rows)
    q = rows_of(rows, q_heads, dim, dtype, paged.rng, scale=2.0)
    got = run_step(ctx, paged, q, q_heads, dim**-0.5, out)
    check(got, q, lens, lambda r, h: paged.entries(r, lens[r], h), q_heads, kv_heads, dim, dim**-0.5, dtype, out, "short rows")


def test_too_many_groups_are_refused(ctx):
    """More prefix groups than a launch has threads for are an error before anything reads them."""
    paged = Paged([900, 700], 2, 64, 16, "bf16", seed=1)
    x, i32 = device(np.zeros(1 << 14, np.uint16)), device(np.zeros(64, np.int32))
    prefix = SharedPrefix((1 << 31) - 1, i32, i32, 600, True)
    n = ctx.attn_step_workspace(64, 4, paged.cache, 900, prefix)
    work = device(np.zeros(n, np.uint8))
    with pytest.raises(SamplerError):
        ctx.attn_step_device(64, 4, x, 256, paged.cache, i32, 900, 0.1, x, 256, "bf16", prefix=prefix, workspace=work, workspace_bytes=n)
    q = rows_of(2, 4, 64, "bf16", paged.rng)
    run_step(ctx, paged, q, 4, 0.1)


@pytest.mark.parametrize("dim,dtype", [(64, "f16"), (128, "bf16"), (256, "bf16")])
def test_a_workspace_too_small_is_refused(ctx, dim, dtype):
    """One byte less than vxs_attn_step_workspace says, with and without a prefix, and nothing is written to it."""
    paged = Paged([1000, 900, 800], 2, dim, 16, dtype, seed=1)
    rows, q_heads = 3, 4
    q = rows_of(rows, q_heads, dim, dtype, paged.rng)
    dq, out, lens = device(q), out_array(rows, q_heads * dim, "f32"), device(np.array(paged.lens, np.int32))
    prefix = SharedPrefix(1, device(np.array([0, 3], np.int32)), device(np.array([500], np.int32)), 500, True)
    for p in (None, prefix):
        n = ctx.attn_step_workspace(rows, q_heads, paged.cache, 1000, p)
        assert n > 0
        work = device(np.zeros(n, np.uint8))
        for short in (n - 1, 16, 0, -1):
            with pytest.raises(SamplerError) as e:
                ctx.attn_step_device(rows, q_heads, dq, q_heads * dim, paged.cache, lens, 1000, 0.1, out, q_heads * dim, "f32", prefix=p,
                                     workspace=work, workspace_bytes=short)
            assert e.value.code == _lib.VXS_ERR_INVALID_ARG and "vxs_attn_step_workspace" in ctx.last_error()
        ctx.synchronize()
        assert not work.numpy().any() and (out.numpy() == 7).all()
    with_prefix = ctx.attn_step_workspace(rows, q_heads, paged.cache, 1000, prefix)
    without = ctx.attn_step_workspace(rows, q_heads, paged.cache, 1000)
    assert without < with_prefix  # (a workspace for calls without a prefix does not serve one with it)
    with pytest.raises(SamplerError):
        ctx.attn_step_device(rows, q_heads, dq, q_heads * dim, paged.cache, lens, 1000, 0.1, out, q_heads * dim, "f32", prefix=prefix,
                             workspace=device(np.zeros(without, np.uint8)), workspace_bytes=without)


@pytest.mark.parametrize("seqs", [64, 65, 130, 200])
@pytest.mark.parametrize("q_heads,kv_heads,dim,dtype,out", [(4, 2, 64, "bf16", "f32"), (16, 8, 128, "f16", "f16"), (40, 1, 128, "bf16", "bf16")])
def test_prompts_of_many_sequences(ctx, seqs, q_heads, kv_heads, dim, dtype, out):
    """A tile's sequence is looked for among 64 at a time: more of them, empty ones and ones without keys among them."""
    new = [(3, 0, 1, 40, 0, 9, 33)[i % 7] for i in range(seqs)]
    lens = [0 if i % 11 == 3 else n + (i * 5) % 23 for i, n in enumerate(new)]
    paged = Paged(lens, kv_heads, dim, 16, dtype, seed=seqs)
    off = np.concatenate([[0], np.cumsum(new)])
    q = rows_of(int(off[-1]), q_heads, dim, dtype, paged.rng, scale=2.0)
    got = run_prompt(ctx, paged, q, off, q_heads, dim**-0.5, out)
    whose = np.repeat(np.arange(seqs), new)
    limits = [max(0, lens[i] - new[i] + j + 1) for i in range(seqs) for j in range(new[i])]
    check(got, q, limits, lambda r, h: paged.entries(whose[r], limits[r], h), q_heads, kv_heads, dim, dim**-0.5, dtype, out, f"{seqs} prompts")


@pytest.mark.parametrize("q_heads,kv_heads,dim,dtype,out", [(4, 2, 64, "f16", "f32"), (16, 1, 128, "bf16", "bf16")])
def test_step_of_many_groups(ctx, q_heads, kv_heads, dim, dtype, out):
    """More than 64 groups of different prefixes: of several rows, of one, of none; rows outside every group after them."""
    share, lens = [], []
    for g in range(150):
        rows, prefix = (2, 0, 3, 1, 5)[g % 5], 17 + (g * 13) % 120
        share.append((len(lens), len(lens) + rows, prefix))
        lens += [prefix + 1 + (g + i * 7) % 40 for i in range(rows)]
    lens += [0, 77, 300]
    paged = Paged(lens, kv_heads, dim, 16, dtype, seed=9, share=share)
    q = rows_of(len(lens), q_heads, dim, dtype, paged.rng, scale=2.0)
    got = run_step(ctx, paged, q, q_heads, dim**-0.5, out, share=share)
    check(got, q, lens, lambda r, h: paged.entries(r, lens[r], h), q_heads, kv_heads, dim, dim**-0.5, dtype, out, "many groups")


@pytest.mark.parametrize("q_heads,kv_heads,dim,dtype,out", [(8, 2, 128, "bf16", "f32"), (4, 1, 64, "f16", "f16"), (2, 1, 256, "bf16", "bf16")])
def test_step_and_prompt_long_rows(ctx, q_heads, kv_heads, dim, dtype, out):
    lens = [20011, 9000, 1]
    paged = Paged(lens, kv_heads, dim, 32, dtype, "tokens", seed=5)
    q = rows_of(3, q_heads, dim, dtype, paged.rng, scale=2.0)
    for what, got in (("step", run_step(ctx, paged, q, q_heads, dim**-0.5, out)), ("prompt", run_prompt(ctx, paged, q, [0, 1, 2, 3], q_heads, dim**-0.5, out))):
        check(got, q, lens, lambda r, h: paged.entries(r, lens[r], h), q_heads, kv_heads, dim, dim**-0.5, dtype, out, what)


def test_steps_of_two_contexts_at_once(ctx):
    """Two threads, a context, a stream and a workspace each, over one cache: every step has the bits that it has alone."""
    share = [(0, 24, 400)]
    paged = Paged([700 + 11 * i for i in range(24)], 2, 128, 16, "bf16", seed=3, share=share)
    qs = [rows_of(24, 8, 128, "bf16", paged.rng, scale=2.0) for _ in range(2)]
    alone = [run_step(ctx, paged, q, 8, 0.1, "f32", share=share) for q in qs]
    rounds, failed = 20, []

    def work(q, want):
        try:
            with Context(0) as own:
                for i in range(rounds):
                    got = run_step(own, paged, q, 8, 0.1, "f32", share=share)
                    if not np.array_equal(got.view(np.uint32), want.view(np.uint32)):
                        failed.append(i)
        except Exception as e:  # noqa: BLE001 (reported by the test)
            failed.append(e)

    threads = [threading.Thread(target=work, args=x) for x in zip(qs, alone)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not failed and not any(t.is_alive() for t in threads), failed
