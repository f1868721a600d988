"""GPU checks of packed attention over an 8-bit cache against the 64-bit oracle where a tile's scales are folded in on its way into LDS: blocks whose
scales are far apart, in each shape of workgroup; of cross attention as a step's rows; and of appends and cross attention at byte offsets past 2^32."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import attention8_np as o8
from voxwerk_amd import hip
from voxwerk_amd.attention import Kv8Cache, KvPrep, rope_frequencies

import attention_cases
from attention_cases import Paged, device, out_array, rows_of, run_prompt, run_step
from attention8_cases import Paged8, check, run_cross

pytestmark = pytest.mark.gpu

# (tokens in the cache, new ones): a table of at most 256 tokens, of more, and of more than 2048: the rule's three shapes of workgroup
SIZES = [(250, 250), (300, 300), (2150, 37)]
TYPES = [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")]


@pytest.mark.parametrize("cross", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("n,new", SIZES)
def test_scales_far_apart(ctx, n, new, dtype, out, dim, cross):
    """Each block and head has scales of its own: keys' from 2^-107 to those of scores of a few, values' over 190 powers of two (fp16 outputs: 24)."""
    paged = Paged8([n], 2, dim, 16, dtype, seed=n + dim)
    r, b = paged.rng, np.arange(-(-n // 16))
    low, high = (108, 132) if out == "f16" else (27, 217)
    paged.ks[paged.table[0, b], :, 0] = np.where(r.random((len(b), 2)) < 0.3, r.integers(20, 110, (len(b), 2)), r.integers(116, 122, (len(b), 2)))
    # a third of the blocks at each end, the others between: a token's largest values come from different blocks along the keys
    paged.vs[paged.table[0, b], :, 0] = np.clip(r.integers(2 * low - high, 2 * high - low, (len(b), 2)), low, high)
    paged.upload()
    q = rows_of(new, 4, dim, dtype, r, scale=2.0)
    scale = dim**-0.5
    got = (run_cross if cross else run_prompt)(ctx, paged, q, [0, new], 4, scale, out)
    limits = [n if cross else n - new + j + 1 for j in range(new)]
    check(got, q, limits, lambda i, h: paged.entries(0, limits[i], h), 4, 2, dim, scale, out, "cross" if cross else "prompt")


@pytest.mark.parametrize("kind", [Paged, Paged8])
@pytest.mark.parametrize("dim,dtype,out", [(64, "f16", "f16"), (128, "bf16", "f32"), (256, "bf16", "bf16")])
def test_few_tokens_over_long_states_as_a_step(ctx, dim, dtype, out, kind):
    """Rows of a step whose groups share all that their sequence has are a cross call: one to several tokens a sequence, states of any length."""
    lens, new = [4001, 700, 0, 33, 2050, 31], [4, 1, 3, 2, 9, 5]
    paged = kind(lens, 2, dim, 16, dtype, seed=dim)
    off, whose = np.concatenate([[0], np.cumsum(new)]), np.repeat(np.arange(len(new)), new)
    q = rows_of(len(whose), 8, dim, dtype, paged.rng, scale=2.0)
    limits = [lens[i] for i in whose]
    got = run_step(ctx, paged, q, 8, dim**-0.5, out, kv_len=limits, slots=whose, share=list(zip(off[:-1], off[1:], lens)))
    args = q, limits, lambda r, h: paged.entries(whose[r], limits[r], h), 8, 2, dim, dim**-0.5
    for y, what in ((got, "step"), (run_cross(ctx, paged, q, off, 8, dim**-0.5, out), "cross")):
        if kind is Paged8:
            check(y, *args, out, what)
        else:
            attention_cases.check(y, *args, dtype, out, what)


def far_pool(paged, far):
    """The pages of paged's one sequence in a pool whose byte offsets pass 2^32, at `far`: the cache, its arrays, and how to read them back."""
    size, blocks = paged.page * paged.kv_heads * paged.dim, paged.kv_heads * (paged.page // o8.BLOCK)
    pages = max(far) + 1
    big = [hip.DeviceArray((pages * n,), np.uint8) for n in (size, size, blocks, blocks)]
    small = paged.dk, paged.dv, paged.dks, paged.dvs

    def copy(back):
        for i, p in enumerate(far):
            for d, s, n in zip(big, small, (size, size, blocks, blocks)):
                there, here = d.ptr + n * p, s.ptr + n * int(paged.table[0, i])
                hip.check(hip.lib().hipMemcpy(here if back else there, there if back else here, n, hip.D2D), "copy")

    copy(False)
    table = device(np.array([far], np.int32))
    return Kv8Cache(*big, paged.dtype, paged.kv_heads, paged.dim, pages, paged.page, table, 1, len(far)), copy


def test_offsets_past_32_bits(ctx):
    page, kv_heads, dim, q_heads = 1024, 8, 128, 16
    pages = (9 << 29) // (page * kv_heads * dim) + 1
    paged = Paged8([2500], kv_heads, dim, page, "bf16", seed=1)
    q = rows_of(40, q_heads, dim, "bf16", paged.rng)
    near, cross = paged.cache, run_cross(ctx, paged, q, [0, 40], q_heads, 0.1, "f32")
    paged.cache, copy = far_pool(paged, [pages - 1, 3, pages - 2])
    assert np.array_equal(run_cross(ctx, paged, q, [0, 40], q_heads, 0.1, "f32"), cross)
    # rows alone in their blocks, and blocks that come whole or in parts: to the far pages first, then to the near ones
    freq, _ = rope_frequencies(dim)
    prep = KvPrep(None, None, 0.0, device(freq), dim)
    start = paged.download()
    for place in (np.array([2500]), np.arange(1000, 1100), np.array([20, 2049, 1500])):
        x = device(rows_of(len(place), q_heads + 2 * kv_heads, dim, "f32", paged.rng, scale=30.0))
        ld, at = (q_heads + 2 * kv_heads) * dim, (x.ptr, x.ptr + 4 * q_heads * dim, x.ptr + 4 * (q_heads + kv_heads) * dim)
        out, places, slots = out_array(len(place), q_heads * dim, "bf16"), device(place.astype(np.int32)), device(np.zeros(len(place), np.int32))
        found = []
        for cache in (paged.cache, near):
            hip.synchronize()
            status = device(np.full(len(place), 9, np.int32))
            ctx.kv_append_device(len(place), q_heads, at[0], ld, at[1], ld, at[2], ld, "f32", cache, places, slots, out, q_heads * dim, prep=prep, status=status)
            ctx.synchronize()
            assert not status.numpy().any()
            if cache is near:
                found.append([y.copy() for y in paged.download()])
            else:  # (what the near pages held comes back after the far ones have been read)
                copy(True)
                found.append([y.copy() for y in paged.download()])
                for d, y in zip((paged.dk, paged.dv, paged.dks, paged.dvs), start):
                    d.upload(y)
        assert all(np.array_equal(a, b) for a, b in zip(*found)), place[:3]
        assert not all(np.array_equal(a, b) for a, b in zip(found[0], start))
        start = found[0]
