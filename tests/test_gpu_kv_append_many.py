"""GPU check that a 16-bit append of many tokens, whose rows share workgroups where they are short, leaves the bits that calls of few tokens
leave: input types, head counts and sizes on both sides of the rule, one position a token and three axes, odd numbers of tokens, some of
them outside the cache."""
from __future__ import annotations

import numpy as np
import pytest

from voxwerk_amd import _lib, hip
from voxwerk_amd.attention import KvPrep, RopeAxes, rope_axes, rope_frequencies

from attention_cases import Paged, device, out_array, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("axes", [1, 3])
@pytest.mark.parametrize("tokens", [2047, 2048, 2051, 3301])
@pytest.mark.parametrize("q_heads,kv_heads,dim,in_dtype,dtype", [
    (4, 4, 64, "bf16", "bf16"), (16, 8, 64, "f16", "f16"), (16, 8, 128, "bf16", "bf16"), (6, 2, 256, "bf16", "f16"),
    (64, 8, 64, "bf16", "bf16"), (40, 8, 128, "f16", "bf16"), (4, 4, 64, "f32", "bf16")])
def test_many_tokens_are_few(ctx, q_heads, kv_heads, dim, in_dtype, dtype, tokens, axes):
    r = np.random.default_rng(tokens + dim)
    paged = Paged([tokens + 9, tokens // 2], kv_heads, dim, 16, dtype, seed=dim)
    heads = q_heads + 2 * kv_heads
    x = device(rows_of(tokens, heads, dim, in_dtype, r, scale=1.5))
    size, ld = 4 if in_dtype == "f32" else 2, heads * dim
    weight = device((1 + 0.3 * r.standard_normal(dim)).astype(np.float32))
    freq, _ = rope_frequencies(dim, 1e4)
    prep = KvPrep(weight, weight, 1e-6, device(freq), dim)
    pos = r.integers(0, 1 << 16, (axes, tokens)).astype(np.int32)
    slots = np.zeros(tokens, np.int32)
    slots[r.choice(tokens, 5, replace=False)] = 2  # (there are two)
    place = (9 + np.arange(tokens)).astype(np.int32)
    part = dim // 12
    axis = device(rope_axes([dim // 2 - 2 * part, part, part], True))
    dp, ds, di = device(pos), device(slots), device(place)

    def call(a, n):
        out, status = out_array(n, q_heads * dim, dtype), device(np.full(n, 9, np.int32))
        hip.synchronize()
        at = x.ptr + size * a * ld
        ctx.kv_append_device(n, q_heads, at, ld, at + size * q_heads * dim, ld, at + size * (q_heads + kv_heads) * dim, ld, in_dtype, paged.cache,
                             dp.ptr + 4 * a, ds.ptr + 4 * a, out, q_heads * dim, prep=prep, index=di.ptr + 4 * a, status=status,
                             axes=RopeAxes(axis, 3, tokens) if axes == 3 else None)
        ctx.synchronize()
        return out.numpy(), status.numpy()

    few = [call(a, min(700, tokens - a)) for a in range(0, tokens, 700)]
    kept = [y.view(np.uint16) for y in paged.download()]
    paged.upload()
    q, status = call(0, tokens)
    assert np.array_equal(status, np.concatenate([s for _, s in few])) and (status == np.where(slots == 2, _lib.VXS_ERR_ID_OUT_OF_RANGE, 0)).all()
    assert np.array_equal(q, np.concatenate([y for y, _ in few]))
    assert all(np.array_equal(a, b.view(np.uint16)) for a, b in zip(kept, paged.download()))
