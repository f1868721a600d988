"""GPU checks of the bits that softmax weights keep on their way through the second product, from closed forms.

Queries are the first unit vector and keys multiples of it, so that a score is one exact product: one key (the peak) scores `scale`,
all others 0, and scale = x ln 2 gives those the weight 2^-x of the peak's. With n others of value 1 and a peak of value v the output is
(v + n w) / (1 + n w), w = exp(-scale), in every entry."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import attention_np as on

from attention_cases import Paged, run_prompt, run_step

pytestmark = pytest.mark.gpu


def peaked(n, peak_at, peak_value, kv_heads, dim, dtype):
    """A sequence of n + 1 keys, the peak at place peak_at."""
    paged = Paged([n + 1], kv_heads, dim, 64, dtype, seed=n)
    k, v = np.zeros((n + 1, kv_heads, dim)), np.ones((n + 1, kv_heads, dim))
    k[peak_at, :, 0], v[peak_at] = 1.0, peak_value
    t = np.arange(n + 1)
    paged.k[paged.table[0, t // 64], :, t % 64] = on.pack(k, dtype)
    paged.v[paged.table[0, t // 64], :, t % 64] = on.pack(v, dtype)
    paged.upload()
    return paged


def unit_queries(rows, q_heads, dim, dtype):
    q = np.zeros((rows, q_heads, dim))
    q[:, :, 0] = 1.0
    return on.pack(q.reshape(rows, -1), dtype)


def expected(n, seen_peak, value, scale):
    w = np.exp(-np.float64(scale))
    return (seen_peak * value + n * w) / (seen_peak + n * w), n * w / (seen_peak + n * w)


def tolerance(out, share, x, sums, dtype, out_dtype):
    """share: the others' part of the output. A score's exponent x is off by its scale's rounding, the maximum's and its own, (3 x + 8)
    2^-24 together, an exponential by 2^-22 of itself; fp32 outputs keep 22 bits of a weight (fp16: an error of at least 2^-44 of the
    peak's), others the type's, half an ulp off (fp16: at least 2^-32 of the peak's); `sums` roundings of each of both sums."""
    e = (3 * x + 8) * 2.0**-24 + 2.0**-22
    if out_dtype == "f32":
        e += max(2.0**-22, 2.0**(x - 44) if dtype == "f16" else 0.0)
    else:
        e += max(on.UNIT[dtype], 2.0**(x - 32) if dtype == "f16" else 0.0)
    return e * share + 2 * sums * 2.0**-24 * out + on.UNIT[out_dtype] * out + (2.0**-25 if out_dtype == "f16" else 0.0)


# (query heads, key heads, head size, type, outputs)
FORMS = [(2, 1, 128, "f16", "f32"), (2, 1, 128, "f16", "f16"), (4, 1, 64, "f16", "f32"), (1, 1, 256, "f16", "f32"), (8, 2, 64, "f16", "f16"),
         (2, 1, 256, "f16", "f16"), (2, 1, 128, "bf16", "f32")]


@pytest.mark.parametrize("x", [10.3, 12.3, 16.3, 17.4, 20.6, 24.0])
@pytest.mark.parametrize("q_heads,kv_heads,dim,dtype,out", FORMS)
def test_step_long_tail(ctx, q_heads, kv_heads, dim, dtype, out, x):
    """A peak and 65,535 keys far below it, each negligible, together not: as behind an attention sink. The parts of a row are of 512
    keys at most, a wave's tiles a quarter of them, and 256 parts are joined: fewer than 256 roundings of a sum."""
    n, scale = 65535, np.float32(x * np.log(2.0))
    q = unit_queries(1, q_heads, dim, dtype)
    for at, value in ((0, 0.0), (0, 1.0), (n, 0.0), (40000, 0.5)):
        got = on.widen(run_step(ctx, peaked(n, at, value, kv_heads, dim, dtype), q, q_heads, float(scale), out))
        want, share = expected(n, 1, value, scale)
        err = np.abs(got - want).max()
        assert err <= tolerance(want, share, x, 256, dtype, out), f"peak {value} at {at}: {got.min()} to {got.max()}, not {want}: {err}"


@pytest.mark.parametrize("x", [12.3, 16.3, 17.4, 20.6])
@pytest.mark.parametrize("q_heads,kv_heads,dim,dtype,out", FORMS)
def test_prompt_long_tail(ctx, q_heads, kv_heads, dim, dtype, out, x):
    """The same for the last tokens of a prompt of 8192, one wave through all keys, 16 of them a product: fewer than 600 roundings."""
    n, scale = 8191, np.float32(x * np.log(2.0))
    q = unit_queries(3, q_heads, dim, dtype)
    for at, value in ((0, 0.0), (0, 1.0), (n, 0.0)):
        got = on.widen(run_prompt(ctx, peaked(n, at, value, kv_heads, dim, dtype), q, [0, 3], q_heads, float(scale), out))
        for r in range(3):
            seen = n + 1 - 2 + r
            peak = int(at < seen)
            want, share = expected(seen - peak, peak, value, scale)
            err = np.abs(got[r] - want).max()
            assert err <= tolerance(want, share, x, 600, dtype, out), f"peak {value} at {at}, row {r}: {got[r].min()} to {got[r].max()}, not {want}"


@pytest.mark.parametrize("q_heads,kv_heads,dim", [(2, 1, 128), (4, 2, 64), (1, 1, 256), (40, 1, 128)])
def test_weights_of_fp32_outputs_keep_their_bits(ctx, q_heads, kv_heads, dim):
    """All values 1, so every output is 1 whatever the scores are, but for what weights lose on their way to the product: weights near
    (1 + 2^-9 + 0.9 2^-17) / 2 are 7e-6 of themselves off where only two bf16 parts are kept. 33 keys: 33 terms in each sum."""
    w = (1.0 + 2.0**-9 + 0.9 * 2.0**-17) / 2
    scale = float(np.float32(-np.log(w)))
    tol = (2 * 33 + 2) * 2.0**-24
    for at in (0, 32):
        paged = peaked(32, at, 1.0, kv_heads, dim, "bf16")
        step = run_step(ctx, paged, unit_queries(1, q_heads, dim, "bf16"), q_heads, scale, "f32")
        assert np.abs(step - 1.0).max() <= tol
        prompt = run_prompt(ctx, paged, unit_queries(33, q_heads, dim, "bf16"), [0, 33], q_heads, scale, "f32")
        assert np.abs(prompt - 1.0).max() <= tol
