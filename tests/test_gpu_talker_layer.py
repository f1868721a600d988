"""GPU check of examples/talker_layer.py: projections, append, prompt and step attention, heads, sampling and embedding together."""
from __future__ import annotations

import os
import sys

import numpy as np
import pytest

from oracle import attention_np as on

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,voice,steps", [(3, 70, 6), (1, 40, 3), (20, 300, 4)])
def test_layer(ctx, rows, voice, steps):
    import talker_layer as tl

    layer, lens, codes, y = tl.run(ctx, rows, voice, steps)
    apart, lens2, codes2, y2 = tl.run(ctx, rows, voice, steps, share=False)
    assert lens == lens2 and codes.shape == (steps, rows) and (codes >= 0).all() and (codes < tl.VOCAB).all()
    # the shared prefix and each row by itself sum the same weights in another order (fp32 outputs, fp32 projection)
    same = (codes == codes2).all(0)
    assert np.linalg.norm((y - y2)[same]) <= 1e-4 * np.linalg.norm(y2[same]) and same.mean() > 0.5
    # the last step against the 64-bit oracle over the cache as it is: queries as the append stores them (bf16), outputs within
    # their rounding (2^-8 of an entry) and the attention's own bound, both far below 1 % of the output's norm
    emb = on.widen(layer.codes.numpy())[codes[-1]]
    qkv = emb @ on.widen(layer.w_qkv.numpy()).T
    q = qkv[:, :tl.Q_HEADS * tl.DIM].reshape(rows, tl.Q_HEADS, tl.DIM)
    freq, _ = tl.rope_frequencies(tl.DIM, 1e6)
    pos = np.array(lens) + steps - 1
    q, _ = on.prep_heads(q, layer.norms[0], 1e-6, pos, freq, tl.DIM, False)
    k, v = layer.k.numpy(), layer.v.numpy()
    att = np.zeros((rows, tl.Q_HEADS, tl.DIM))
    g = tl.Q_HEADS // tl.KV_HEADS
    for r in range(rows):
        n = lens[r] + steps
        for h in range(tl.KV_HEADS):
            kk, vv = (on.gather(x, layer.pages.table[r], n, tl.PAGE, h) for x in (k, v))
            att[r, h * g:(h + 1) * g], *_ = on.attend(q[r, h * g:(h + 1) * g], kk, vv, [n] * g, tl.DIM**-0.5)
    want = att.reshape(rows, -1) @ on.widen(layer.w_out.numpy()).T
    assert np.linalg.norm(y - want) <= 0.01 * np.linalg.norm(want)
    # A sequence's tokens as one prompt: the last has the same output. (Its projections are summed in another order than the steps',
    # so that now and then an entry is rounded to another bf16: both are held to the oracle, not to each other.)
    fed = [on.widen(layer.codes.numpy())[codes[:, r]] for r in range(rows)]
    out = layer.prompt(list(range(rows)), lens, fed).numpy().reshape(rows, steps, tl.HIDDEN)
    assert np.linalg.norm(out[:, -1] - want) <= 0.01 * np.linalg.norm(want)
