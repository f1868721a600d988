"""A batch of sequences through one attention layer on the GPU: the paged cache's operators as a serving program calls them.

The sequences share a voice prompt: it goes through the layer once, its pages are held by every sequence, and each generation step
reads it once for all of them. Then, per sequence, its own prompt (packed, attending to the voice prompt too), and steps: projections
(``head_device``), append with head norms and rotation, attention, output projection, logits, sampling over resident histories and the
embedding of the sampled codes, all on one stream with nothing copied back but the codes.

    python examples/talker_layer.py [rows] [voice tokens] [steps]

A real model has many such layers, each with a cache of its own and the same page table, and norms and a feed-forward part between.
"""
from __future__ import annotations

import os
import sys
import time

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from voxwerk_amd import hip  # noqa: E402
from voxwerk_amd._lib import PARAMS_DTYPE  # noqa: E402
from voxwerk_amd.attention import KvCache, KvPrep, SharedPrefix, rope_frequencies  # noqa: E402
from voxwerk_amd.sampler import Context  # noqa: E402

HIDDEN, Q_HEADS, KV_HEADS, DIM, PAGE, VOCAB = 1024, 16, 8, 128, 16, 2048
WIDTH = (Q_HEADS + 2 * KV_HEADS) * DIM


def to_bf16(x):
    """Bits of a finite fp32 array as bf16, to nearest even."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((b + np.uint32(0x7FFF) + ((b >> np.uint32(16)) & np.uint32(1))) >> np.uint32(16)).astype(np.uint16)


def device(x):
    return hip.DeviceArray.from_numpy(x)


class Pages:
    """Hands out pages; slots of one table."""

    def __init__(self, slots: int, width: int, pages: int):
        self.table = np.zeros((slots, width), np.int32)
        self.free = list(range(pages))[::-1]
        self.held = [0] * slots

    def grow(self, slot: int, tokens: int) -> None:
        while self.held[slot] * PAGE < tokens:
            self.table[slot, self.held[slot]] = self.free.pop()
            self.held[slot] += 1

    def share(self, slot: int, other: int, pages: int) -> None:
        self.table[slot, :pages] = self.table[other, :pages]
        self.held[slot] = pages


class TalkerLayer:
    def __init__(self, ctx: Context, slots: int, max_tokens: int, seed: int = 0):
        r = np.random.default_rng(seed)
        self.ctx, self.slots = ctx, slots
        self.wide = -(-max_tokens // PAGE)
        self.pages = Pages(slots, self.wide, slots * self.wide)
        self.k, self.v = (hip.DeviceArray((slots * self.wide, KV_HEADS, PAGE, DIM), np.uint16) for _ in range(2))
        self.table = device(self.pages.table)
        self.cache = KvCache(self.k, self.v, "bf16", KV_HEADS, DIM, slots * self.wide, PAGE, self.table, slots, self.wide)
        self.w_qkv = device(to_bf16(r.standard_normal((WIDTH, HIDDEN)) * 0.03))
        self.w_out = device(to_bf16(r.standard_normal((HIDDEN, Q_HEADS * DIM)) * 0.02))
        self.w_head = device(to_bf16(r.standard_normal((VOCAB, HIDDEN)) * 0.05))
        self.codes = device(to_bf16(r.standard_normal((VOCAB, HIDDEN))))
        self.norms = [(1 + 0.1 * r.standard_normal(DIM)).astype(np.float32) for _ in range(2)]
        freq, scale = rope_frequencies(DIM, 1e6)
        self.prep = KvPrep(device(self.norms[0]), device(self.norms[1]), 1e-6, device(freq), DIM, rope_scale=scale)

    def _project(self, tokens, x, qkv, q, pos, slots):
        """qkv = W x; queries to q, keys and values to their pages."""
        self.ctx.head_device(tokens, HIDDEN, WIDTH, x, HIDDEN, self.w_qkv, HIDDEN, qkv, WIDTH)
        k = qkv.ptr + 4 * Q_HEADS * DIM
        self.ctx.kv_append_device(tokens, Q_HEADS, qkv, WIDTH, k, WIDTH, k + 4 * KV_HEADS * DIM, WIDTH, "f32", self.cache, pos, slots, q,
                                  Q_HEADS * DIM, prep=self.prep)

    def prompt(self, slots, before, rows):
        """New tokens of the slots, `before` of whose tokens are in the cache: rows[i] fp32 [n, HIDDEN]; returns the layer's
        outputs, packed alike."""
        n, total = [len(x) for x in rows], sum(len(x) for x in rows)
        for s, b, m in zip(slots, before, n):
            self.pages.grow(s, b + m)
        self.table.upload(self.pages.table)
        x = device(np.concatenate(rows).astype(np.float32))
        pos = device(np.concatenate([np.arange(b, b + m) for b, m in zip(before, n)]).astype(np.int32))
        own, whole = device(np.repeat(slots, n).astype(np.int32)), device(np.array(slots, np.int32))
        off, lens = device(np.cumsum([0] + n).astype(np.int32)), device(np.array([b + m for b, m in zip(before, n)], np.int32))
        qkv, q = hip.DeviceArray((total, WIDTH), np.float32), hip.DeviceArray((total, Q_HEADS * DIM), np.uint16)
        att, out = hip.DeviceArray((total, Q_HEADS * DIM), np.float32), hip.DeviceArray((total, HIDDEN), np.float32)
        self._project(total, x, qkv, q, pos, own)
        self.ctx.attn_prompt_device(len(n), total, Q_HEADS, q, Q_HEADS * DIM, self.cache, off, lens, DIM**-0.5, att, Q_HEADS * DIM, "f32",
                                    slots=whole)
        self.ctx.head_device(total, Q_HEADS * DIM, HIDDEN, att, Q_HEADS * DIM, self.w_out, Q_HEADS * DIM, out, HIDDEN)
        self.ctx.synchronize()
        return out

    def generate(self, lens, y, steps, voice=0, share=True):
        """`steps` greedy codes for each of len(lens) sequences (slot r: row r) with lens[r] tokens in the cache, from the last
        outputs y [rows, HIDDEN]; the first `voice` tokens are the same for all. Returns codes [steps, rows] and the last outputs."""
        ctx, rows, most = self.ctx, len(lens), max(lens) + steps
        for s, n in enumerate(lens):
            self.pages.grow(s, n + steps)
        self.table.upload(self.pages.table)
        y, logits, status = device(y), hip.DeviceArray((rows, VOCAB), np.float32), hip.DeviceArray((rows,), np.int32)
        codes = hip.DeviceArray((steps, rows), np.int32)
        x, qkv = hip.DeviceArray((rows, HIDDEN), np.float32), hip.DeviceArray((rows, WIDTH), np.float32)
        q, att = hip.DeviceArray((rows, Q_HEADS * DIM), np.uint16), hip.DeviceArray((rows, Q_HEADS * DIM), np.float32)
        # a step's positions and lengths: known ahead, as every sequence takes one token a step
        pos = device(np.array(lens, np.int32) + np.arange(steps, dtype=np.int32)[:, None])
        have = device(np.array(lens, np.int32) + np.arange(1, steps + 1, dtype=np.int32)[:, None])
        slots = device(np.arange(rows, dtype=np.int32))
        prefix = SharedPrefix(1, device(np.array([0, rows], np.int32)), device(np.array([voice], np.int32)), voice) if share and voice else None
        size = ctx.attn_step_workspace(rows, Q_HEADS, self.cache, most, prefix)
        work = device(np.zeros(max(size, 16), np.uint8))
        greedy = np.zeros(1, PARAMS_DTYPE)
        greedy["rep_penalty"], greedy["keep_id"], greedy["ban_id"] = 1.0, -1, -1
        params = device(greedy.view(np.uint8))
        with ctx.history(rows, steps) as store:
            hip.synchronize()
            began = time.perf_counter()
            for i in range(steps):
                at = 4 * i * rows
                ctx.head_device(rows, HIDDEN, VOCAB, y, HIDDEN, self.w_head, HIDDEN, logits, VOCAB)
                ctx.sample_batch_device(store, rows, VOCAB, logits, VOCAB, slots, params, 0, None, codes.ptr + at, append=True)
                ctx.embed_device(rows, HIDDEN, codes.ptr + at, self.codes, VOCAB, x, HIDDEN, False, status)
                self._project(rows, x, qkv, q, pos.ptr + at, slots)
                ctx.attn_step_device(rows, Q_HEADS, q, Q_HEADS * DIM, self.cache, have.ptr + at, most, DIM**-0.5, att, Q_HEADS * DIM, "f32",
                                     slots=slots, prefix=prefix, workspace=work, workspace_bytes=work.nbytes)
                ctx.head_device(rows, Q_HEADS * DIM, HIDDEN, att, Q_HEADS * DIM, self.w_out, Q_HEADS * DIM, y, HIDDEN)
            ctx.synchronize()
            self.seconds = time.perf_counter() - began
        return codes.numpy(), y.numpy()


def run(ctx: Context, rows: int, voice: int, steps: int, share: bool = True, seed: int = 0):
    """The whole example; returns the layer, the prompts' lengths, all codes and the last outputs."""
    r = np.random.default_rng(seed)
    own = (5 + np.arange(rows) * 7 % 23).tolist()
    layer = TalkerLayer(ctx, rows, voice + max(own) + steps, seed)
    whole = voice // PAGE
    layer.prompt([0], [0], [r.standard_normal((voice, HIDDEN))])  # the voice prompt, once
    rest = r.standard_normal((voice - whole * PAGE, HIDDEN))       # what does not fill a page is each sequence's own
    for s in range(1, rows):
        layer.pages.share(s, 0, whole)
    lens, first = [], []
    texts = [r.standard_normal((n, HIDDEN)) for n in own]
    tails = [x if s == 0 else np.concatenate([rest, x]) for s, x in enumerate(texts)]
    before = [voice if s == 0 else whole * PAGE for s in range(rows)]
    out = layer.prompt(list(range(rows)), before, tails).numpy()
    ends = np.cumsum([len(x) for x in tails])
    for s in range(rows):
        lens.append(before[s] + len(tails[s]))
        first.append(out[ends[s] - 1])
    codes, y = layer.generate(lens, np.stack(first), steps, voice=whole * PAGE, share=share)
    return layer, lens, codes, y


def main() -> None:
    rows, voice, steps = (int(a) for a in (sys.argv[1:] + ["16", "1000", "50"][len(sys.argv) - 1:]))
    with Context(0) as ctx:
        run(ctx, rows, voice, 2)  # (the first call of each kernel loads it)
        for share in (True, False):
            layer, lens, codes, _ = run(ctx, rows, voice, steps, share)
            print(f"{rows} sequences, voice prompt of {voice} tokens {'read once' if share else 'read by each'}: {steps} steps, "
                  f"{1e6 * layer.seconds / steps:.0f} us a step; first codes {codes[0][:6].tolist()}")


if __name__ == "__main__":
    main()
