"""GPU check of the 8-bit cache's operators together, as a layer uses them: prompts with positions of three axes are appended and
attended, steps follow (a replayed graph of append and attention), and an encoder's states in a second cache are crossed to. The cache ends
with what its own appends wrote; every result is held to the 64-bit oracle over what the cache stands for."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from oracle import attention_np as on
from voxwerk_amd import hip
from voxwerk_amd.attention import Kv8Cache, KvCache, KvPrep, RopeAxes, rope_axes, rope_frequencies
from voxwerk_amd.sampler import Context

from attention_cases import device, out_array
from attention8_cases import Paged8, check

pytestmark = pytest.mark.gpu

Q, KV, DIM, PAGE = 8, 2, 64, 16
WIDTH = (Q + 2 * KV) * DIM


class Layer:
    """One layer's cache and what goes with it; prompts of `lens`, room for `steps` more tokens each."""

    def __init__(self, lens, steps, bits=8, seed=0):
        self.rng, self.lens, self.bits = np.random.default_rng(seed), list(lens), bits
        self.paged = Paged8([n + steps for n in lens], KV, DIM, PAGE, "bf16", seed=seed)
        if bits == 16:
            zeros = np.zeros(self.paged.k.shape, np.uint16)
            self.k, self.v = device(zeros), device(zeros)
            self.cache = KvCache(self.k, self.v, "bf16", KV, DIM, self.paged.pages, PAGE, self.paged.dtable, len(lens), self.paged.width)
        else:
            self.cache = self.paged.cache
        freq, scale = rope_frequencies(DIM, 1e4)
        self.axis = device(rope_axes([12, 10, 10], interleaved=True))
        w = device((1 + 0.2 * self.rng.standard_normal(DIM)).astype(np.float32))
        self.prep = KvPrep(w, w, 1e-6, device(freq), DIM, False, scale)

    def positions(self, place):
        return np.stack([place, place // 3, place % 7]).astype(np.int32)

    def refresh(self):
        """The host's copy of what the cache holds now."""
        if self.bits == 8:
            self.paged.k, self.paged.v, self.paged.ks, self.paged.vs = self.paged.download()
        else:
            self.host = self.k.numpy(), self.v.numpy()

    def entries(self, slot, n, head):
        if self.bits == 8:
            return self.paged.entries(slot, n, head)
        return tuple(on.gather(x, self.paged.table[slot], n, PAGE, head) for x in self.host)

    def rows(self, tokens):
        return self.rng.standard_normal((tokens, WIDTH)).astype(np.float32)


def append(ctx, layer, x, tokens, pos, slots, place, q_out, status):
    ctx.kv_append_device(tokens, Q, x, WIDTH, x.ptr + 4 * Q * DIM, WIDTH, x.ptr + 4 * (Q + KV) * DIM, WIDTH, "f32", layer.cache, pos, slots,
                         q_out, Q * DIM, prep=layer.prep, index=place, status=status, axes=RopeAxes(layer.axis, 3, tokens))


@pytest.mark.parametrize("bits", [8, 16])
def test_layer(bits):
    lens, steps, lib = [37, 1, 200, 90], 20, hip.lib()
    layer, n = Layer(lens, steps, bits), len(lens)
    stream, graph, run = (ctypes.c_void_p() for _ in range(3))
    hip.check(lib.hipStreamCreateWithFlags(ctypes.byref(stream), 1), "stream")
    with Context(0) as ctx:
        ctx.set_stream(stream.value)  # (all on a stream of the caller's)
        # ---- prompts, packed
        tokens = sum(lens)
        place = np.concatenate([np.arange(a) for a in lens]).astype(np.int32)
        keep = [device(x) for x in (layer.rows(tokens), layer.positions(place), np.repeat(np.arange(n, dtype=np.int32), lens), place)]
        q, status, out = out_array(tokens, Q * DIM, "bf16"), device(np.full(tokens, 9, np.int32)), out_array(tokens, Q * DIM, "bf16")
        off, kv = device(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)), device(np.array(lens, np.int32))
        hip.synchronize()
        append(ctx, layer, keep[0], tokens, keep[1], keep[2], keep[3], q, status)
        ctx.attn_prompt_device(n, tokens, Q, q, Q * DIM, layer.cache, off, kv, DIM**-0.5, out, Q * DIM, "bf16")
        ctx.synchronize()
        assert not status.numpy().any()
        layer.refresh()
        whose = np.repeat(np.arange(n), lens)
        check(out.numpy(), q.numpy(), [int(p) + 1 for p in place], lambda r, h: layer.entries(whose[r], int(place[r]) + 1, h), Q, KV, DIM, DIM**-0.5,
              "bf16", "prompts")
        # ---- steps: append and attention in one graph, replayed with other inputs
        x, place1 = device(layer.rows(n)), device(np.array(lens, np.int32))
        pos, kv1 = device(layer.positions(np.array(lens))), device(np.array(lens, np.int32) + 1)
        q1, out1, status1 = out_array(n, Q * DIM, "bf16"), out_array(n, Q * DIM, "f32"), device(np.full(n, 9, np.int32))
        most = max(lens) + steps
        work = device(np.zeros(max(ctx.attn_step_workspace(n, Q, layer.cache, most), 16), np.uint8))
        hip.synchronize()
        hip.check(lib.hipStreamBeginCapture(stream, 2), "begin")
        append(ctx, layer, x, n, pos, None, place1, q1, status1)
        ctx.attn_step_device(n, Q, q1, Q * DIM, layer.cache, kv1, most, DIM**-0.5, out1, Q * DIM, "f32", workspace=work, workspace_bytes=work.nbytes)
        hip.check(lib.hipStreamEndCapture(stream, ctypes.byref(graph)), "end")
        hip.check(lib.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0), "instantiate")
        for s in range(steps):
            at = np.array(lens, np.int32) + s
            for d, h in ((x, layer.rows(n)), (place1, at), (pos, layer.positions(at)), (kv1, at + 1)):
                d.upload(h)
            hip.synchronize()
            hip.check(lib.hipGraphLaunch(run, stream), "launch")
            hip.check(lib.hipStreamSynchronize(stream), "wait")
            assert not status1.numpy().any()
            if s % 4 == 3 or s == steps - 1:
                layer.refresh()
                check(out1.numpy(), q1.numpy(), (at + 1).tolist(), lambda r, h: layer.entries(r, int(at[r]) + 1, h), Q, KV, DIM, DIM**-0.5,
                      "f32", f"step {s}")
                eager = out_array(n, Q * DIM, "f32")  # the same call by itself
                ctx.attn_step_device(n, Q, q1, Q * DIM, layer.cache, kv1, most, DIM**-0.5, eager, Q * DIM, "f32", workspace=work, workspace_bytes=work.nbytes)
                ctx.synchronize()
                assert np.array_equal(eager.numpy().view(np.uint32), out1.numpy().view(np.uint32))
        # ---- an encoder's states: no norm, no rotation, of other lengths; the last steps' queries cross to them, and are steps over them
        states = [70, 0, 33, 140]
        other = Layer(states, 0, bits, seed=5)
        m = sum(states)
        place2 = np.concatenate([np.arange(a) for a in states]).astype(np.int32)
        y, slots2, place2, status2 = device(other.rows(m)), device(np.repeat(np.arange(n, dtype=np.int32), states)), device(place2), device(np.full(m, 9, np.int32))
        ctx.kv_append_device(m, Q, None, 0, y.ptr + 4 * Q * DIM, WIDTH, y.ptr + 4 * (Q + KV) * DIM, WIDTH, "f32", other.cache, None, slots2, None, 0,
                             index=place2, status=status2)
        out2, kv2, off2 = out_array(n, Q * DIM, "bf16"), device(np.array(states, np.int32)), device(np.arange(n + 1, dtype=np.int32))
        ctx.attn_cross_device(n, n, Q, q1, Q * DIM, other.cache, off2, kv2, DIM**-0.5, out2, Q * DIM, "bf16")
        ctx.synchronize()
        assert not status2.numpy().any()
        other.refresh()
        check(out2.numpy(), q1.numpy(), states, lambda r, h: other.entries(r, states[r], h), Q, KV, DIM, DIM**-0.5, "bf16", "cross")
        ctx.set_stream(None)
    hip.check(lib.hipGraphExecDestroy(run), "destroy")
    hip.check(lib.hipGraphDestroy(graph), "destroy")
    hip.check(lib.hipStreamDestroy(stream), "destroy")


def test_both_caches_agree():
    """The same tokens in 8 and in 16 bits: the queries are the same, and an entry differs by its two roundings at most: half a step of e4m3
    (2^-4 of it, or 2^-10 of its block's scale) and of bf16 (2^-8 of it)."""
    got = []
    for bits in (8, 16):
        layer = Layer([150], 0, bits, seed=3)
        with Context(0) as ctx:
            place = np.arange(150, dtype=np.int32)
            x, p, s = device(layer.rows(150)), device(place), device(np.zeros(150, np.int32))
            q, pos = out_array(150, Q * DIM, "bf16"), device(layer.positions(place))
            hip.synchronize()
            append(ctx, layer, x, 150, pos, s, p, q, None)
            ctx.synchronize()
            layer.refresh()
            got.append((q.numpy(), layer))
    assert np.array_equal(got[0][0], got[1][0])
    small, wide = got[0][1], got[1][1]
    t = np.arange(150)
    for h in range(KV):
        for a, b, scales in zip(small.entries(0, 150, h), wide.entries(0, 150, h), (small.paged.ks, small.paged.vs)):
            scale = 2.0 ** (scales[small.paged.table[0, t // PAGE], h, 0].astype(float) - 127)
            exact = np.abs(b) / (1 - 2.0**-8)  # (at most)
            assert (np.abs(a - b) <= np.maximum(2.0**-4 * exact, 2.0**-10 * scale[:, None]) + 2.0**-8 * exact).all()
