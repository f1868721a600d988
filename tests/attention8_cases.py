"""Test helpers: paged 8-bit caches filled with poison outside their sequences, and calls checked against the 64-bit oracle."""
from __future__ import annotations

import numpy as np

from oracle import attention8_np as o8
from oracle import attention_np as on
from voxwerk_amd import hip
from voxwerk_amd.attention import Kv8Cache

from attention_cases import as_out, device, out_array, rows_of, run_prompt, run_step  # noqa: F401

POISON = np.array([0x7F, 0xFF, 0x7E, 0xFE], np.uint8)        # NaN and the largest entries
POISON_SCALE = np.array([255, 0, 254, 127], np.uint8)        # NaN, none, the largest


class Paged8:
    """A cache of `slots` sequences of lens[s] tokens in pages of random places, poison elsewhere, in entries and scales.
    order: "heads" ([pages, heads, page, dim]) or "tokens" ([pages, page, heads, dim], in device memory)."""

    def __init__(self, lens, kv_heads, dim, page=16, dtype="bf16", order="heads", seed=0, width=None, share=(), k_scale=1.0, spread=3):
        r = self.rng = np.random.default_rng(seed)
        self.lens, self.kv_heads, self.dim, self.page, self.dtype, self.order = list(lens), kv_heads, dim, page, dtype, order
        need = [-(-n // page) for n in lens]
        self.width = width or max(need + [1])
        self.pages = sum(need) + 3
        places = r.permutation(self.pages).astype(np.int32)
        self.table = np.full((len(lens), self.width), -7, np.int32)  # (entries past the end are no pages)
        shape, blocks = (self.pages, kv_heads, page, dim), (self.pages, kv_heads, page // o8.BLOCK)
        self.k, self.v = r.choice(POISON, size=shape), r.choice(POISON, size=shape)
        self.ks, self.vs = r.choice(POISON_SCALE, size=blocks), r.choice(POISON_SCALE, size=blocks)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = places[at:at + n]
            at += n
        for s, n in enumerate(lens):  # (scales beside those that the entries' sizes call for: any are allowed)
            t = np.arange(n)
            b = np.arange(-(-n // o8.BLOCK))
            for x, xs, loc, size in ((self.k, self.ks, 0.0, k_scale), (self.v, self.vs, 0.25, 1.0)):
                byte = 121 + r.integers(-spread, spread + 1, (len(b), kv_heads))
                xs[self.table[s, b * o8.BLOCK // page], :, b * o8.BLOCK % page // o8.BLOCK] = byte
                y = (r.standard_normal((n, kv_heads, dim)) + loc) * size * 2.0 ** (byte[t // o8.BLOCK] - 121.0)[..., None]
                x[self.table[s, t // page], :, t % page] = o8.encode(np.clip(y / o8.power(byte[t // o8.BLOCK])[..., None], -448, 448))
        for lo, hi, n in share:  # rows [lo, hi) share their first n tokens: whole pages, and a copy of the page with the rest
            whole, rest = n // page, n % page
            for s in range(lo + 1, hi):
                if rest:
                    a, b = self.table[lo, whole], self.table[s, whole]
                    first, blocks = -(-rest // o8.BLOCK) * o8.BLOCK, -(-rest // o8.BLOCK)
                    for x, xs in ((self.k, self.ks), (self.v, self.vs)):
                        old = x[b, :, rest:first].copy()  # a row's own tokens stay, under the block's scale
                        x[b, :, :first], xs[b, :, :blocks] = x[a, :, :first], xs[a, :, :blocks]
                        x[b, :, rest:first] = old
                self.table[s, :whole] = self.table[lo, :whole]
        self.upload()

    def upload(self):
        if self.order == "tokens":
            self.dk, self.dv = (device(np.ascontiguousarray(x.transpose(0, 2, 1, 3))) for x in (self.k, self.v))
            strides = dict(page_stride=self.page * self.kv_heads * self.dim, head_stride=self.dim,
                           token_stride=self.kv_heads * self.dim)
        else:
            self.dk, self.dv, strides = device(self.k), device(self.v), {}
        self.dks, self.dvs, self.dtable = device(self.ks), device(self.vs), device(self.table)
        self.cache = Kv8Cache(self.dk, self.dv, self.dks, self.dvs, self.dtype, self.kv_heads, self.dim, self.pages, self.page,
                              self.dtable, len(self.lens), self.width, **strides)

    def download(self):
        """k, v, k_scale, v_scale as they are now, [pages, heads, page, dim] and [pages, heads, blocks]."""
        k, v = self.dk.numpy(), self.dv.numpy()
        if self.order == "tokens":
            k, v = (x.reshape(self.pages, self.page, self.kv_heads, self.dim).transpose(0, 2, 1, 3) for x in (k, v))
        return k, v, self.dks.numpy(), self.dvs.numpy()

    def entries(self, slot, n, head):
        """The first n keys and values of one slot and head, as the numbers they stand for."""
        if n <= 0:
            return (np.zeros((0, self.dim)),) * 2
        t = np.arange(n)
        p = self.table[slot, t // self.page]
        block = t % self.page // o8.BLOCK
        return tuple(o8.VALUES[x[p, head, t % self.page]] * o8.power(xs[p, head, block])[:, None]
                     for x, xs in ((self.k, self.ks), (self.v, self.vs)))


WEIGHT = {"bf16": 2.0**-8, "f16": 2.0**-16, "f32": 2.0**-24}  # of one, two and three bf16 parts, each rounded by half a step


def bound(out, mean, reach, top, limit, dim, out_dtype):
    """As the 16-bit caches' (oracle/attention_np.py), with weights in as many bf16 parts as the outputs have use for; the factor of
    a key's block is one more rounding of its score, and a value's scale is exact."""
    n = np.maximum(np.asarray(limit, np.float64), 0)
    e = (dim + 3) * 2.0**-24 * reach + top * 2.0**-22 + 2.0**-20
    weight = 2 * e + WEIGHT[out_dtype] + 2 * n * 2.0**-24
    least = {"bf16": 2.0**-133, "f16": 2.0**-24, "f32": 2.0**-149}[out_dtype]
    return (2 * weight)[:, None] * mean + on.UNIT[out_dtype] * np.abs(out) + least


def check(got, q, limits, entries, q_heads, kv_heads, dim, scale, out_dtype, what, bounds=bound):
    """got [rows, q_heads * dim + pad] against the oracle; limits[r]: the keys that row r sees of entries(r, head)."""
    g = q_heads // kv_heads
    got = on.widen(got)[:, :q_heads * dim].reshape(len(q), q_heads, dim)
    qq = on.widen(q)[:, :q_heads * dim].reshape(len(q), q_heads, dim)
    for r, n in enumerate(limits):
        for h in range(kv_heads):
            k, v = entries(r, h)
            rows = slice(h * g, (h + 1) * g)
            out, *stats = on.attend(qq[r, rows], k, v, [n] * g, scale)
            tol = bounds(out, *stats, [n] * g, dim, out_dtype)
            err = np.abs(got[r, rows] - out)
            assert (err <= tol).all(), f"{what}: row {r} of {n} keys, key head {h}: {np.nanmax(err / tol)} of the bound"
            if n <= 0:
                assert not got[r, rows].any(), f"{what}: row {r} sees nothing and is not zero"


def run_cross(ctx, paged, q, q_off, q_heads, scale, out_dtype="f32", kv_len=None, slots=None, ldo_pad=0):
    kv_len = paged.lens if kv_len is None else kv_len
    ldo = q_heads * paged.dim + ldo_pad
    out, dq, do = out_array(len(q), ldo, out_dtype), device(q), device(np.array(q_off, np.int32))
    dl, ds = device(np.array(kv_len, np.int32)), None if slots is None else device(np.array(slots, np.int32))
    hip.synchronize()
    ctx.attn_cross_device(len(q_off) - 1, len(q), q_heads, dq, q.shape[1], paged.cache, do, dl, scale, out, ldo, out_dtype,
                          slots=ds)
    ctx.synchronize()
    return as_out(out.numpy(), out_dtype)
