"""Test helpers: paged caches filled with poison outside their sequences, and calls checked against the 64-bit oracle."""
from __future__ import annotations

import numpy as np

from oracle import attention_np as on
from voxwerk_amd import hip
from voxwerk_amd.attention import KvCache, SharedPrefix


def device(a):
    return None if a is None else hip.DeviceArray.from_numpy(a)


def poison(shape, dtype, rng):
    """What pages hold where no sequence reads: NaN, infinities and the type's largest values."""
    odd = np.array([0x7FC0, 0x7F80, 0xFF80, 0x7F7F] if dtype == "bf16" else [0x7E00, 0x7C00, 0xFC00, 0x7BFF], np.uint16)
    x = rng.choice(odd, size=shape)
    return x if dtype == "bf16" else x.view(np.float16)


class Paged:
    """A cache of `slots` sequences of lens[s] tokens in pages of random places, poison elsewhere.
    order: "heads" ([pages, heads, page, dim]) or "tokens" ([pages, page, heads, dim], in device memory)."""

    def __init__(self, lens, kv_heads, dim, page=16, dtype="bf16", order="heads", seed=0, width=None, share=(), k_scale=1.0):
        r = self.rng = np.random.default_rng(seed)
        self.lens, self.kv_heads, self.dim, self.page, self.dtype, self.order = list(lens), kv_heads, dim, page, dtype, order
        need = [-(-n // page) for n in lens]
        self.width = width or max(need + [1])
        self.pages = sum(need) + 3
        places = r.permutation(self.pages).astype(np.int32)
        self.table = np.full((len(lens), self.width), -7, np.int32)  # (entries past the end are no pages)
        self.k = poison((self.pages, kv_heads, page, dim), dtype, r)
        self.v = poison((self.pages, kv_heads, page, dim), dtype, r)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = places[at:at + n]
            at += n
        for s, n in enumerate(lens):
            t = np.arange(n)
            p = self.table[s, t // page]
            self.k[p, :, t % page] = on.pack(r.standard_normal((n, kv_heads, dim)) * k_scale, dtype)
            self.v[p, :, t % page] = on.pack(r.standard_normal((n, kv_heads, dim)) + 0.25, dtype)
        for lo, hi, n in share:  # rows [lo, hi) share their first n tokens: whole pages, and a copy of the rest
            whole, rest = n // page, n % page
            for s in range(lo + 1, hi):
                if rest:
                    a, b = self.table[lo, whole], self.table[s, whole]
                    self.k[b, :, :rest], self.v[b, :, :rest] = self.k[a, :, :rest], self.v[a, :, :rest]
                self.table[s, :whole] = self.table[lo, :whole]
        self.upload()

    def upload(self):
        if self.order == "tokens":
            self.dk, self.dv = (device(np.ascontiguousarray(x.transpose(0, 2, 1, 3))) for x in (self.k, self.v))
            strides = dict(page_stride=self.page * self.kv_heads * self.dim, head_stride=self.dim,
                           token_stride=self.kv_heads * self.dim)
        else:
            self.dk, self.dv, strides = device(self.k), device(self.v), {}
        self.dtable = device(self.table)
        self.cache = KvCache(self.dk, self.dv, self.dtype, self.kv_heads, self.dim, self.pages, self.page, self.dtable,
                             len(self.lens), self.width, **strides)

    def download(self):
        k, v = self.dk.numpy(), self.dv.numpy()
        if self.order == "tokens":
            k, v = (x.reshape(self.pages, self.page, self.kv_heads, self.dim).transpose(0, 2, 1, 3) for x in (k, v))
        return k, v

    def entries(self, slot, n, head):
        return (on.gather(x, self.table[slot], n, self.page, head) for x in (self.k, self.v))


def rows_of(tokens, heads, dim, dtype, rng, pad=0, scale=1.0):
    """[tokens, heads * dim + pad] rows; the pad is poison."""
    x = np.empty((tokens, heads * dim + pad), np.uint16 if dtype == "bf16" else np.float16 if dtype == "f16" else np.float32)
    x[:, :heads * dim] = on.pack(rng.standard_normal((tokens, heads * dim)) * scale, dtype)
    if pad:
        x[:, heads * dim:] = poison((tokens, pad), dtype, rng) if dtype != "f32" else np.nan
    return x


def check(got, q, limits, entries, q_heads, kv_heads, dim, scale, dtype, out_dtype, what):
    """got [rows, q_heads * dim + pad] against the oracle; limits[r]: the keys that row r sees of entries(r, head)."""
    g = q_heads // kv_heads
    got = on.widen(got)[:, :q_heads * dim].reshape(len(q), q_heads, dim)
    qq = on.widen(q)[:, :q_heads * dim].reshape(len(q), q_heads, dim)
    for r, n in enumerate(limits):
        for h in range(kv_heads):
            k, v = entries(r, h)
            rows = slice(h * g, (h + 1) * g)
            out, *stats = on.attend(qq[r, rows], k, v, [n] * g, scale)
            tol = on.bound(out, *stats, [n] * g, dim, dtype, out_dtype)
            err = np.abs(got[r, rows] - out)
            assert (err <= tol).all(), f"{what}: row {r} of {n} keys, key head {h}: {np.nanmax(err / tol)} of the bound"
            if n <= 0:
                assert not got[r, rows].any(), f"{what}: row {r} sees nothing and is not zero"


def out_array(rows, width, out_dtype):
    """Outputs start as a pattern, so that what is not written shows."""
    kind = np.float32 if out_dtype == "f32" else np.uint16
    return device(np.full((rows, width), 7, kind))


def as_out(x, out_dtype):
    return x.view(np.float16) if out_dtype == "f16" else x


def run_step(ctx, paged, q, q_heads, scale, out_dtype="f32", kv_len=None, slots=None, share=(), max_len=None, work="own",
             ldo_pad=0, always=True):
    """One step over `paged`; returns the outputs [rows, q_heads * dim + ldo_pad]."""
    rows = len(q)
    kv_len = paged.lens if kv_len is None else kv_len
    prefix = None
    if share:
        off = [share[0][0]] + [hi for _, hi, _ in share]
        keep = device(np.array(off, np.int32)), device(np.array([n for *_, n in share], np.int32))
        prefix = SharedPrefix(len(share), *keep, max(n for *_, n in share), always)
    ldo = q_heads * paged.dim + ldo_pad
    out, dq = out_array(rows, ldo, out_dtype), device(q)
    max_len = max(max(kv_len, default=0), 0) if max_len is None else max_len
    dl, ds = device(np.array(kv_len, np.int32)), None if slots is None else device(np.array(slots, np.int32))
    n = 0
    if isinstance(work, str):
        n = ctx.attn_step_workspace(rows, q_heads, paged.cache, max_len, prefix)
        work = device(np.zeros(max(n, 16), np.uint8)) if n else None
    elif work is not None:
        n = work.nbytes
    hip.synchronize()
    ctx.attn_step_device(rows, q_heads, dq, q.shape[1], paged.cache, dl, max_len, scale, out, ldo, out_dtype, slots=ds,
                         prefix=prefix, workspace=work, workspace_bytes=n)
    ctx.synchronize()
    return as_out(out.numpy(), out_dtype)


def run_prompt(ctx, paged, q, q_off, q_heads, scale, out_dtype="f32", kv_len=None, slots=None, ldo_pad=0):
    kv_len = paged.lens if kv_len is None else kv_len
    ldo = q_heads * paged.dim + ldo_pad
    out, dq, do = out_array(len(q), ldo, out_dtype), device(q), device(np.array(q_off, np.int32))
    dl, ds = device(np.array(kv_len, np.int32)), None if slots is None else device(np.array(slots, np.int32))
    hip.synchronize()
    ctx.attn_prompt_device(len(q_off) - 1, len(q), q_heads, dq, q.shape[1], paged.cache, do, dl, scale, out, ldo, out_dtype,
                           slots=ds)
    ctx.synchronize()
    return as_out(out.numpy(), out_dtype)
