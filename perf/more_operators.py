"""The 8-bit paged cache, positions of several axes and cross attention, as cases that can be timed and checked.

A case is a dict of plain values. Its ``kind`` says which operator one pass goes through, its ``bits`` the cache (8: e4m3
entries with a scale for each block of 16 tokens and key head; 16: entries of ``type``):

``append``  ``Context.kv_append_device``: the projections' queries, keys and values of new tokens, normed head by head and
            rotated, by one position a token or by one of several axes for each frequency; keys and values go to their pages.
``prompt``  ``Context.attn_prompt_device``: causal attention of packed sequences' new tokens over their pages.
``step``    ``Context.attn_step_device``: one token per sequence over its pages, some cases with shared prefixes.
``cross``   ``Context.attn_cross_device``: packed tokens that see all of their sequence's cached states, an encoder's.

``run`` makes these calls where ``own`` is set, else the same in elementary 32-bit torch operations; ``exact`` has them in
64 bits. Query, key and value heads are of 64 to 256 entries, bf16 or fp16; the cache is ``[pages, heads, page_size,
head_dim]``, its scales (E8M0: powers of two) ``[pages, heads, page_size / 16]``.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
BLOCK = 16  # tokens of a scale
HEADS = [(16, 8), (32, 8), (32, 4), (8, 8), (12, 4), (28, 4), (16, 1)]
MAX_SCORES = 32 * 8192 * 8192     # of the largest prompt, whole rectangles
MAX_STEP_ENTRIES = 256 * 3000 * 8 * 128  # keys' entries of the largest step
MAX_APPEND_ENTRIES = 16384 * 32 * 128


def listed():
    return [
        # the next tokens of a serving batch into an 8-bit cache: most join a block that has tokens already
        {"name": "append8_batch", "kind": "append", "bits": 8, "seqs": 256, "new": 1, "start": 4000, "ragged": True, "q_heads": 16,
         "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "in": "bf16", "norm": True, "rot": 128, "axes": 1,
         "interleaved": False, "theta": 1e6},
        # the prompts of a batch into an 8-bit cache, fp32 projections, half of each head rotated in interleaved pairs
        {"name": "append8_prompts", "kind": "append", "bits": 8, "seqs": 24, "new": 1000, "start": 0, "ragged": True, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "type": "f16", "in": "f32", "norm": False, "rot": 64, "axes": 1,
         "interleaved": True, "theta": 1e4},
        # one token among text and video, positions of three axes: latency
        {"name": "append_axes_one", "kind": "append", "bits": 16, "seqs": 1, "new": 1, "start": 700, "ragged": False, "q_heads": 16,
         "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "in": "f32", "norm": True, "rot": 128, "axes": 3,
         "interleaved": False, "theta": 1e6},
        # the patches of four videos
        {"name": "append_axes_video", "kind": "append", "bits": 16, "seqs": 4, "new": 4096, "start": 40, "ragged": True, "q_heads": 16,
         "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "in": "bf16", "norm": True, "rot": 128, "axes": 3,
         "interleaved": False, "theta": 1e6},
        # a few new tokens of each sequence of a batch over its encoder's states
        {"name": "cross_few", "kind": "cross", "bits": 16, "seqs": 24, "new": 4, "context": 1500, "ragged": True, "q_heads": 16,
         "kv_heads": 8, "dim": 64, "page": 16, "type": "f16", "out": "f16", "empty": True},
        # whole targets over their sources, 8-bit states
        {"name": "cross_long", "kind": "cross", "bits": 8, "seqs": 8, "new": 1000, "context": 1500, "ragged": True, "q_heads": 16,
         "kv_heads": 16, "dim": 128, "page": 64, "type": "bf16", "out": "bf16", "empty": False},
        # the prompts of a batch, packed; fp32 outputs for this library's projections
        {"name": "prompt8_packed", "kind": "prompt", "bits": 8, "seqs": 24, "new": 1000, "context": 0, "ragged": True, "q_heads": 16,
         "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "out": "f32", "empty": False},
        # one long prompt, where the matrix cores count
        {"name": "prompt8_long", "kind": "prompt", "bits": 8, "seqs": 1, "new": 8192, "context": 0, "ragged": False, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "type": "bf16", "out": "bf16", "empty": False},
        # a single sequence early in its generation: latency
        {"name": "step8_one", "kind": "step", "bits": 8, "rows": 1, "len": 37, "ragged": False, "prefix": 0, "groups": 0, "q_heads": 16,
         "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "out": "f32", "empty": False},
        # an ordinary batch
        {"name": "step8_batch", "kind": "step", "bits": 8, "rows": 24, "len": 2000, "ragged": True, "prefix": 0, "groups": 0,
         "q_heads": 16, "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "out": "f32", "empty": True},
        # a few long sequences, many query heads to a key head
        {"name": "step8_long", "kind": "step", "bits": 8, "rows": 4, "len": 65000, "ragged": True, "prefix": 0, "groups": 0,
         "q_heads": 32, "kv_heads": 4, "dim": 128, "page": 64, "type": "f16", "out": "f16", "empty": False},
        # a large batch: the cache read at the memory's rate
        {"name": "step8_wide", "kind": "step", "bits": 8, "rows": 256, "len": 3000, "ragged": True, "prefix": 0, "groups": 0,
         "q_heads": 16, "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "out": "bf16", "empty": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    q_heads, kv_heads = rng.choice(HEADS)
    dim, kind = rng.choice([64, 128, 128, 256]), rng.choice(["append", "append", "prompt", "step", "step", "cross"])
    case = {"kind": kind, "bits": 8 if kind in ("prompt", "step") else rng.choice([8, 16]), "ragged": rng.random() < 0.7, "q_heads": q_heads,
            "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 16, 32, 64, 128]), "type": rng.choice(["bf16", "bf16", "f16"])}
    if kind == "append":
        seqs = _log_int(rng, 1, 256)
        most = max(1, MAX_APPEND_ENTRIES // (seqs * q_heads * dim))
        case.update(seqs=seqs, new=rng.choice([1, _log_int(rng, 1, min(most, 16384))]), start=_log_int(rng, 1, 32768),
                    norm=rng.random() < 0.6, rot=rng.choice([dim, dim, dim // 2, 0]), interleaved=rng.random() < 0.4,
                    axes=rng.choice([1, 3]), theta=rng.choice([1e4, 1e6]), **{"in": rng.choice(["f32", case["type"]])})
        if case["bits"] == 16:
            case.update(axes=3, rot=case["rot"] or dim)
        elif not case["rot"]:
            case["axes"] = 1
        return case
    case.update(out=rng.choice([case["type"], case["type"], "f32"]), empty=rng.random() < 0.2)
    if kind != "step":
        new = _log_int(rng, 1, 8192 if kind == "prompt" else 2048)
        context = rng.choice([0, 0, _log_int(rng, 1, 8192)]) if kind == "prompt" else _log_int(rng, 1, 8192)
        keys = new + context if kind == "prompt" else context
        most = max(1, MAX_SCORES // 2 // (q_heads * max(dim, 128) // 128 * new * keys))
        return dict(case, seqs=_log_int(rng, 1, min(most, 64)), new=new, context=context)
    length = _log_int(rng, 1, 65536)
    rows = _log_int(rng, 1, max(1, min(512, MAX_STEP_ENTRIES // (length * kv_heads * dim))))
    case.update(rows=rows, len=length, prefix=0, groups=0)
    if rng.random() < 0.35:
        case.update(groups=rng.randint(1, min(4, rows)), prefix=_log_int(rng, 16, 16384))
        case["rows"] = max(case["groups"], min(rows, MAX_STEP_ENTRIES // ((case["prefix"] + length) * kv_heads * dim)))
        case["len"] = max(1, min(length, MAX_STEP_ENTRIES // (case["rows"] * kv_heads * dim) - case["prefix"]))
    return case


# ---- inputs -----------------------------------------------------------------------------------

_context = None


def _ctx():
    """The one context a program keeps (its stream)."""
    global _context
    if _context is None:
        from voxwerk_amd.sampler import Context

        _context = Context(0)
    return _context


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _spread(n, most, ragged):
    """n lengths from half of `most` up to it, as a batch has them; their sum is the same for every seed."""
    if not ragged or n < 2:
        return [most] * n
    least = min(most, max(1, most // 2))
    return [least + i * (most - least) // (n - 1) for i in range(n)]


def _order(n, seed):
    return torch.randperm(n, generator=torch.Generator().manual_seed(seed)).tolist()


def _pairs(case):
    """(new tokens, tokens before them, or an encoder's states) of each sequence; long ones after short ones."""
    n, before = case["seqs"], case["start"] if case["kind"] == "append" else case["context"]
    return list(zip(_spread(n, case["new"], case["ragged"]), _spread(n, before, case["ragged"])[::-1]))


def _power(byte):
    """2^(byte - 127) of bytes from 1 to 254, exactly."""
    return (byte.to(torch.int32) << 23).view(torch.float32)


def _byte_for(top):
    """The least byte b from 1 whose 448 * 2^(b - 127) is not below `top` >= 0."""
    bits = top.view(torch.int32)  # 448 = 1.75 2^8: exponents' bytes 8 apart, one less where the mantissa is above 1.75's
    return ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).to(torch.int32)).clamp(min=1)


def _entries(shape, loc, case, g):
    """Entries of cached tokens, [pages, heads, page, dim]; some of the heads' channels are larger, as keys' are."""
    x = torch.randn(shape, generator=g, device="cuda").add_(loc)
    x *= torch.rand((shape[1], 1, shape[3]), generator=g, device="cuda").mul_(1.5).add_(0.5)
    if case["bits"] == 16:
        return x.to(TYPES[case["type"]]), None
    blocks = x.view(shape[0], shape[1], -1, BLOCK, shape[3])
    byte = _byte_for(blocks.abs().amax((3, 4)))
    blocks /= _power(byte)[..., None, None]
    return x.to(E4M3), byte.to(torch.uint8).view(E8M0)


def _cache(case, lens, seed, shared=()):
    """Pages for sequences of `lens` tokens, in a random order with some spare, as a cache looks after a while.
    shared: (first row, end row, prefix) of groups whose rows hold the first row's pages for the prefix; the
    page in which it ends, each row's own, holds the same entries."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    page, shape = case["page"], (case["kv_heads"], case["page"], case["dim"])
    need = [-(-n // page) for n in lens]
    width, pages = max(max(need), 1), sum(need) + 4
    order = torch.randperm(pages, generator=g, device="cuda", dtype=torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    (k, ks), (v, vs) = _entries((pages, *shape), 0.0, case, g), _entries((pages, *shape), 0.25, case, g)
    for lo, hi, prefix in shared:
        whole, rest = prefix // page, prefix % page
        table[lo + 1:hi, :whole] = table[lo, :whole]
        if rest and hi - lo > 1:  # (whole blocks: the last of the prefix holds the rows' next tokens too, the same for all)
            for x in (k, v, ks, vs):
                bits = x.view(torch.uint8)
                bits[table[lo + 1:hi, whole].long()] = bits[table[lo, whole].long()].clone()
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs, "table": table, "pages": pages, "width": width}


def _handle(case, s):
    """The cache as the operators take it."""
    if not own:
        return None
    from voxwerk_amd import attention

    sizes = (case["kv_heads"], case["dim"], s["pages"], case["page"], s["table"], s["table"].shape[0], s["width"])
    if case["bits"] == 16:
        return attention.KvCache(s["k"], s["v"], case["type"], *sizes)
    return attention.Kv8Cache(s["k"], s["v"], s["k_scale"], s["v_scale"], case["type"], *sizes)


def _groups(case):
    cut = [round(i * case["rows"] / case["groups"]) for i in range(case["groups"] + 1)]
    return cut, [(a, b, case["prefix"]) for a, b in zip(cut, cut[1:])]


def _axis_of(pairs):
    """Each frequency's axis: height and width take every third one until each has 5/16 of them, time the rest."""
    section = pairs * 5 // 16
    return [i % 3 if i % 3 and i < 3 * section else 0 for i in range(pairs)]


def _positions(case, place, first, count):
    """[axes, tokens]: text advances all axes together; after a quarter of a sequence come frames of 24 x 24 patches."""
    if case["axes"] == 1:
        return place[None].clone()
    text = first + count // 4
    patch = (place - text).clamp(min=0)
    frame, row, column = patch // 576, patch % 576 // 24, patch % 24
    return torch.stack([torch.where(place < text, place, text + x) for x in (frame, row, column)]).to(torch.int32)


def _prepare_append(case, seed, s, g):
    n, hq, hk, d = case["seqs"], case["q_heads"], case["kv_heads"], case["dim"]
    new, start = zip(*(_pairs(case)[i] for i in _order(n, seed)))
    s.update(_cache(case, [a + b for a, b in zip(new, start)], seed))
    tokens = sum(new)
    new, start = _ints(new), _ints(start)
    slots = torch.repeat_interleave(torch.arange(n, device="cuda", dtype=torch.int32), new.long())
    off = torch.cumsum(new, 0) - new
    place = (torch.arange(tokens, device="cuda") - off[slots.long()] + start[slots.long()]).to(torch.int32)
    x = torch.randn((tokens, hq + 2 * hk, d), generator=g, device="cuda").mul_(1.5).to(TYPES[case["in"]])
    s.update(tokens=tokens, x=x, place=place, slots=slots, status=_ints([0] * tokens), q_norm=None, k_norm=None, freq=None,
             axis=None, pos=_positions(case, place, start[slots.long()], new[slots.long()]),
             q=torch.empty((tokens, hq, d), dtype=TYPES[case["type"]], device="cuda"), prep=None, axes=None)
    if case["norm"]:
        s["q_norm"], s["k_norm"] = (1.0 + 0.2 * torch.randn((2, d), generator=g, device="cuda")).unbind(0)
    if case["rot"]:
        i = torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64)
        s["freq"] = (case["theta"] ** (-i / case["rot"])).float()
        s["axis"] = _ints(_axis_of(case["rot"] // 2) if case["axes"] == 3 else [0] * (case["rot"] // 2))
    # the blocks that get tokens: which ones, each token's among them, and whether one begins there
    key = s["table"][slots.long(), place.long() // case["page"]].long() * (case["page"] // BLOCK) + place % case["page"] // BLOCK
    s["blocks"], s["block_of"] = torch.unique(key, return_inverse=True)
    s["fresh"] = torch.zeros(len(s["blocks"]), dtype=torch.bool, device="cuda")
    s["fresh"][s["block_of"][place % BLOCK == 0]] = True
    if own:
        from voxwerk_amd.attention import KvPrep, RopeAxes

        s["prep"] = KvPrep(s["q_norm"], s["k_norm"], 1e-6, s["freq"], case["rot"], case["interleaved"])
        if case["axes"] == 3:
            s["axes"] = RopeAxes(s["axis"], 3, tokens)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    hq, d = case["q_heads"], case["dim"]
    s = {"case": case, "scale": 1.0 / math.sqrt(d)}
    if case["kind"] == "append":
        _prepare_append(case, seed, s, g)
    elif case["kind"] != "step":
        n = case["seqs"]
        new, before = zip(*(_pairs(case)[i] for i in _order(n, seed)))
        kv = [a + b for a, b in zip(new, before)] if case["kind"] == "prompt" else list(before)
        if case["empty"]:  # a prompt whose first tokens see nothing: fewer keys than tokens; a sequence without states
            kv[-1] = new[-1] // 2 if case["kind"] == "prompt" else 0
        s.update(_cache(case, kv, seed))
        tokens = sum(new)
        q_off = [0]
        for a in new:
            q_off.append(q_off[-1] + a)
        s.update(tokens=tokens, q_off=_ints(q_off), kv_len=_ints(kv), max_new=max(new),
                 row=torch.cat([torch.arange(a, device="cuda") + i * max(new) for i, a in enumerate(new)]),  # of padded batches
                 q=torch.randn((tokens, hq, d), generator=g, device="cuda").mul_(2.0).to(TYPES[case["type"]]),
                 out=torch.empty((tokens, hq, d), dtype=TYPES[case["out"]], device="cuda"))
    else:
        n, cut, shared = case["rows"], None, ()
        own_lens = _spread(n, case["len"], case["ragged"])
        kv = [case["prefix"] + own_lens[i] for i in _order(n, seed)]
        if case["empty"] and not case["prefix"]:
            kv[0] = 0
        if case["groups"]:
            cut, shared = _groups(case)
        s.update(_cache(case, kv, seed, shared))
        s.update(kv_len=_ints(kv), max_len=max(kv), prefix=None,
                 q=torch.randn((n, hq, d), generator=g, device="cuda").mul_(2.0).to(TYPES[case["type"]]),
                 out=torch.empty((n, hq, d), dtype=TYPES[case["out"]], device="cuda"))
        if own:
            from voxwerk_amd.attention import SharedPrefix

            if case["groups"]:
                s["prefix"] = SharedPrefix(case["groups"], _ints(cut), _ints([case["prefix"]] * case["groups"]), case["prefix"])
            need = _ctx().attn_step_workspace(n, hq, _handle(case, s), s["max_len"], s["prefix"])
            s["work"] = torch.zeros(max(need, 1), dtype=torch.uint8, device="cuda")
    s["cache"] = _handle(case, s)
    if own:
        _ctx()
    torch.cuda.synchronize()
    return s


# ---- one pass ---------------------------------------------------------------------------------


def run(s):
    case = s["case"]
    if not own:
        return {"append": _plain_append, "prompt": _plain_packed, "cross": _plain_packed, "step": _plain_step}[case["kind"]](case, s)
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "append":
        x, ld = s["x"], (hq + 2 * hk) * d
        _ctx().kv_append_device(s["tokens"], hq, x, ld, x[:, hq:], ld, x[:, hq + hk:], ld, case["in"], s["cache"], s["pos"],
                                s["slots"], s["q"], hq * d, prep=s["prep"], index=s["place"], status=s["status"], axes=s["axes"])
        return _appended(s)
    if case["kind"] == "step":
        _ctx().attn_step_device(case["rows"], hq, s["q"], hq * d, s["cache"], s["kv_len"], s["max_len"], s["scale"],
                                s["out"], hq * d, case["out"], prefix=s["prefix"], workspace=s["work"],
                                workspace_bytes=s["work"].numel())
    else:
        attend = _ctx().attn_prompt_device if case["kind"] == "prompt" else _ctx().attn_cross_device
        attend(case["seqs"], s["tokens"], hq, s["q"], hq * d, s["cache"], s["q_off"], s["kv_len"], s["scale"], s["out"], hq * d,
               case["out"])
    return s["out"]


def _appended(s):
    return {name: s[name] for name in ("q", "k", "v", "k_scale", "v_scale", "status") if s[name] is not None}


# ---- the same in elementary operations, 32 bits ----------------------------------------------------


def _plain_norm(x, weight):
    if weight is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight


def _plain_rotate(x, cos, sin, rot, interleaved):
    """x [tokens, heads, dim]: its first `rot` entries in pairs (i, i + rot/2) or (2i, 2i + 1)."""
    if not rot:
        return x
    half = rot // 2
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :half], x[..., half:rot])
    c, d = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((c, d), -1).flatten(-2) if interleaved else torch.cat((c, d), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _plain_store(case, s, x, cache, scale):
    """x [tokens, heads, dim] to its places in 8 bits: `cache` and its `scale`."""
    hk, d = case["kv_heads"], case["dim"]
    n, block, inside = len(s["blocks"]), s["block_of"], (s["place"] % BLOCK).long()
    where = s["blocks"] // (case["page"] // BLOCK), s["blocks"] % (case["page"] // BLOCK)  # page, and block of the page
    top = torch.zeros((n, hk), device=x.device).scatter_reduce_(0, block[:, None].expand(-1, hk), x.abs().amax(-1), "amax")
    bytes_ = scale.view(torch.uint8)  # [pages, heads, blocks of a page]
    old = bytes_[where[0], :, where[1]].to(torch.int32).masked_fill(s["fresh"][:, None], 1)
    byte = torch.maximum(_byte_for(top), old)
    there = cache.view(torch.uint8).view(s["pages"], hk, -1, BLOCK, d)
    entries = there[where[0], :, where[1]].view(E4M3).float()  # [blocks, heads, 16, dim]
    entries = entries * torch.where(s["fresh"][:, None], 1.0, _power((127 - byte + old).clamp(min=1)))[..., None, None]
    entries[block, :, inside] = x / _power(byte)[block][..., None]
    there[where[0], :, where[1]] = entries.to(E4M3).view(torch.uint8)
    bytes_[where[0], :, where[1]] = byte.to(torch.uint8)


def _plain_append(case, s):
    x, hq, hk = s["x"].float(), case["q_heads"], case["kv_heads"]
    cos = sin = None
    if case["rot"]:
        angle = s["pos"].double()[s["axis"].long()].t()[:, None] * s["freq"].double()
        cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q = _plain_rotate(_plain_norm(x[:, :hq], s["q_norm"]), cos, sin, case["rot"], case["interleaved"])
    k = _plain_rotate(_plain_norm(x[:, hq:hq + hk], s["k_norm"]), cos, sin, case["rot"], case["interleaved"])
    v = x[:, hq + hk:]
    if case["bits"] == 8:
        _plain_store(case, s, k, s["k"], s["k_scale"])
        _plain_store(case, s, v, s["v"], s["v_scale"])
    else:
        place = s["place"].long()
        page = s["table"][s["slots"].long(), place // case["page"]].long()
        s["k"][page, :, place % case["page"]] = k.to(s["k"].dtype)
        s["v"][page, :, place % case["page"]] = v.to(s["v"].dtype)
    s["q"].copy_(q)
    return _appended(s)


def _gather(x, scale, table):
    """Pages [pages, heads, page, dim] as [sequences, heads, tokens, dim] in 32 bits."""
    at = table.long().clamp(min=0)
    if scale is None:
        y = x[at].float()
    else:
        y = x.view(torch.uint8)[at].view(E4M3).float()
        y = (y.unflatten(3, (-1, BLOCK)).mul_(_power(scale.view(torch.uint8)[at])[..., None, None])).flatten(3, 4)
    return y.transpose(1, 2).flatten(2, 3)


def _attend(q, k, v, seen, scale):
    """softmax(scale q k^T) v over the keys that `seen` tells; zeros for a row that sees none."""
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / total.masked_fill(total == 0, 1.0)


def _plain_packed(case, s):
    n, hk, d, new = case["seqs"], case["kv_heads"], case["dim"], s["max_new"]
    g = case["q_heads"] // hk
    k, v = _gather(s["k"], s["k_scale"], s["table"]), _gather(s["v"], s["v_scale"], s["table"])
    off, lens = s["q_off"].long(), s["kv_len"].long()
    count = off[1:] - off[:-1]
    i = torch.arange(new, device=k.device)
    there = i < count[:, None]                              # [sequences, new]
    at = (off[:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"][at].float().reshape(n, new, hk, g, d).permute(0, 2, 3, 1, 4).reshape(n, hk, g * new, d)
    # the last key that a token sees
    last = (lens - count)[:, None] + i if case["kind"] == "prompt" else (lens - 1)[:, None].expand(n, new)
    j = torch.arange(k.shape[2], device=k.device)
    seen = ((j <= last[..., None]) & there[..., None])[:, None, None].expand(n, 1, g, new, -1).reshape(n, 1, g * new, -1)
    o = _attend(q, k, v, seen, s["scale"]).reshape(n, hk, g, new, d).permute(0, 3, 1, 2, 4).reshape(n, new, hk * g, d)
    s["out"].copy_(o.flatten(0, 1)[s["row"]])
    return s["out"]


def _plain_step(case, s):
    n, hk, d = case["rows"], case["kv_heads"], case["dim"]
    k, v = _gather(s["k"], s["k_scale"], s["table"]), _gather(s["v"], s["v_scale"], s["table"])
    seen = torch.arange(k.shape[2], device=k.device) < s["kv_len"][:, None, None, None]
    q = s["q"].float().reshape(n, hk, -1, d)
    s["out"].copy_(_attend(q, k, v, seen, s["scale"]).reshape(n, -1, d))
    return s["out"]


# ---- what a pass cannot do without ---------------------------------------------------------------


def work(case):
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    size = {"f32": 4, "bf16": 2, "f16": 2}
    entry = 2.0 if case["bits"] == 16 else 1.0 + 1.0 / (BLOCK * d)
    if case["kind"] == "append":
        tokens = sum(new for new, _ in _pairs(case))
        return {"bytes": tokens * (hq * d * (size[case["in"]] + 2) + 2 * hk * d * (size[case["in"]] + entry) + 12 + 4 * case["axes"]),
                "flops": tokens * (hq + hk) * d * 7}
    out = 2 + size[case["out"]]
    if case["kind"] != "step":
        pairs = [(new, new + before if case["kind"] == "prompt" else before) for new, before in _pairs(case)]
        tokens = sum(new for new, _ in pairs)
        keys = sum(n for _, n in pairs)
        seen = sum(new * n - (new * (new - 1) / 2 if case["kind"] == "prompt" else 0) for new, n in pairs)
        return {"bytes": keys * hk * d * 2 * entry + tokens * hq * d * out, "flops": 4 * d * hq * seen}
    lens = sum(_spread(case["rows"], case["len"], case["ragged"]))
    return {"bytes": (case["groups"] * case["prefix"] + lens) * hk * d * 2 * entry + case["rows"] * hq * d * out,
            "flops": 4 * d * hq * (case["rows"] * case["prefix"] + lens)}


# ---- the same from the definition, 64 bits ---------------------------------------------------------


def _exact_block(case, s, x, cache, scale):
    """Entries over their scales, and scales, after x [tokens, heads, dim] has gone to its places: not rounded to 8 bits."""
    shape = (s["pages"], case["kv_heads"], case["page"] // BLOCK)
    held = cache.double().view(*shape, BLOCK, case["dim"])
    old = scale.double()
    held *= old[..., None, None]
    place = s["place"].long()
    page = s["table"].long()[s["slots"].long(), place // case["page"]]
    block = place % case["page"] // BLOCK
    touched, top = torch.zeros(shape, dtype=torch.bool, device=x.device), torch.zeros(shape, dtype=torch.float64, device=x.device)
    new = old.clone()
    begins = place % BLOCK == 0
    new[page[begins], :, block[begins]] = 0.0
    touched[page, :, block] = True
    height = x.abs().amax(-1)
    for i in range(BLOCK):  # tokens of one place in a block are in different blocks
        at = place % BLOCK == i
        top[page[at], :, block[at]] = torch.maximum(top[page[at], :, block[at]], height[at])
        held[page[at], :, block[at], i] = x[at]
    least = torch.exp2(torch.ceil(torch.log2(top / 448.0)).clamp(min=-126.0))
    new = torch.where(touched, torch.maximum(new, least), old)
    held /= new[..., None, None]
    # what a block held before a token began it anew counts for nothing, and keeps its bits
    begun = torch.zeros(shape, dtype=torch.bool, device=x.device)
    begun[page[begins], :, block[begins]] = True
    written = torch.zeros((*shape, BLOCK), dtype=torch.bool, device=x.device)
    written[page, :, block, place % BLOCK] = True
    keep = (begun[..., None] & ~written)[..., None]
    return torch.where(keep, cache.double().view(held.shape), held).view(cache.shape), new


def _exact_append(case, s):
    hq, hk, rot = case["q_heads"], case["kv_heads"], case["rot"]
    x = s["x"].double()
    heads = x[:, :hq + hk].clone()
    if case["norm"]:
        heads /= torch.sqrt(heads.pow(2).sum(-1, keepdim=True) / case["dim"] + 1e-6)
        heads[:, :hq] *= s["q_norm"].double()
        heads[:, hq:] *= s["k_norm"].double()
    if rot:
        by = torch.stack([s["pos"][a] for a in s["axis"].tolist()], 1).double()
        turn = torch.polar(torch.ones_like(by), by * s["freq"].double())[:, None]
        first = torch.arange(0, rot, 2, device="cuda") if case["interleaved"] else torch.arange(rot // 2, device="cuda")
        second = first + (1 if case["interleaved"] else rot // 2)
        z = torch.complex(heads[..., first], heads[..., second]) * turn
        heads[..., first], heads[..., second] = z.real, z.imag
    found = {"q": heads[:, :hq], "status": torch.zeros_like(s["status"])}
    if case["bits"] == 8:
        for name, y in (("k", heads[:, hq:]), ("v", x[:, hq + hk:])):
            found[name], found[name + "_scale"] = _exact_block(case, s, y, s[name], s[name + "_scale"])
        return found
    place = s["place"].long()
    page = s["table"].long()[s["slots"].long(), place // case["page"]]
    for name, y in (("k", heads[:, hq:]), ("v", x[:, hq + hk:])):
        found[name] = s[name].double()
        found[name][page, :, place % case["page"]] = y
    return found


def _exact_rows(q, k, v, limit, scale):
    """q [rows, dim] of one head over k, v [keys, dim]; row i sees the first limit[i] keys."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for a in range(0, len(q), 2048):
        part = q[a:a + 2048] @ k.t() * scale
        hidden = torch.arange(len(k), device=q.device)[None] >= limit[a:a + 2048, None]
        got = torch.softmax(part.masked_fill(hidden, -math.inf), 1) @ v
        out[a:a + 2048] = torch.where((limit[a:a + 2048] > 0)[:, None], got, torch.zeros_like(got))
    return out


def _exact_head(s, name, pages, h, n):
    """The first n entries of one head of a sequence."""
    x = s[name].view(torch.uint8)[pages, h].view(s[name].dtype).double()  # [pages, page, dim]
    if s[name + "_scale"] is not None:
        x = x.unflatten(1, (-1, BLOCK)) * s[name + "_scale"].double()[pages, h][..., None, None]
    return x.reshape(-1, x.shape[-1])[:n]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(case, s)
    hk, page = case["kv_heads"], case["page"]
    g = case["q_heads"] // hk
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    lens = s["kv_len"].tolist()
    off = list(range(case["rows"] + 1)) if case["kind"] == "step" else s["q_off"].tolist()
    for i, n in enumerate(lens):
        a, b = off[i], off[i + 1]
        if not n:
            continue
        pages = s["table"][i, :-(-n // page)].long()
        if case["kind"] == "cross":
            limit = torch.full((b - a,), n, device="cuda")
        else:
            limit = (n - (b - a) + 1 + torch.arange(b - a, device="cuda")).clamp(min=0)
        for h in range(hk):
            k, v = _exact_head(s, "k", pages, h, n), _exact_head(s, "v", pages, h, n)
            q = s["q"][a:b, h * g:(h + 1) * g].double().reshape(-1, case["dim"])
            got = _exact_rows(q, k, v, limit.repeat_interleave(g), s["scale"])
            out[a:b, h * g:(h + 1) * g] = got.reshape(b - a, g, -1)
    return out
