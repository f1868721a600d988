"""The attention work of a generation step around the sampler, as cases that can be timed and checked.

A case is a dict of plain values. Its ``kind`` says which operator one pass goes through:

``append``  ``Context.kv_append_device``: the projections' queries, keys and values of new tokens, normed head
            by head and rotated to their positions; keys and values go to their pages of the cache.
``prompt``  ``Context.attn_prompt_device``: causal attention of packed sequences' new tokens over their pages.
``step``    ``Context.attn_step_device``: one token per sequence over its pages, some cases with a prefix that
            groups of sequences share.

``run`` makes these calls where ``own`` is set, else the same in elementary 32-bit torch operations;
``exact`` has them in 64 bits. Query, key and value heads are of 64 to 256 entries, bf16 or fp16; the cache
is ``[pages, heads, page_size, head_dim]``.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HEADS = [(16, 8), (32, 8), (32, 4), (8, 8), (12, 4), (28, 4), (16, 1)]
MAX_SCORES = 32 * 8192 * 8192     # of the largest prompt, whole rectangles
MAX_STEP_ENTRIES = 256 * 3000 * 8 * 128  # keys' entries of the largest step
MAX_APPEND_ENTRIES = 16384 * 32 * 128


def listed():
    return [
        # a single sequence's next token, where only latency counts; the projections of this library give fp32
        {"name": "append_one", "kind": "append", "seqs": 1, "new": 1, "start": 700, "ragged": False, "q_heads": 16,
         "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "in": "f32", "norm": True, "rot": 128,
         "interleaved": False, "theta": 1e6},
        # the next tokens of a serving batch
        {"name": "append_batch", "kind": "append", "seqs": 256, "new": 1, "start": 4000, "ragged": True, "q_heads": 16,
         "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "in": "bf16", "norm": True, "rot": 128,
         "interleaved": False, "theta": 1e6},
        # the prompts of a batch, half of each head rotated in interleaved pairs, no norms
        {"name": "append_prompts", "kind": "append", "seqs": 24, "new": 1000, "start": 0, "ragged": True, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "type": "f16", "in": "f32", "norm": False, "rot": 64,
         "interleaved": True, "theta": 1e4},
        # one short prompt: latency
        {"name": "prompt_short", "kind": "prompt", "seqs": 1, "new": 93, "context": 0, "ragged": False, "q_heads": 16,
         "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "out": "bf16", "empty": False},
        # the prompts of a batch, packed; fp32 outputs for this library's projections
        {"name": "prompt_packed", "kind": "prompt", "seqs": 24, "new": 1000, "context": 0, "ragged": True, "q_heads": 16,
         "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "out": "f32", "empty": False},
        # new turns on long cached contexts
        {"name": "prompt_resumed", "kind": "prompt", "seqs": 4, "new": 130, "context": 8000, "ragged": True, "q_heads": 32,
         "kv_heads": 4, "dim": 64, "page": 64, "type": "f16", "out": "f16", "empty": True},
        # one long prompt, where the matrix cores count
        {"name": "prompt_long", "kind": "prompt", "seqs": 1, "new": 8192, "context": 0, "ragged": False, "q_heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "type": "bf16", "out": "bf16", "empty": False},
        # a single sequence early in its generation: latency
        {"name": "step_one", "kind": "step", "rows": 1, "len": 37, "ragged": False, "prefix": 0, "groups": 0, "q_heads": 16,
         "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "out": "f32", "empty": False},
        # an ordinary batch
        {"name": "step_batch", "kind": "step", "rows": 24, "len": 2000, "ragged": True, "prefix": 0, "groups": 0,
         "q_heads": 16, "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "out": "f32", "empty": True},
        # a few long sequences, many query heads to a key head
        {"name": "step_long", "kind": "step", "rows": 4, "len": 65000, "ragged": True, "prefix": 0, "groups": 0,
         "q_heads": 32, "kv_heads": 4, "dim": 128, "page": 64, "type": "f16", "out": "f16", "empty": False},
        # a large batch: the cache read at the memory's rate
        {"name": "step_wide", "kind": "step", "rows": 256, "len": 3000, "ragged": True, "prefix": 0, "groups": 0,
         "q_heads": 16, "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "out": "bf16", "empty": False},
        # a batch in which two voices' long prompts are each shared by half of the sequences
        {"name": "step_shared", "kind": "step", "rows": 96, "len": 300, "ragged": True, "prefix": 4100, "groups": 2,
         "q_heads": 16, "kv_heads": 8, "dim": 128, "page": 16, "type": "bf16", "out": "bf16", "empty": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    q_heads, kv_heads = rng.choice(HEADS)
    dim, ragged = rng.choice([64, 128, 128, 256]), rng.random() < 0.7
    case = {"kind": rng.choice(["append", "prompt", "step", "step"]), "ragged": ragged, "q_heads": q_heads,
            "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 16, 32, 64, 128]), "type": rng.choice(["bf16", "bf16", "f16"])}
    if case["kind"] == "append":
        seqs = _log_int(rng, 1, 256)
        most = max(1, MAX_APPEND_ENTRIES // (seqs * q_heads * dim))
        return dict(case, seqs=seqs, new=rng.choice([1, _log_int(rng, 1, min(most, 16384))]), start=_log_int(rng, 1, 32768),
                    norm=rng.random() < 0.6, rot=rng.choice([dim, dim, dim // 2, 0]), interleaved=rng.random() < 0.4,
                    theta=rng.choice([1e4, 1e6]), **{"in": rng.choice(["f32", "bf16" if case["type"] == "bf16" else "f16"])})
    case.update(out=rng.choice([case["type"], case["type"], "f32"]), empty=rng.random() < 0.2)
    if case["kind"] == "prompt":
        new = _log_int(rng, 1, 8192)
        context = rng.choice([0, 0, _log_int(rng, 1, 8192)])
        most = max(1, MAX_SCORES // 2 // (q_heads * max(dim, 128) // 128 * new * (new + context)))
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
    """(new tokens, tokens before them) of each sequence of an append or a prompt; long ones after short ones."""
    n, before = case["seqs"], case["start"] if case["kind"] == "append" else case["context"]
    return list(zip(_spread(n, case["new"], case["ragged"]), _spread(n, before, case["ragged"])[::-1]))


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
    kind = TYPES[case["type"]]
    k = torch.randn((pages, *shape), generator=g, device="cuda").to(kind)
    v = torch.randn((pages, *shape), generator=g, device="cuda").add_(0.25).to(kind)
    for lo, hi, prefix in shared:
        whole, rest = prefix // page, prefix % page
        table[lo + 1:hi, :whole] = table[lo, :whole]
        if rest and hi - lo > 1:
            for x in (k, v):
                x[table[lo + 1:hi, whole].long(), :, :rest] = x[table[lo, whole].long(), :, :rest]
    return {"k": k, "v": v, "table": table, "pages": pages, "width": width}


def _handle(case, s):
    """The cache as the operators take it."""
    if not own:
        return None
    from voxwerk_amd.attention import KvCache

    return KvCache(s["k"], s["v"], case["type"], case["kv_heads"], case["dim"], s["pages"], case["page"], s["table"],
                   s["table"].shape[0], s["width"])


def _groups(case):
    cut = [round(i * case["rows"] / case["groups"]) for i in range(case["groups"] + 1)]
    return cut, [(a, b, case["prefix"]) for a, b in zip(cut, cut[1:])]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    s = {"case": case, "scale": 1.0 / math.sqrt(d)}
    if case["kind"] == "append":
        n = case["seqs"]
        new, start = zip(*(_pairs(case)[i] for i in _order(n, seed)))
        s.update(_cache(case, [a + b for a, b in zip(new, start)], seed))
        tokens = sum(new)
        new, start = _ints(new), _ints(start)
        slots = torch.repeat_interleave(torch.arange(n, device="cuda", dtype=torch.int32), new.long())
        off = torch.cumsum(new, 0) - new
        pos = (torch.arange(tokens, device="cuda") - off[slots.long()] + start[slots.long()]).to(torch.int32)
        x = torch.randn((tokens, hq + 2 * hk, d), generator=g, device="cuda").mul_(1.5).to(TYPES[case["in"]])
        s.update(tokens=tokens, x=x, pos=pos, slots=slots, status=_ints([0] * tokens), q_norm=None, k_norm=None, freq=None,
                 q=torch.empty((tokens, hq, d), dtype=TYPES[case["type"]], device="cuda"))
        if case["norm"]:
            s["q_norm"], s["k_norm"] = (1.0 + 0.2 * torch.randn((2, d), generator=g, device="cuda")).unbind(0)
        if case["rot"]:
            i = torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64)
            s["freq"] = (case["theta"] ** (-i / case["rot"])).float()
        if own:
            from voxwerk_amd.attention import KvPrep

            s["prep"] = KvPrep(s["q_norm"], s["k_norm"], 1e-6, s["freq"], case["rot"], case["interleaved"])
    elif case["kind"] == "prompt":
        n = case["seqs"]
        new, before = zip(*(_pairs(case)[i] for i in _order(n, seed)))
        kv = [a + b for a, b in zip(new, before)]
        if case["empty"]:  # a sequence whose first tokens see nothing: fewer keys than tokens
            kv[-1] = new[-1] // 2
        s.update(_cache(case, kv, seed))
        tokens = sum(new)
        q_off = [0]
        for a in new:
            q_off.append(q_off[-1] + a)
        s.update(tokens=tokens, q_off=_ints(q_off), kv_len=_ints(kv), max_new=max(new),
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
        return {"append": _plain_append, "prompt": _plain_prompt, "step": _plain_step}[case["kind"]](case, s)
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "append":
        x, ld = s["x"], (hq + 2 * hk) * d
        _ctx().kv_append_device(s["tokens"], hq, x, ld, x[:, hq:], ld, x[:, hq + hk:], ld, case["in"], s["cache"], s["pos"],
                                s["slots"], s["q"], hq * d, prep=s["prep"], status=s["status"])
        return {"q": s["q"], "k": s["k"], "v": s["v"], "status": s["status"]}
    if case["kind"] == "prompt":
        _ctx().attn_prompt_device(case["seqs"], s["tokens"], hq, s["q"], hq * d, s["cache"], s["q_off"], s["kv_len"],
                                  s["scale"], s["out"], hq * d, case["out"])
    else:
        _ctx().attn_step_device(case["rows"], hq, s["q"], hq * d, s["cache"], s["kv_len"], s["max_len"], s["scale"],
                                s["out"], hq * d, case["out"], prefix=s["prefix"], workspace=s["work"],
                                workspace_bytes=s["work"].numel())
    return s["out"]


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


def _plain_append(case, s):
    x, hq, hk = s["x"].float(), case["q_heads"], case["kv_heads"]
    cos = sin = None
    if case["rot"]:
        angle = s["pos"].float()[:, None, None] * s["freq"]
        cos, sin = torch.cos(angle), torch.sin(angle)
    q = _plain_rotate(_plain_norm(x[:, :hq], s["q_norm"]), cos, sin, case["rot"], case["interleaved"])
    k = _plain_rotate(_plain_norm(x[:, hq:hq + hk], s["k_norm"]), cos, sin, case["rot"], case["interleaved"])
    pos = s["pos"].long()
    page = s["table"][s["slots"].long(), pos // case["page"]].long()
    s["k"][page, :, pos % case["page"]] = k.to(s["k"].dtype)
    s["v"][page, :, pos % case["page"]] = x[:, hq + hk:].to(s["v"].dtype)
    s["q"].copy_(q)
    return {"q": s["q"], "k": s["k"], "v": s["v"], "status": s["status"]}


def _gather(x, table, kind):
    """Pages [pages, heads, page, dim] as [sequences, heads, tokens, dim]."""
    y = x[table.long().clamp(min=0)].to(kind)
    return y.transpose(1, 2).flatten(2, 3)


def _attend(q, k, v, seen, scale):
    """softmax(scale q k^T) v over the keys that `seen` tells; zeros for a row that sees none."""
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / total.masked_fill(total == 0, 1.0)


def _plain_prompt(case, s):
    n, hk, d, new = case["seqs"], case["kv_heads"], case["dim"], s["max_new"]
    g = case["q_heads"] // hk
    k, v = _gather(s["k"], s["table"], torch.float32), _gather(s["v"], s["table"], torch.float32)
    off, lens = s["q_off"].long(), s["kv_len"].long()
    count = off[1:] - off[:-1]
    i = torch.arange(new, device=k.device)
    there = i < count[:, None]                              # [sequences, new]
    at = (off[:-1, None] + i).clamp(max=s["tokens"] - 1)
    q = s["q"][at].float().reshape(n, new, hk, g, d).permute(0, 2, 3, 1, 4).reshape(n, hk, g * new, d)
    last = (lens - count)[:, None] + i                      # the last key that a token sees
    j = torch.arange(k.shape[2], device=k.device)
    seen = ((j <= last[..., None]) & there[..., None])[:, None, None].expand(n, 1, g, new, -1).reshape(n, 1, g * new, -1)
    o = _attend(q, k, v, seen, s["scale"]).reshape(n, hk, g, new, d).permute(0, 3, 1, 2, 4).reshape(n, new, hk * g, d)
    s["out"].copy_(o[there])
    return s["out"]


def _plain_step(case, s):
    n, hk, d = case["rows"], case["kv_heads"], case["dim"]
    k, v = _gather(s["k"], s["table"], torch.float32), _gather(s["v"], s["table"], torch.float32)
    seen = torch.arange(k.shape[2], device=k.device) < s["kv_len"][:, None, None, None]
    q = s["q"].float().reshape(n, hk, -1, d)
    s["out"].copy_(_attend(q, k, v, seen, s["scale"]).reshape(n, -1, d))
    return s["out"]


# ---- what a pass cannot do without ---------------------------------------------------------------


def work(case):
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if case["kind"] == "append":
        tokens = sum(new for new, _ in _pairs(case))
        entries = tokens * (hq + 2 * hk) * d
        return {"bytes": entries * (size[case["in"]] + 2) + 12 * tokens, "flops": tokens * (hq + hk) * d * 7}
    out = 2 + size[case["out"]]
    if case["kind"] == "prompt":
        keys = sum(new + before for new, before in _pairs(case))
        tokens = sum(new for new, _ in _pairs(case))
        seen = sum(new * before + new * (new + 1) / 2 for new, before in _pairs(case))
        return {"bytes": keys * hk * d * 4 + tokens * hq * d * out, "flops": 4 * d * hq * seen}
    lens = sum(_spread(case["rows"], case["len"], case["ragged"]))
    return {"bytes": (case["groups"] * case["prefix"] + lens) * hk * d * 4 + case["rows"] * hq * d * out,
            "flops": 4 * d * hq * (case["rows"] * case["prefix"] + lens)}


# ---- the same from the definition, 64 bits ---------------------------------------------------------


def _exact_append(case, s):
    hq, hk, d, rot = case["q_heads"], case["kv_heads"], case["dim"], case["rot"]
    x = s["x"].double()
    heads = x[:, :hq + hk].clone()
    if case["norm"]:
        heads /= torch.sqrt(heads.pow(2).sum(-1, keepdim=True) / d + 1e-6)
        heads[:, :hq] *= s["q_norm"].double()
        heads[:, hq:] *= s["k_norm"].double()
    if rot:
        turn = torch.polar(torch.ones((s["tokens"], rot // 2), dtype=torch.float64, device="cuda"),
                           s["pos"].double()[:, None] * s["freq"].double())[:, None]
        first = torch.arange(0, rot, 2, device="cuda") if case["interleaved"] else torch.arange(rot // 2, device="cuda")
        second = first + (1 if case["interleaved"] else rot // 2)
        z = torch.complex(heads[..., first], heads[..., second]) * turn
        heads[..., first], heads[..., second] = z.real, z.imag
    k, v = s["k"].double(), s["v"].double()
    place, pos = s["slots"].tolist(), s["pos"].tolist()
    table = s["table"].cpu()
    page = torch.tensor([int(table[r, p // case["page"]]) for r, p in zip(place, pos)], device="cuda")
    inside = torch.tensor([p % case["page"] for p in pos], device="cuda")
    for h in range(hk):
        k[page, h, inside] = heads[:, hq + h]
        v[page, h, inside] = x[:, hq + hk + h]
    return {"q": heads[:, :hq], "k": k, "v": v, "status": torch.zeros_like(s["status"])}


def _exact_rows(q, k, v, limit, scale):
    """q [rows, dim] of one head over k, v [keys, dim]; row i sees the first limit[i] keys."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for a in range(0, len(q), 2048):
        part = q[a:a + 2048] @ k.t() * scale
        hidden = torch.arange(len(k), device=q.device)[None] >= limit[a:a + 2048, None]
        got = torch.softmax(part.masked_fill(hidden, -math.inf), 1) @ v
        out[a:a + 2048] = torch.where((limit[a:a + 2048] > 0)[:, None], got, torch.zeros_like(got))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(case, s)
    hq, hk, page = case["q_heads"], case["kv_heads"], case["page"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    lens = s["kv_len"].tolist()
    off = s["q_off"].tolist() if case["kind"] == "prompt" else list(range(case["rows"] + 1))
    for i, n in enumerate(lens):
        a, b = off[i], off[i + 1]
        if not n:
            continue
        pages = s["table"][i, :-(-n // page)].long()
        limit = (n - (b - a) + 1 + torch.arange(b - a, device="cuda")).clamp(min=0)
        for h in range(hk):
            k = s["k"][pages, h].reshape(-1, case["dim"])[:n].double()
            v = s["v"][pages, h].reshape(-1, case["dim"])[:n].double()
            g = hq // hk
            q = s["q"][a:b, h * g:(h + 1) * g].double().reshape(-1, case["dim"])
            got = _exact_rows(q, k, v, limit.repeat_interleave(g), s["scale"])
            out[a:b, h * g:(h + 1) * g] = got.reshape(b - a, g, -1)
    return out
