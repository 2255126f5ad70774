"""Attention over a paged INT4 key/value cache: the operators of `ane_fieldfare_b200.attention`, each beside its
plain form.

A case is a dict:
  op        "plan"    block tables and slot maps from request lengths
            "append"  rotary positions of queries and keys, keys and values quantized into the cache, and the rows
                      read back as the cache holds them
            "attend"  attention of every request's newest rows over its cache
  heads, kvHeads, dim    query heads, key/value heads, values of a head
  page      tokens of a cache page
and, by operator,
  plan:    requests, context (the longest request), step: "decode" (one row each) or "mixed" (decode rows, verify
           blocks, rows taken back, requests that end, prompts that begin)
  append:  tokens, rotary (values of a head that rotate), interleaved, padding (one row in 16 has no slot)
  attend:  requests, rows (new rows of a request), context (keys of the longest request), ragged (lengths spread over
           a factor of 64 and one request in eight idle; rows spread, too), window (0: none), sinks

A page of a layer is [kvHeads][block], a block [page][dim/2] key codes | [page][dim/64] key scale words | value codes |
value scale words; a scale word is a bf16 scale (low half) and bias, for 64 codes, two codes a byte, the first in the
low nibble.
"""
import math
import random

import torch

own = False

GROUP = 64


def listed():
    def attend(name, requests, rows, context, ragged, heads, kvHeads, dim, page, window=0, sinks=0):
        return {"name": name, "op": "attend", "requests": requests, "rows": rows, "context": context, "ragged": ragged,
                "heads": heads, "kvHeads": kvHeads, "dim": dim, "page": page, "window": window, "sinks": sinks}

    def append(name, tokens, heads, kvHeads, dim, page, rotary, interleaved, padding):
        return {"name": name, "op": "append", "tokens": tokens, "heads": heads, "kvHeads": kvHeads, "dim": dim,
                "page": page, "rotary": rotary, "interleaved": interleaved, "padding": padding}

    def plan(name, requests, context, step, page):
        return {"name": name, "op": "plan", "requests": requests, "context": context, "step": step, "heads": 16,
                "kvHeads": 8, "dim": 128, "page": page}

    return [
        # a decode step of a small batch
        plan("plan decode 16", 16, 4096, "decode", 64),
        # a step of a busy server: decode rows, verify blocks taken back, requests that end, prompts
        plan("plan mixed 1000", 1000, 8192, "mixed", 16),
        # one decoded token
        append("append 1", 1, 16, 8, 256, 64, 256, False, False),
        # a chunk of a prompt, part of the head rotating, interleaved pairs, padded rows
        append("append 1500 interleaved", 1500, 32, 8, 128, 32, 64, True, True),
        # a full prefill chunk
        append("append 4096", 4096, 16, 8, 256, 64, 256, False, False),
        # one user's decode step
        attend("decode 1 x 2000", 1, 1, 2000, False, 16, 8, 256, 64),
        # one user's decode step deep in a long context
        attend("decode 1 x 131072", 1, 1, 131072, False, 32, 8, 128, 64),
        # a batch of decode steps at all depths, some request slots idle
        attend("decode 64 ragged", 64, 1, 16384, True, 32, 8, 128, 32),
        # speculative blocks of the largest size on a layer with a sliding window and sinks
        attend("verify 16 window", 4, 16, 8000, False, 16, 8, 256, 64, window=1024, sinks=4),
        # short prompts of several requests with what they have cached, an odd number of heads a group
        attend("prefill 613 ragged", 5, 613, 1613, True, 14, 2, 64, 16),
        # a prefill chunk on a layer with a sliding window
        attend("prefill 4096 window", 1, 4096, 12288, False, 16, 8, 256, 64, window=1024, sinks=4),
        # a prefill chunk at the end of a long context
        attend("prefill 4096 x 36864", 1, 4096, 36864, False, 16, 8, 256, 64),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    heads, kvHeads = rng.choice([(16, 8), (32, 8), (8, 8), (14, 2), (12, 4), (16, 1)])
    dim, page = rng.choice([64, 128, 256]), rng.choice([16, 32, 64, 128])
    shape = {"heads": heads, "kvHeads": kvHeads, "dim": dim, "page": page}
    op = rng.choice(["plan", "append", "attend", "attend", "attend"])
    if op == "plan":
        return {"op": op, "requests": _log_int(rng, 1, 2000), "context": _log_int(rng, 64, 16384),
                "step": rng.choice(["decode", "mixed"]), **shape}
    if op == "append":
        return {"op": op, "tokens": _log_int(rng, 1, 4096), "rotary": rng.choice([dim, dim // 2, dim // 4]),
                "interleaved": rng.choice([False, True]), "padding": rng.choice([False, True]), **shape}
    kind = rng.choice(["decode", "verify", "prefill"])
    if kind == "decode":
        requests, rows = _log_int(rng, 1, 64), 1
        context = _log_int(rng, 1, min(131072, 500000 // requests))
    elif kind == "verify":
        requests, rows = _log_int(rng, 1, 16), rng.randint(2, 16)
        context = _log_int(rng, rows, min(40000, 200000 // requests))
    else:
        requests, rows = rng.randint(1, 4), _log_int(rng, 17, 2000)
        context = rows + rng.choice([0, _log_int(rng, 1, 20000 // requests)])
    window = rng.choice([0, 0, _log_int(rng, 1, 4096)])
    return {"op": op, "requests": requests, "rows": rows, "context": context, "ragged": rng.choice([False, True]),
            "window": window, "sinks": rng.choice([0, 4, 37]) if window else 0, **shape}


# ---- inputs ----------------------------------------------------------------------------------

_contexts = {}


def _context(requests, tokens, case):
    """The framework's handle for a shape, which a program keeps; the plain form needs none."""
    if not own:
        return None
    from ane_fieldfare_b200 import attention

    key = (case["heads"], case["kvHeads"], case["dim"], case["page"], requests, tokens)
    if key not in _contexts:
        _contexts[key] = attention.AttentionContext(
            heads=case["heads"], kvHeads=case["kvHeads"], headDim=case["dim"], pageTokens=case["page"],
            maxRequests=requests, maxTokens=tokens, device=torch.cuda.current_device())
    return _contexts[key]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _lengths(case, seed):
    """(keys, new rows) of every request. The set is the case's, its order the seed's."""
    requests, rows, context = case["requests"], case["rows"], case["context"]
    keys, new = [context] * requests, [rows] * requests
    if case["ragged"]:
        for i in range(requests):
            part = (i + 1) / requests
            keys[i] = max(1, int(context * 64 ** (part - 1)))
            new[i] = max(1, min(keys[i], int(round(rows * part))))
            if i % 8 == 3:  # an idle slot of the batch
                keys[i] = new[i] = 0
    order = list(range(requests))
    random.Random(seed).shuffle(order)
    return [keys[i] for i in order], [new[i] for i in order]


def _page_bytes(case):
    return case["page"] * (case["dim"] + case["dim"] // 8)


def _cache(case, gen, pages):
    """Pages of a cache that has been written: keys with a few loud channels, as rotary models have them, and values."""
    page, kvHeads, dim = case["page"], case["kvHeads"], case["dim"]
    parts = []
    for kind in range(2):
        x = torch.randn((pages, kvHeads, page, dim), device="cuda", generator=gen)
        if kind == 0:
            loud = 1 + 3 * (torch.rand((kvHeads, 1, dim), device="cuda", generator=gen) < 0.05)
            x = x * loud
        codes, words = _quantize(x.bfloat16())
        parts += [_packed(codes).flatten(2), words.view(torch.uint8).flatten(2)]
    return torch.cat(parts, dim=2).contiguous()


def _packed(codes):
    return (codes[..., 0::2] + 16 * codes[..., 1::2]).to(torch.uint8)


def _table(positions, rotary):
    """cos and sin of a model's positions, laid out once."""
    freq = 10000.0 ** (-torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * freq
    return torch.stack([angle.cos(), angle.sin()], dim=2).float().contiguous()


def _prepare_plan(case, seed):
    gen, rng = _generator(seed), random.Random(seed)
    requests, page, context = case["requests"], case["page"], case["context"]
    old, new = [], []
    for i in range(requests):  # the steps are the case's, so that every seed has as many rows
        have = min(int(context ** rng.random()) - 1, context - 17)
        kind = "decode" if case["step"] == "decode" else ("verify", "decode", "decode", "back", "verify", "idle", "decode", "end",
                                                          "verify", "decode", "prompt", "decode", "verify", "decode")[i % 14]
        if kind == "prompt":
            have = 0
        old.append(have)
        new.append({"decode": have + 1, "verify": have + 2 + 7 * i % 15, "back": max(0, have - rng.randint(1, 15)), "end": 0,
                    "prompt": 1 + 11 * i % 40, "idle": have}[kind])
    order = list(range(requests))
    rng.shuffle(order)
    old, new = [old[i] for i in order], [new[i] for i in order]
    width = -(-context // page)
    pages = -(-3 * requests * width // 2) + 8
    ids = torch.randperm(pages, device="cuda", generator=gen).int()
    used = [-(-n // page) for n in old]
    table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    mine = torch.arange(width, device="cuda")[None] < _int32(used)[:, None]
    table[mine] = ids[: sum(used)]
    free = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    free[: pages - sum(used)] = ids[sum(used):]
    rows = sum(max(0, n - o) for o, n in zip(old, new)) + 3  # a graph's rows, the last of them padding
    return {"case": case, "context": _context(requests, rows, case), "old": _int32(old), "new": _int32(new), "blockTable": table,
            "freePages": free, "freeCount": _int32([pages - sum(used)]), "freeCountOut": _int32([0]),
            "rowStart": torch.empty(requests + 1, dtype=torch.int32, device="cuda"),
            "positions": torch.empty(rows, dtype=torch.int32, device="cuda"),
            "slots": torch.empty(rows, dtype=torch.int32, device="cuda")}


def _prepare_append(case, seed):
    gen = _generator(seed)
    tokens, heads, kvHeads, dim, page = (case[k] for k in ("tokens", "heads", "kvHeads", "dim", "page"))
    # one product's output rows: queries, keys and values side by side
    qkv = torch.randn((tokens, (heads + 2 * kvHeads) * dim), device="cuda", generator=gen).bfloat16()
    q, k, v = qkv.split([heads * dim, kvHeads * dim, kvHeads * dim], dim=1)
    pages = -(-2 * tokens // page) + 1
    first = random.Random(seed).randint(0, 30000)
    slots = torch.randperm(pages * page, device="cuda", generator=gen)[:tokens].int()
    if case["padding"]:
        slots[15::16] = -1
    positions = first + torch.arange(tokens, device="cuda", dtype=torch.int32)
    row = lambda n: torch.empty((tokens, n, dim), dtype=torch.bfloat16, device="cuda")  # noqa: E731
    return {"case": case, "context": _context(1, tokens, case), "q": q.unflatten(1, (heads, dim)), "k": k.unflatten(1, (kvHeads, dim)),
            "v": v.unflatten(1, (kvHeads, dim)), "table": _table(first + tokens, case["rotary"]), "positions": positions,
            "slots": slots, "pages": torch.zeros((pages, kvHeads, _page_bytes(case)), dtype=torch.uint8, device="cuda"),
            "qOut": row(heads), "kOut": row(kvHeads), "vOut": row(kvHeads)}


def _prepare_attend(case, seed):
    gen = _generator(seed)
    keys, rows = _lengths(case, seed)
    page, heads, dim = case["page"], case["heads"], case["dim"]
    used = [-(-n // page) for n in keys]
    pages = sum(used) + 1
    ids = torch.randperm(pages, device="cuda", generator=gen).int()
    table = torch.zeros((len(keys), max(used)), dtype=torch.int32, device="cuda")
    table[torch.arange(max(used), device="cuda")[None] < _int32(used)[:, None]] = ids[: sum(used)]
    start = [0]
    for n in rows:
        start.append(start[-1] + n)
    q = torch.randn((start[-1], heads, dim), device="cuda", generator=gen).bfloat16()
    return {"case": case, "context": _context(len(keys), start[-1], case), "q": q, "pages": _cache(case, gen, pages), "blockTable": table,
            "rowStart": _int32(start), "lengths": _int32(keys), "maxRows": max(rows), "scale": dim ** -0.5, "out": torch.empty_like(q)}


def prepare(case, seed):
    return {"plan": _prepare_plan, "append": _prepare_append, "attend": _prepare_attend}[case["op"]](case, seed)


# ---- the plain forms ---------------------------------------------------------------------------


def _quantize(x):
    """Codes (uint8) and scale words (int32) of bf16 heads [..., dim]."""
    groups = x.float().unflatten(-1, (-1, GROUP))
    low, high = groups.amin(-1, keepdim=True), groups.amax(-1, keepdim=True)
    scale = ((high - low) / 15).bfloat16()
    inverse = torch.where(scale > 0, 1 / scale.float(), torch.zeros_like(low))
    codes = ((groups - low) * inverse).round().clamp(0, 15).flatten(-2).to(torch.uint8)
    word = lambda t: t.squeeze(-1).view(torch.int16).int()  # noqa: E731
    return codes, (word(scale) & 0xFFFF) | (word(low.bfloat16()) << 16)


def _values(codes, words):
    """What codes [..., dim] and scale words [..., dim/64] stand for, in 32 bits."""
    scale = (words << 16).view(torch.float32).unsqueeze(-1)
    bias = (words & -65536).view(torch.float32).unsqueeze(-1)
    return (codes.unflatten(-1, (-1, GROUP)).float() * scale + bias).flatten(-2)


def _rotated(x, angles, rotary, interleaved):
    """bf16 heads [tokens, heads, dim] by the cosines and sines of their rows [tokens, rotary/2, 2], rounded to bf16."""
    turned, rest = x[..., :rotary].float(), x[..., rotary:]
    c, s = angles[:, None, :, 0], angles[:, None, :, 1]
    pairs = turned.unflatten(-1, (-1, 2)) if interleaved else turned.unflatten(-1, (2, -1)).transpose(-1, -2)
    a, b = pairs[..., 0], pairs[..., 1]
    pairs = torch.stack([a * c - b * s, a * s + b * c], dim=-1)
    turned = (pairs if interleaved else pairs.transpose(-1, -2)).flatten(-2)
    return torch.cat([turned.bfloat16(), rest], dim=-1)


def _plain_plan(s):
    page, table, free, count = s["case"]["page"], s["blockTable"], s["freePages"], s["freeCount"]
    old, new = s["old"], s["new"]
    had, has = (old + page - 1) // page, (new + page - 1) // page
    at = torch.arange(table.shape[1], device=table.device)[None]
    back = (at >= has[:, None]) & (at < had[:, None])
    place = torch.where(back, count + back.flatten().cumsum(0).view_as(table) - 1, free.numel())
    stack = torch.cat([free, free[:1]]).scatter(0, place.flatten(), table.flatten())[:-1]
    count = count + back.sum()
    more = (at >= had[:, None]) & (at < has[:, None])
    order = more.flatten().cumsum(0).view_as(table)
    table = torch.where(more, stack[(count - order).clamp(min=0)], table)
    count = count - more.sum()
    rows = (new - old).clamp(min=0)
    start = torch.cat([torch.zeros_like(rows[:1]), rows.cumsum(0)])
    row = torch.arange(s["slots"].numel(), device=table.device)
    request = torch.searchsorted(start[1:], row, right=True).clamp(max=rows.numel() - 1)
    live = row < start[-1]
    position = torch.where(live, old[request] + row - start[request], 0)
    slot = torch.where(live, table[request, position // page] * page + position % page, -1)
    return [t.int() for t in (table, stack, count, start, position, slot)]


def _plain_append(s):
    case = s["case"]
    angles = s["table"][s["positions"].long()]
    q = _rotated(s["q"], angles, case["rotary"], case["interleaved"])
    k = _rotated(s["k"], angles, case["rotary"], case["interleaved"])
    live = (s["slots"] >= 0)[:, None, None]
    held = [torch.where(live, _values(*_quantize(x)), 0).bfloat16() for x in (k, s["v"])]
    return [q, *held]


def _unpacked(case, pages):
    """Key and value heads in 32 bits [..., kvHeads, page, dim] of cache pages."""
    page, dim = case["page"], case["dim"]
    sizes = [page * dim // 2, page * dim // 16]
    out = []
    for codes, words in zip(*[iter(pages.split(2 * sizes, dim=-1))] * 2):
        codes = codes.unflatten(-1, (page, dim // 2))
        codes = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
        out.append(_values(codes, words.contiguous().view(torch.int32).unflatten(-1, (page, dim // GROUP))))
    return out


def _plain_attend(s):
    case, q, start, lengths, most = s["case"], s["q"], s["rowStart"].long(), s["lengths"].long(), s["maxRows"]
    heads, kvHeads, dim = case["heads"], case["kvHeads"], case["dim"]
    keys, values = _unpacked(case, s["pages"][s["blockTable"].long()])  # [requests, pages, kvHeads, page, dim]
    keys, values = (t.transpose(1, 2).flatten(2, 3) for t in (keys, values))
    rows = start[1:] - start[:-1]
    i = torch.arange(most, device=q.device)
    at = (start[:-1, None] + torch.minimum(i[None], (rows - 1).clamp(min=0)[:, None])).clamp(max=q.shape[0] - 1)
    queries = q.float()[at].unflatten(2, (kvHeads, heads // kvHeads)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = torch.matmul(queries, keys.transpose(2, 3)).mul_(s["scale"]).unflatten(2, (-1, most))
    position = (lengths - rows)[:, None, None] + i[None, :, None]
    j = torch.arange(keys.shape[2], device=q.device)[None, None]
    seen = (j <= position) & (j < lengths[:, None, None]) & (i[None, :, None] < rows[:, None, None])
    if case["window"]:
        seen &= (j > position - case["window"]) | (j < case["sinks"])
    seen = seen[:, None, None]
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1, keepdim=True).flatten(2, 3)
    values = values.masked_fill(~(j[0, 0][None, None, :, None] < lengths[:, None, None, None]), 0)
    out = torch.matmul(weights.flatten(2, 3), values) / torch.where(total > 0, total, 1)
    out = out.unflatten(2, (-1, most)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    row = torch.arange(q.shape[0], device=q.device)
    request = torch.searchsorted(start[1:], row, right=True)
    return out[request, row - start[request]].to(q.dtype)


def run(s):
    op, ctx = s["case"]["op"], s["context"]
    if not own:
        return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend}[op](s)
    if op == "plan":
        ctx.plan(s["old"], s["new"], s["blockTable"], s["freePages"], s["freeCount"], s["freeCountOut"], s["rowStart"],
                 s["positions"], s["slots"])
        return [s[k] for k in ("blockTable", "freePages", "freeCountOut", "rowStart", "positions", "slots")]
    if op == "append":
        ctx.append(s["q"], s["k"], s["v"], s["table"], s["positions"], s["slots"], s["pages"], s["qOut"],
                   interleaved=s["case"]["interleaved"])
        ctx.read(s["pages"], s["slots"], s["kOut"], s["vOut"])
        return [s["qOut"], s["kOut"], s["vOut"]]
    return ctx.attend(s["q"], s["pages"], s["blockTable"], s["rowStart"], s["lengths"], s["maxRows"], scale=s["scale"],
                      window=s["case"]["window"], sinks=s["case"]["sinks"], out=s["out"])


# ---- the same from the definition, in 64 bits ------------------------------------------------------


def _exact_append(case, s):
    rotary, half = case["rotary"], case["rotary"] // 2
    out = []
    at = s["positions"].long()
    for name in ("q", "k", "v"):
        x = s[name].double()
        if name != "v":
            turned = x.clone()
            for i in range(half):
                a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
                c, t = s["table"][at, i, 0].double()[:, None], s["table"][at, i, 1].double()[:, None]
                turned[..., a] = x[..., a] * c - x[..., b] * t
                turned[..., b] = x[..., b] * c + x[..., a] * t
            x = turned
        if name != "q":
            x = x.bfloat16().double()  # what is quantized are bf16 heads
            for g in range(0, case["dim"], GROUP):
                part = x[..., g:g + GROUP]
                low, high = part.min(-1, keepdim=True)[0], part.max(-1, keepdim=True)[0]
                scale = ((high - low) / 15).bfloat16().double()
                code = ((part - low) / torch.where(scale > 0, scale, 1)).round().clamp(0, 15)
                x[..., g:g + GROUP] = low + code * scale
            x[s["slots"] < 0] = 0
        out.append(x)
    return out


def _exact_attend(case, s):
    keys, new = s["lengths"].tolist(), (s["rowStart"][1:] - s["rowStart"][:-1]).tolist()
    page, dim, group = case["page"], case["dim"], case["heads"] // case["kvHeads"]
    half, words = page * dim // 2, page * dim // 16
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for r, (n, m) in enumerate(zip(keys, new)):
        mine = s["pages"][s["blockTable"][r, : -(-n // page)].long()]
        for h in range(case["kvHeads"] if m else 0):
            kv = []
            for base in (0, half + words):
                codes = mine[:, h, base:base + half].reshape(-1, dim // 2)[:n]
                word = mine[:, h, base + half:base + half + words].contiguous().view(torch.bfloat16)
                word = word.reshape(-1, dim // GROUP, 2)[:n].double()
                value = torch.empty((n, dim), dtype=torch.float64, device="cuda")
                value[:, 0::2], value[:, 1::2] = (codes % 16).double(), (codes // 16).double()
                kv.append(value * word[..., 0].repeat_interleave(GROUP, 1) + word[..., 1].repeat_interleave(GROUP, 1))
            p = torch.arange(n - m, n, device="cuda")[:, None]
            j = torch.arange(n, device="cuda")[None]
            hidden = j > p
            if case["window"]:
                hidden |= (j <= p - case["window"]) & (j >= case["sinks"])
            for head in range(h * group, (h + 1) * group):
                score = s["q"][first:first + m, head].double() @ kv[0].T * s["scale"]
                out[first:first + m, head] = torch.softmax(score.masked_fill_(hidden, -math.inf), dim=1) @ kv[1]
        first += m
    return out


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    return _exact_append(case, s) if case["op"] == "append" else _exact_attend(case, s)


# ---- what a pass cannot do without -----------------------------------------------------------------


def _pairs(keys, rows, window, sinks):
    """(visible (row, key) pairs, keys that any row sees) of one request."""
    if not rows:
        return 0, 0
    if not window:
        return rows * keys - rows * (rows - 1) // 2, keys
    pairs = 0
    for p in range(keys - rows, keys):
        low = max(0, p - window + 1)
        pairs += p + 1 - low + min(low, sinks)
    low = max(0, keys - rows - window + 1)
    return pairs, keys - low + min(low, sinks)


def work(case):
    held = 2 * case["kvHeads"] * (case["dim"] // 2 + case["dim"] // 16)  # bytes of a token in the cache
    if case["op"] == "plan":
        rows = case["requests"] * (1 if case["step"] == "decode" else 4)
        return {"bytes": 12 * case["requests"] + 8 * rows + 4 * rows / case["page"], "flops": 0}
    if case["op"] == "append":
        tokens, width = case["tokens"], 2 * case["dim"]
        moved = 2 * case["heads"] * width + 4 * case["kvHeads"] * width + 2 * held + 4 * case["rotary"] + 12
        return {"bytes": tokens * moved, "flops": tokens * (case["heads"] + case["kvHeads"]) * 3 * case["rotary"]}
    pairs, seen, rows = 0, 0, 0
    for n, m in zip(*_lengths(case, 0)):
        a, b = _pairs(n, m, case["window"], case["sinks"])
        pairs, seen, rows = pairs + a, seen + b, rows + m
    return {"bytes": seen * held + 4 * rows * case["heads"] * case["dim"], "flops": 4 * pairs * case["heads"] * case["dim"]}
