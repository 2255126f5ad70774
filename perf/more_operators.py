"""Long contexts over the paged INT4 key/value cache: further operators of `ane_fieldfare_b200.attention`, each beside its
plain form.

A case is a dict:
  op        "shared"    attention of a batch whose requests share a long prefix, computed once for all
            "means"     the mean keys of the blocks of 64 keys that a step completes
            "select"    for every row and key/value head, the blocks whose mean keys its queries score highest
            "selected"  attention over listed blocks
  heads, kvHeads, dim    query heads, key/value heads, values of a head
  page      tokens of a cache page
  requests, rows    requests; new rows of a request (ragged: of the longest)
  ragged    lengths spread over a factor of 64 and rows spread, too
and, by operator,
  shared:           groups (of consecutive requests with a prefix each), prefix (keys of the longest), suffix (keys of a
                    request behind it)
  means:            context (keys of a request after the step)
  select, selected: context, blocks (of a list), first and last (blocks that are always in it)

A page of a layer is [kvHeads][block], a block [page][dim/2] key codes | [page][dim/64] key scale words | value codes |
value scale words; a scale word is a bf16 scale (low half) and bias, for 64 codes, two codes a byte, the first in the
low nibble.  Mean keys are bf16 [pages][kvHeads][page/64, at least 1][dim]; a block of 64 keys that lies on several pages has its mean
at the last of them.
"""
import math
import random

import torch

own = False

GROUP = 64
BLOCK = 64


def listed():
    def shared(name, requests, rows, ragged, groups, prefix, suffix, heads, kvHeads, dim, page):
        return {"name": name, "op": "shared", "requests": requests, "rows": rows, "ragged": ragged, "groups": groups, "prefix": prefix,
                "suffix": suffix, "heads": heads, "kvHeads": kvHeads, "dim": dim, "page": page}

    def means(name, requests, rows, context, heads, kvHeads, dim, page):
        return {"name": name, "op": "means", "requests": requests, "rows": rows, "context": context, "ragged": False, "heads": heads,
                "kvHeads": kvHeads, "dim": dim, "page": page}

    def listing(op, name, requests, rows, context, ragged, blocks, heads, kvHeads, dim, page):
        return {"name": name, "op": op, "requests": requests, "rows": rows, "context": context, "ragged": ragged, "blocks": blocks,
                "first": 1, "last": 1, "heads": heads, "kvHeads": kvHeads, "dim": dim, "page": page}

    return [
        # a decode step of a few users behind one system prompt
        shared("shared 8 x 2000", 8, 1, False, 1, 2000, 90, 16, 8, 256, 64),
        # a decode step of a batch that asks about one long document, conversations of all lengths
        shared("shared 64 x 32768", 64, 1, True, 1, 32768, 2048, 32, 8, 128, 32),
        # speculative blocks behind three system prompts, an odd number of heads a group
        shared("shared 3 prompts verify", 21, 5, True, 3, 8192, 500, 14, 2, 64, 16),
        # questions of several hundred tokens to one document, all of them new
        shared("shared 4 x 500 prefill", 4, 500, True, 1, 16384, 500, 16, 8, 256, 64),
        # a decode step of a batch: one request in 64 completes a block
        means("means decode 64", 64, 1, 8192, 32, 8, 128, 32),
        # a long prompt, all at once
        means("means prompt 36864", 1, 36864, 36864, 16, 8, 256, 64),
        # one user's decode step deep in a long context
        listing("select", "select 1 x 131072", 1, 1, 131072, False, 64, 32, 8, 128, 64),
        # a batch of decode steps at all depths
        listing("select", "select 64 ragged", 64, 1, 16384, True, 32, 32, 8, 128, 32),
        # the prompts of a few requests behind what they have cached
        listing("select", "select prompts 613", 5, 613, 20000, True, 48, 14, 2, 64, 16),
        # attention of the same decode steps
        listing("selected", "selected 1 x 131072", 1, 1, 131072, False, 64, 32, 8, 128, 64),
        listing("selected", "selected 64 ragged", 64, 1, 16384, True, 32, 32, 8, 128, 32),
        # speculative blocks of the largest size
        listing("selected", "selected 4 x 16 verify", 4, 16, 8000, False, 24, 16, 8, 256, 64),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most = [work(c) for c in listed()]
    while True:  # (none that costs more than the largest listed)
        case = _draw(rng)
        cost = work(case)
        if all(cost[k] <= max(w[k] for w in most) for k in cost):
            return case


def _draw(rng):
    heads, kvHeads = rng.choice([(16, 8), (32, 8), (8, 8), (14, 2), (12, 4), (16, 1)])
    case = {"heads": heads, "kvHeads": kvHeads, "dim": rng.choice([64, 128, 256]), "page": rng.choice([16, 32, 64, 128, 256]),
            "ragged": rng.choice([False, True])}
    op = rng.choice(["shared", "shared", "means", "select", "selected"])
    if op == "shared":
        requests = _log_int(rng, 1, 64)
        rows = rng.choice([1, rng.randint(2, 16), _log_int(rng, 17, max(17, 1000 // requests))])
        return {"op": op, "requests": requests, "rows": rows, "groups": rng.randint(1, min(4, requests)), "prefix": _log_int(rng, 1, 20000),
                "suffix": rows + rng.choice([0, _log_int(rng, 1, 30000 // requests)]), **case}
    if op == "means":
        requests = _log_int(rng, 1, 200)
        rows = _log_int(rng, 1, 20000 // requests)
        return {"op": op, "requests": requests, "rows": rows, "context": rows + rng.choice([0, _log_int(rng, 1, 20000 // requests)]),
                **case, "ragged": False}
    rows = rng.choice([1, 1, rng.randint(2, 16), _log_int(rng, 17, 400)])
    requests = _log_int(rng, 1, 64 if rows == 1 else 12 if rows <= 16 else 3)
    first, last = rng.randint(0, 3), rng.randint(1, 3)
    return {"op": op, "requests": requests, "rows": rows, "context": rows + _log_int(rng, 1, min(131072, 300000 // requests)),
            "blocks": first + last + _log_int(rng, 1, 64), "first": first, "last": last, **case}


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


def _part(case, i):
    """Which part of the longest the i-th request is."""
    return 64 ** ((i + 1) / case["requests"] - 1) if case["ragged"] else 1.0


def _groups(case):
    """(first request, shared keys) of every group: whole pages."""
    groups, page = case["groups"], case["page"]
    return [(g * case["requests"] // groups, int(case["prefix"] * (1 - 0.3 * g)) // page * page) for g in range(groups)]


def _lengths(case, seed):
    """(keys, new rows) of every request. The set is the case's, its order the seed's."""
    requests, rows = case["requests"], case["rows"]
    order = list(range(requests))
    random.Random(seed).shuffle(order)
    if case["op"] == "shared":
        prefix = [0] * requests
        for first, n in _groups(case):
            prefix[first:] = [n] * (requests - first)
        new = [max(1, int(round(rows * _part(case, i) ** 0.25))) for i in order]
        return [p + max(m, int(case["suffix"] * _part(case, i))) for p, m, i in zip(prefix, new, order)], new
    if case["op"] == "means":  # the last block of every request holds another number of keys
        return [max(rows, case["context"] - (7 * i) % 64) for i in order], [rows] * requests
    keys = [max(1, int(case["context"] * _part(case, i))) for i in order]
    return keys, [max(1, min(n, int(round(rows * _part(case, i) ** 0.25)))) for n, i in zip(keys, order)]


def _page_bytes(case):
    return case["page"] * (case["dim"] + case["dim"] // 8)


def _cache(case, gen, pages):
    """Pages of a cache that has been written: keys with a few loud channels, as rotary models have them, and values."""
    page, kvHeads, dim = case["page"], case["kvHeads"], case["dim"]
    out = torch.empty((pages, kvHeads, _page_bytes(case)), dtype=torch.uint8, device="cuda")
    loud = 1 + 3 * (torch.rand((kvHeads, 1, dim), device="cuda", generator=gen) < 0.05)
    for at in range(0, pages, 256):  # (a part at a time: the cache is small beside what it is made from)
        parts = []
        for kind in range(2):
            x = torch.randn((min(256, pages - at), kvHeads, page, dim), device="cuda", generator=gen)
            if kind == 0:  # keys of a page lie around one of their own
                x = (x + torch.randn((x.shape[0], kvHeads, 1, dim), device="cuda", generator=gen)) * loud
            groups = x.bfloat16().float().unflatten(-1, (-1, GROUP))
            low, high = groups.amin(-1, keepdim=True), groups.amax(-1, keepdim=True)
            scale = ((high - low) / 15).bfloat16()
            codes = ((groups - low) / scale.float()).round().clamp(0, 15).flatten(-2).to(torch.uint8)
            words = torch.cat([scale, low.bfloat16()], dim=-1).contiguous().view(torch.uint8)
            parts += [(codes[..., 0::2] + 16 * codes[..., 1::2]).flatten(2), words.flatten(2)]
        out[at:at + 256] = torch.cat(parts, dim=2)
    return out


def _tables(case, gen, keys, shared):
    """(block table, pages): every request's pages, in no order; the first shared[r][1] pages of request r are those of
    request shared[r][0]."""
    used = [-(-n // case["page"]) for n in keys]
    mine = [n - s if r != of else n for r, (n, (of, s)) in enumerate(zip(used, shared))]
    ids = torch.randperm(sum(mine) + 1, device="cuda", generator=gen).int()
    table, at = torch.zeros((len(keys), max(used)), dtype=torch.int32, device="cuda"), 0
    for r, (n, m, (of, s)) in enumerate(zip(used, mine, shared)):
        table[r, :n - m] = table[of, :n - m]
        table[r, n - m:n] = ids[at:at + m]
        at += m
    return table, sum(mine) + 1


def _starts(rows):
    start = [0]
    for n in rows:
        start.append(start[-1] + n)
    return start


def _mean_blocks(case):
    return max(1, case["page"] // BLOCK)


def _held(x, exponent):
    """x in whole numbers of 2^(exponent - 6), up to 127 of them."""
    return torch.ldexp(torch.ldexp(x, 6 - exponent).round().clamp(-127, 127), exponent - 6)


def _exponent(x):
    """floor(log2) of the largest magnitude along the last dimension, from -1000 for none."""
    top = x.abs().amax(-1, keepdim=True)
    return torch.where(top > 0, torch.frexp(top).exponent - 1, -1000)


def _lists(case, keys, rows, seed):
    """Block lists [tokens][kvHeads][blocks] as neighbouring rows choose them: three quarters the same for the rows of a
    request, the others each row's own."""
    rng, blocks, first, last = random.Random(seed), case["blocks"], case["first"], case["last"]
    out = []
    for n, m in zip(keys, rows):
        free = blocks - first - last
        middle = list(range(first, max(first, (n - m) // BLOCK + 1 - last)))
        orders = []
        for _ in range(case["kvHeads"]):
            rng.shuffle(middle)
            orders.append(list(middle))
        common = 3 * free // 4
        for i in range(m):
            seen = (n - m + i) // BLOCK + 1
            for order in orders:
                if seen <= blocks or len(order) <= free:
                    mine = list(range(seen))[-blocks:]
                else:
                    rest = order[common:]
                    at = i * (free - common) % len(rest)
                    mine = sorted(list(range(first)) + order[:common] + (rest + rest)[at:at + free - common] + list(range(seen - last, seen)))
                out.append(mine + [-1] * (blocks - len(mine)))
    return _int32(out).view(-1, case["kvHeads"], blocks)


def prepare(case, seed):
    gen = _generator(seed)
    keys, rows = _lengths(case, seed)
    start = _starts(rows)
    shared = [(r, 0) for r in range(len(keys))]
    state = {"case": case, "context": _context(len(keys), max(1, start[-1]), case), "keys": keys, "rows": rows, "lengths": _int32(keys),
             "rowStart": _int32(start), "maxRows": max(rows), "scale": case["dim"] ** -0.5}
    if case["op"] == "shared":
        groups = _groups(case) + [(len(keys), 0)]
        for (first, n), (end, _) in zip(groups, groups[1:]):
            shared[first:end] = [(first, n // case["page"])] * (end - first)
        state["groupStart"], state["prefixLengths"] = _int32([g[0] for g in groups]), _int32([g[1] for g in groups[:-1]])
    state["blockTable"], pages = _tables(case, gen, keys, shared)
    if case["op"] != "select":
        state["pages"] = _cache(case, gen, pages)
    if case["op"] != "means":
        state["q"] = torch.randn((start[-1], case["heads"], case["dim"]), device="cuda", generator=gen).bfloat16()
    if case["op"] in ("means", "select"):
        shape = (pages, case["kvHeads"], _mean_blocks(case), case["dim"])
        x = torch.randn(shape, device="cuda", generator=gen) if case["op"] == "select" else torch.zeros(shape, device="cuda")
        state["means"] = _held(x, _exponent(x).clamp(-60, 60)).bfloat16()
    if case["op"] == "means":
        state["before"] = _int32([n - m for n, m in zip(keys, rows)])
    if case["op"] == "selected":
        state["ids"] = _lists(case, keys, rows, seed)
    if case["op"] in ("shared", "selected"):
        state["out"] = torch.empty_like(state["q"])
    return state


# ---- the plain forms ---------------------------------------------------------------------------


def _unpacked(case, pages):
    """Keys and values in 32 bits [..., kvHeads, page, dim] of cache pages."""
    page, dim = case["page"], case["dim"]
    out = []
    for codes, words in zip(*[iter(pages.split(2 * [page * dim // 2, page * dim // 16], dim=-1))] * 2):
        codes = codes.unflatten(-1, (page, dim // 2))
        codes = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).unflatten(-1, (-1, GROUP))
        words = words.contiguous().view(torch.int32).unflatten(-1, (page, dim // GROUP)).unsqueeze(-1)
        out.append((codes.float() * (words << 16).view(torch.float32) + (words & -65536).view(torch.float32)).flatten(-2))
    return out


def _request(s, r, keys):
    """Keys and values [kvHeads, keys, dim] of a request."""
    pages = s["pages"][s["blockTable"][r, : -(-keys // s["case"]["page"])].long()]
    return [t.transpose(0, 1).flatten(1, 2)[:, :keys] for t in _unpacked(s["case"], pages)]


def _plain_shared(s):
    case, first, out = s["case"], 0, []
    for r, (n, m) in enumerate(zip(s["keys"], s["rows"])):
        k, v = _request(s, r, n)
        q = s["q"][first:first + m].float().unflatten(1, (case["kvHeads"], -1)).permute(1, 2, 0, 3)
        scores = torch.matmul(q, k[:, None].transpose(2, 3)) * s["scale"]
        unseen = torch.arange(n, device=q.device) > torch.arange(n - m, n, device=q.device)[:, None]
        scores = scores.masked_fill(unseen, -math.inf)
        weights = (scores - scores.amax(-1, keepdim=True)).exp()
        out.append((torch.matmul(weights, v[:, None]) / weights.sum(-1, keepdim=True)).permute(2, 0, 1, 3).flatten(1, 2))
        first += m
    return torch.cat(out).to(s["q"].dtype)


def _mean_places(s, r, blocks):
    """(page, block of the page) of the given blocks of a request."""
    page = s["case"]["page"]
    end = (blocks + 1) * BLOCK - 1
    return s["blockTable"][r, end // page].long(), end % page // BLOCK


def _plain_means(s):
    case, means = s["case"], s["means"].clone()
    for r, (n, m) in enumerate(zip(s["keys"], s["rows"])):
        begin, end = (n - m) // BLOCK, n // BLOCK
        for at in range(begin, end, 64):  # (a part at a time: 64 bits of a whole prompt are several GB)
            blocks = torch.arange(at, min(end, at + 64), device=means.device)
            low = at * BLOCK // case["page"]
            pages = s["pages"][s["blockTable"][r, low: -(-min(end, at + 64) * BLOCK // case["page"])].long()]
            keys = _unpacked(case, pages)[0].transpose(0, 1).flatten(1, 2)[:, at * BLOCK - low * case["page"]:][:, :BLOCK * len(blocks)]
            mean = keys.double().unflatten(1, (-1, BLOCK)).mean(2)
            page, place = _mean_places(s, r, blocks)
            means[page, :, place] = _held(mean, _exponent(mean).clamp(-60, 60)).transpose(0, 1).to(means.dtype)
    return means


def _plain_select(s):
    case, first, out = s["case"], 0, []
    blocks, always = case["blocks"], case["first"] + case["last"]
    q = s["q"].float().unflatten(1, (case["kvHeads"], -1))
    exponent = _exponent(q).clamp(min=-100)
    top = exponent.amax(2, keepdim=True)
    exponent = torch.maximum(exponent, top - 60)
    q = torch.ldexp(_held(q, exponent), -top)
    for r, (n, m) in enumerate(zip(s["keys"], s["rows"])):
        b = torch.arange(-(-n // BLOCK), device=q.device)
        page, place = _mean_places(s, r, b[: n // BLOCK])
        means = s["means"][page, :, place].float()
        scores = torch.einsum("ihgd,bhd->ihgb", q[first:first + m], means).amax(2)
        scores = torch.nn.functional.pad(scores, (0, len(b) - n // BLOCK))  # (the block that is not complete is the rows' own)
        position = torch.arange(n - m, n, device=q.device)[:, None]
        seen = position // BLOCK + 1
        choice = (b >= case["first"]) & (b < seen - case["last"])
        order = scores.masked_fill(~choice[:, None], -math.inf).sort(dim=-1, descending=True, stable=True).indices[..., : blocks - always]
        chosen = torch.zeros_like(scores, dtype=torch.bool).scatter(-1, order, True) & choice[:, None]
        chosen |= ((b < seen) & ~(choice & (seen > blocks)))[:, None]
        ids = torch.where(chosen, b, 1 << 30).sort(dim=-1).values[..., :blocks]
        ids = torch.nn.functional.pad(ids, (0, blocks - ids.shape[-1]), value=1 << 30)
        out.append(torch.where(ids < 1 << 30, ids, -1).int())
        first += m
    return torch.cat(out)


def _plain_selected(s):
    case, first, out = s["case"], 0, []
    kvHeads, page = case["kvHeads"], case["page"]
    for r, (n, m) in enumerate(zip(s["keys"], s["rows"])):
        for at in range(0, m, 64):
            ids = s["ids"][first + at:first + min(m, at + 64)].long()
            position = torch.arange(n - m + at, n - m + min(m, at + 64), device=ids.device)[:, None, None]
            key = (ids[..., None] * BLOCK + torch.arange(BLOCK, device=ids.device)).flatten(-2)  # [rows, kvHeads, keys]
            seen = (key >= 0) & (key <= position)
            key = torch.where(seen, key, 0)
            pages = s["pages"][s["blockTable"][r, : -(-n // page)].long()]
            k, v = (t.transpose(0, 1).flatten(1, 2) for t in _unpacked(case, pages))
            head = torch.arange(kvHeads, device=ids.device)[:, None]
            q = s["q"][first + at:first + min(m, at + 64)].float().unflatten(1, (kvHeads, -1))
            scores = torch.matmul(q, k[head, key].transpose(2, 3)) * s["scale"]
            scores = scores.masked_fill(~seen[:, :, None], -math.inf)
            weights = (scores - scores.amax(-1, keepdim=True)).exp()
            out.append((torch.matmul(weights, v[head, key]) / weights.sum(-1, keepdim=True)).flatten(1, 2))
        first += m
    return torch.cat(out).to(s["q"].dtype)


def run(s):
    op, ctx = s["case"]["op"], s["context"]
    if not own:
        return {"shared": _plain_shared, "means": _plain_means, "select": _plain_select, "selected": _plain_selected}[op](s)
    if op == "shared":
        return ctx.attendShared(s["q"], s["pages"], s["blockTable"], s["rowStart"], s["lengths"], s["maxRows"], s["groupStart"],
                                s["prefixLengths"], scale=s["scale"], out=s["out"])
    if op == "means":
        ctx.blockMeans(s["pages"], s["blockTable"], s["before"], s["lengths"], s["means"])
        return s["means"]
    if op == "select":
        return ctx.selectBlocks(s["q"], s["means"], s["blockTable"], s["rowStart"], s["lengths"], s["case"]["blocks"],
                                first=s["case"]["first"], last=s["case"]["last"])
    return ctx.attendSelected(s["q"], s["pages"], s["blockTable"], s["rowStart"], s["lengths"], s["ids"], scale=s["scale"], out=s["out"])


# ---- the same from the definition, in 64 bits ------------------------------------------------------


def _numbers(case, s, r, head, kind, n):
    """Keys (0) or values (1) [n][dim] of a head of a request."""
    page, dim = case["page"], case["dim"]
    mine = s["pages"][s["blockTable"][r, : -(-n // page)].long(), head]
    base = kind * (page * dim // 2 + page * dim // 16)
    codes = mine[:, base:base + page * dim // 2].reshape(-1, dim // 2)[:n]
    word = mine[:, base + page * dim // 2:base + page * dim // 2 + page * dim // 16].contiguous().view(torch.bfloat16)
    word = word.reshape(-1, dim // GROUP, 2)[:n].double()
    value = torch.empty((n, dim), dtype=torch.float64, device="cuda")
    value[:, 0::2], value[:, 1::2] = (codes % 16).double(), (codes // 16).double()
    return value * word[..., 0].repeat_interleave(GROUP, 1) + word[..., 1].repeat_interleave(GROUP, 1)


def _exact_means(case, s):
    out = s["means"].double()
    for r, (n, m) in enumerate(zip(s["keys"], s["rows"])):
        for head in range(case["kvHeads"]):
            k = _numbers(case, s, r, head, 0, n)
            for b in range((n - m) // BLOCK, n // BLOCK):
                mean = k[b * BLOCK:(b + 1) * BLOCK].sum(0) / BLOCK
                step = 2.0 ** (min(60, max(-60, math.floor(math.log2(mean.abs().max().item())))) - 6)
                last = b * BLOCK + BLOCK - 1
                out[s["blockTable"][r, last // case["page"]].item(), head, last % case["page"] // BLOCK] = (mean / step).round().clamp(-127, 127) * step
    return out


def _exact_attention(case, s):
    group = case["heads"] // case["kvHeads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for r, (n, m) in enumerate(zip(s["keys"], s["rows"])):
        p = torch.arange(n - m, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None]
        for h in range(case["kvHeads"]):
            k, v = _numbers(case, s, r, h, 0, n), _numbers(case, s, r, h, 1, n)
            hidden = j > p
            if case["op"] == "selected":
                named = torch.zeros((m, -(-n // BLOCK) + 1), dtype=torch.bool, device="cuda")
                named.scatter_(1, s["ids"][first:first + m, h].long() % named.shape[1], True)  # (-1: the last column, which no key has)
                hidden |= ~named[:, :-1].repeat_interleave(BLOCK, 1)[:, :n]
            for head in range(h * group, (h + 1) * group):
                score = s["q"][first:first + m, head].double() @ k.T * s["scale"]
                out[first:first + m, head] = torch.softmax(score.masked_fill_(hidden, -math.inf), dim=1) @ v
        first += m
    return out


def exact(case, seed):
    if case["op"] == "select":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "means":
        blocks = sum(n // BLOCK - (n - m) // BLOCK for n, m in zip(s["keys"], s["rows"]))
        return _exact_means(case, s) if blocks * case["kvHeads"] < 20000 else None  # (a block at a time)
    return _exact_attention(case, s)


# ---- what a pass cannot do without -----------------------------------------------------------------


def _distinct(case, n, m):
    """Blocks that the lists of a request and head name, each once (see `_lists`)."""
    blocks, free, seen = case["blocks"], case["blocks"] - case["first"] - case["last"], (n - 1) // BLOCK + 1
    middle = (n - m) // BLOCK + 1 - case["last"] - case["first"]
    if seen <= blocks or middle <= free:
        return min(seen, blocks)
    return case["first"] + case["last"] + min(middle, 3 * free // 4 + m * (free - 3 * free // 4))


def work(case):
    heads, kvHeads, dim = case["heads"], case["kvHeads"], case["dim"]
    held = kvHeads * (dim // 2 + dim // 16)  # bytes of a token's keys in the cache
    keys, rows = _lengths(case, 0)
    total = sum(rows)
    if case["op"] == "means":
        blocks = sum(n // BLOCK - (n - m) // BLOCK for n, m in zip(keys, rows))
        return {"bytes": blocks * (BLOCK * held + 2 * kvHeads * dim), "flops": 2 * blocks * BLOCK * kvHeads * dim}
    row = heads * dim
    if case["op"] == "shared":
        shared = _groups(case) + [(len(keys), 0)]
        own_, pairs = 0, 0
        for (first, n), (end, _) in zip(shared, shared[1:]):
            own_ += n + sum(k - n for k in keys[first:end])
        for n, m in zip(keys, rows):
            pairs += m * n - m * (m - 1) // 2
        return {"bytes": own_ * 2 * held + 4 * total * row, "flops": 4 * pairs * row}
    if case["op"] == "select":
        read = sum(n // BLOCK for n in keys)
        scored = sum(m * (n // BLOCK) for n, m in zip(keys, rows))
        return {"bytes": 2 * read * kvHeads * dim + 2 * total * row + 4 * total * kvHeads * case["blocks"], "flops": 2 * scored * row}
    read = sum(_distinct(case, n, m) for n, m in zip(keys, rows)) * BLOCK
    pairs = sum(m * min(n, case["blocks"] * BLOCK) for n, m in zip(keys, rows))
    return {"bytes": read * 2 * held + 4 * total * row + 4 * total * kvHeads * case["blocks"], "flops": 4 * pairs * row}
