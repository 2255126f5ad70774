"""A decoder layer and its cache, put together from this package's operators the way a serving loop uses them:

    norm -> QKV product -> [rotary positions, INT4 cache, attention] -> output product -> fused setup -> router,
    shared FFN, routed experts -> combine -> fused tail

`CacheBook` keeps the requests' lengths, block tables and free pages on the GPU, and which requests share the pages of a prefix, whose
attention is then computed once for all of them; `DecoderLayer` is one layer's forward over the rows of a step, be they single tokens,
blocks that are verified, prompts, or a mixture.  A layer may attend to a part of a long context: for requests with few rows in a step, the blocks whose
mean keys a row's queries score highest.  The two matrix products in front of and behind attention are plain library products.
`python -m ane_fieldfare_b200.decoder` runs a small one: a prompt, a block of which some rows are taken back, single tokens, and requests
that go on from a shared prompt.
"""
from __future__ import annotations

from dataclasses import dataclass, field, replace
from itertools import accumulate
from typing import List, Optional, Sequence

import torch

from .attention import AttentionContext
from .hotpath import HotpathContext, MoE, PrefillGroupedRoutedMoE, PrefillLayerGlue, PrefillMoE, PrefillRouter, PrefillSharedExpert

__all__ = ["CacheBook", "DecoderLayer", "LayerWeights", "Selection", "Step"]


@dataclass
class Step:
    """What the layers need to know about the rows of a step (device tensors, and the host's bound on a request's rows)."""
    rowStart: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    lengths: torch.Tensor
    blockTable: torch.Tensor
    maxRows: int
    before: Optional[torch.Tensor] = None  # lengths in front of the step
    groupStart: Optional[torch.Tensor] = None  # requests that share prefixes, where some do
    prefixLengths: Optional[torch.Tensor] = None
    maxPrefix: int = 0
    rows: Optional[Sequence[int]] = None  # new tokens of each request; None: maxRows, a bound, stands for all of them
    sharing: tuple = ((), ())  # groupStart and prefixLengths on the host
    _parts: dict = field(default_factory=dict, repr=False)

    def parts(self, most: int) -> tuple:
        """(requests with up to `most` new tokens, the others), each (rows of the step, a step for the attention of them alone); None for rows
        is all of them, None for a part that there is none."""
        if self.rows is None:
            return ((None, self), None) if self.maxRows <= most else (None, (None, self))
        few = [0 < n <= most for n in self.rows]
        many = [n > most for n in self.rows]
        if not any(many):
            return (None, self), None
        if not any(few):
            return None, (None, self)
        laid = self._parts.get(most)
        if laid is None:
            new = torch.diff(self.rowStart)
            laid = self._part(few, new, (new > 0) & (new <= most)), self._part(many, new, new > most)
            if not (self.rowStart.is_cuda and torch.cuda.is_current_stream_capturing()):  # (what is captured has no values yet)
                self._parts[most] = laid
        # (the rows' places are laid out once for all layers; lengths and tables are taken at every call)
        return tuple((index, replace(part, lengths=self.lengths[chosen], blockTable=self.blockTable[chosen])) for index, chosen, part in laid)

    def _part(self, here: Sequence[bool], new: torch.Tensor, mine: torch.Tensor) -> tuple:
        """Of the requests that are `here`, on the device `mine`, of `new` rows each: their rows, their numbers, a step.  Nothing is copied
        from the host, so that a first call may be captured too."""
        i32, rows = torch.int32, [n for n, is_here in zip(self.rows, here) if is_here]
        first = lambda flags, n: torch.sort(flags.to(i32), descending=True, stable=True).indices[:n]  # noqa: E731  (places of n flags)
        index = first(torch.repeat_interleave(mine, new, output_size=sum(self.rows)), sum(rows))
        chosen = first(mine, len(rows))
        start = torch.zeros(len(rows) + 1, dtype=i32, device=new.device)
        torch.cumsum(new[chosen], 0, dtype=i32, out=start[1:])
        part = Step(start, self.positions, self.slots, self.lengths, self.blockTable, max(rows), rows=rows)
        # groups of which two or more are here; they stand one behind the other as before
        before = [0, *accumulate(here)]
        starts = [before[r] for r in self.sharing[0]]
        there = [g for g in range(len(self.sharing[1])) if starts[g + 1] > starts[g]]
        prefixes = [self.sharing[1][g] if starts[g + 1] - starts[g] > 1 else 0 for g in there]
        if any(prefixes):
            counts = torch.zeros(len(here) + 1, dtype=i32, device=new.device)
            torch.cumsum(mine, 0, dtype=i32, out=counts[1:])
            none = torch.zeros(1, dtype=i32, device=new.device)
            part.sharing, part.maxPrefix = ([*(starts[g] for g in there), starts[-1]], prefixes), max(prefixes)
            part.groupStart = counts[torch.cat([self.groupStart[g:g + 1] for g in there] + [self.groupStart[-1:]])]
            part.prefixLengths = torch.cat([self.prefixLengths[g:g + 1] if prefix else none for g, prefix in zip(there, prefixes)])
        return index, chosen, part


class CacheBook:
    """Lengths, pages and block tables of a batch of requests."""

    def __init__(self, attention: AttentionContext, requests: int, pages: int, pagesPerRequest: int):
        device, i32 = attention.device, torch.int32
        self.attention = attention
        self.lengths = [0] * requests
        self.blockTable = torch.full((requests, pagesPerRequest), -1, dtype=i32, device=device)
        self.freePages = torch.arange(pages - 1, -1, -1, dtype=i32, device=device)
        self.freeCount = torch.tensor([pages], dtype=i32, device=device)
        self._now = torch.zeros(requests, dtype=i32, device=device)
        self.heldPages = torch.zeros(requests, dtype=i32, device=device)  # of a table row, the first that are another request's
        self._prefix = [None] * requests  # (owner, pages) of the prefix that a request shares; the owner's own among them

    def share(self, owner: int, requests: Sequence[int], tokens: int) -> int:
        """`requests`, which have no tokens yet, go on from the first `tokens` of the owner's: as many as fill whole pages, which they
        read and do not own.  Returns how many.  Requests that stand one behind the other have their attention over them in one."""
        size = self.attention.pageTokens
        pages = tokens // size
        if any(not 0 <= r < len(self.lengths) for r in (owner, *requests)):
            raise ValueError(f"requests are 0 .. {len(self.lengths) - 1}")
        if not 0 <= tokens <= self.lengths[owner]:
            raise ValueError(f"the owner holds {self.lengths[owner]} tokens")
        if any(r == owner or self.lengths[r] or self._prefix[r] for r in requests):
            raise ValueError("requests that share a prefix must have no tokens of their own yet")
        if self._prefix[owner] and self._prefix[owner][0] != owner:
            raise ValueError("the owner of a prefix must hold its pages itself")
        if pages == 0 or not requests:
            return 0
        rows = torch.tensor(list(requests)).to(self.blockTable.device)
        self.blockTable[rows, :pages] = self.blockTable[owner, :pages]
        self.heldPages[rows] = pages
        self._now = self._now.clone()  # (an earlier step's lengths are this tensor)
        self._now[rows] = pages * size
        for r in requests:
            self.lengths[r], self._prefix[r] = pages * size, (owner, pages)
        self._prefix[owner] = (owner, pages)
        return pages * size

    def _groups(self) -> tuple:
        """(first requests and the end, prefix lengths) of the runs of requests that share a prefix."""
        start, lengths, at = [], [], 0
        while at < len(self._prefix):
            prefix, first = self._prefix[at], at
            while at < len(self._prefix) and self._prefix[at] == prefix:
                at += 1
            if prefix and at - first > 1:
                if start and start[-1] != first:  # requests between two groups: a group that shares nothing
                    lengths.append(0)
                    start.append(first)
                elif not start:
                    start.append(first)
                lengths.append(prefix[1] * self.attention.pageTokens)
                start.append(at)
        return start, lengths

    def step(self, newLengths: Sequence[int], maxRows: Optional[int] = None) -> Step:
        """Requests go to `newLengths` tokens: pages given back and taken, a row for every new token.  maxRows: a bound on
        the new tokens of one request, where it has to be the same for several steps.  A prefix stays as long as others share it."""
        new = list(newLengths)
        for r, prefix in enumerate(self._prefix):
            if prefix and prefix[0] != r and 0 < new[r] < prefix[1] * self.attention.pageTokens:
                raise ValueError(f"request {r} shares its first {prefix[1] * self.attention.pageTokens} tokens")
            if prefix and prefix[0] != r and new[r] and new[prefix[0]] < prefix[1] * self.attention.pageTokens:
                raise ValueError(f"request {r} shares the first {prefix[1] * self.attention.pageTokens} tokens of request {prefix[0]}")
        rows = [max(0, b - a) for a, b in zip(self.lengths, new)]
        device, i32, total = self.attention.device, torch.int32, sum(rows)
        after = torch.tensor(new, dtype=i32).to(device)
        step = Step(torch.empty(len(new) + 1, dtype=i32, device=device), torch.empty(total, dtype=i32, device=device),
                    torch.empty(total, dtype=i32, device=device), after, self.blockTable, max(rows + [1]) if maxRows is None else maxRows, self._now,
                    rows=rows if maxRows is None else None)
        self.attention.plan(self._now, after, self.blockTable, self.freePages, self.freeCount, self.freeCount, step.rowStart,
                            step.positions, step.slots, heldPages=self.heldPages if any(self._prefix) else None)
        gone = [r for r, prefix in enumerate(self._prefix) if prefix and prefix[0] != r and new[r] == 0]
        if gone:
            self.heldPages[torch.tensor(gone).to(device)] = 0
            for r in gone:
                self._prefix[r] = None
            owners = {prefix[0] for r, prefix in enumerate(self._prefix) if prefix and prefix[0] != r}
            self._prefix = [None if prefix and prefix[0] == r and r not in owners else prefix for r, prefix in enumerate(self._prefix)]
        start, prefixes = self._groups()
        if prefixes:
            step.groupStart, step.prefixLengths = torch.tensor(start, dtype=i32).to(device), torch.tensor(prefixes, dtype=i32).to(device)
            step.maxPrefix, step.sharing = max(prefixes), (start, prefixes)
        self.lengths, self._now = new, after
        return step


@dataclass
class Selection:
    """Attention to a part of the context: `blocks` blocks of 64 keys a row and key/value head, the first and the last among them in
    any case, for requests that bring up to `maxRows` rows to a step (more of them read a block together by reading all).  A request's rows
    attend alike whatever others the step has, but where `CacheBook.step` is given a bound, which then decides for all."""
    blocks: int
    first: int = 1
    last: int = 1
    maxRows: int = 16


@dataclass
class LayerWeights:
    """bf16 on the device: products [outputs][inputs], norms [d]."""
    qkv: torch.Tensor
    out: torch.Tensor
    inputNorm: torch.Tensor
    postAttn: torch.Tensor
    preFfn: torch.Tensor
    preFfn2: torch.Tensor
    postFfn2: torch.Tensor
    postFfn: torch.Tensor


class DecoderLayer:
    """One layer: `layer` of the MoE context's resident layers behind attention over `pages` of a cache of its own."""

    def __init__(self, moe: HotpathContext, attention: AttentionContext, layer: int, weights: LayerWeights, ropeTable: torch.Tensor,
                 pages: int, *, window: int = 0, sinks: int = 0, interleaved: bool = False, eps: float = 1e-6, layerScalar: float = 1.0,
                 selected: Optional[Selection] = None):
        if selected and window:
            raise ValueError("a layer with a window does not select blocks")
        self.moe, self.attention, self.layer, self.weights, self.ropeTable = moe, attention, layer, weights, ropeTable
        self.window, self.sinks, self.interleaved, self.eps, self.layerScalar = window, sinks, interleaved, eps, layerScalar
        self.cache, self.selected = attention.newCache(pages), selected
        self.means = attention.newMeans(pages) if selected else None
        self._ops = (MoE(moe), PrefillRouter(moe), PrefillSharedExpert(moe), PrefillGroupedRoutedMoE(moe), PrefillMoE(moe), PrefillLayerGlue(moe))

    def attend(self, x: torch.Tensor, step: Step) -> torch.Tensor:
        """Attention of normed rows x [rows][d] over their requests' caches, theirs appended; [rows][heads][headDim]."""
        att, w = self.attention, self.weights
        qkv = (x @ w.qkv.T).unflatten(1, (-1, att.headDim))
        q, k, v = qkv.split([att.heads, att.kvHeads, att.kvHeads], dim=1)
        q = att.append(q, k, v, self.ropeTable, step.positions, step.slots, self.cache, interleaved=self.interleaved)
        if not self.selected:
            return self._all_keys(q, step)
        att.blockMeans(self.cache, step.blockTable, step.before, step.lengths, self.means)
        few, many = step.parts(self.selected.maxRows)
        if many is None:
            return self._blocks(q, step)
        if few is None:
            return self._all_keys(q, step)
        out = torch.empty_like(q)
        for (index, part), attention in ((few, self._blocks), (many, self._all_keys)):
            out[index] = attention(q[index], part)
        return out

    def _blocks(self, q: torch.Tensor, step: Step) -> torch.Tensor:
        att, choice = self.attention, self.selected
        ids = att.selectBlocks(q, self.means, step.blockTable, step.rowStart, step.lengths, choice.blocks, first=choice.first, last=choice.last)
        return att.attendSelected(q, self.cache, step.blockTable, step.rowStart, step.lengths, ids)

    def _all_keys(self, q: torch.Tensor, step: Step) -> torch.Tensor:
        att = self.attention
        if step.groupStart is not None and not self.window:
            return att.attendShared(q, self.cache, step.blockTable, step.rowStart, step.lengths, step.maxRows, step.groupStart, step.prefixLengths,
                                    maxPrefix=step.maxPrefix)
        return att.attend(q, self.cache, step.blockTable, step.rowStart, step.lengths, step.maxRows, window=self.window, sinks=self.sinks)

    def forward(self, hidden: torch.Tensor, step: Step) -> torch.Tensor:
        """Updates the residual stream hidden [rows][d] in place."""
        moe, router, shared, routed, combine, glue = self._ops
        w, tokens, topK = self.weights, hidden.shape[0], self.moe.topK
        if tokens == 0:
            return hidden
        attended = self.attend(self.moe.rmsnorm(hidden, w.inputNorm, self.eps), step).flatten(1) @ w.out.T
        denseX, routedX, routerX, h1, h2 = (torch.empty_like(hidden) for _ in range(5))
        ids = torch.empty((tokens, topK), dtype=torch.int32, device=hidden.device)
        routes = torch.empty((tokens, topK), dtype=torch.bfloat16, device=hidden.device)
        glue.encodePostAttnSetupBlock(None, hidden, attended, w.postAttn, w.preFfn, w.preFfn2, self.eps, denseX, routedX, routerX)
        if tokens == 1:
            moe.encodeRouterGemma4(None, self.layer, routerX, ids, routes, topK)
            shared.encode(None, self.layer, denseX, h1)
            moe.encodeRoutedPersistentGPUSlots(None, self.layer, ids, routedX, routes, None, h2)
        else:
            partials = torch.empty((tokens * topK, hidden.shape[1]), dtype=torch.bfloat16, device=hidden.device)
            router.encodeGemma4Block(None, self.layer, routerX, ids, routes, tokens)
            shared.encodeBlock(None, self.layer, denseX, h1, tokens)
            if tokens <= routed.verifyMaxRows:
                routed.encodeVerifyBound(None, self.layer, routedX, ids, partials, tokens)
            else:
                routed.encodeStreamedBatched(None, self.layer, routedX, ids, partials, tokens)
            combine.encodeReduceTokenMajor(None, partials, routes, h2, tokens)
        glue.encodeLayerTailBlock(None, h2, h1, hidden, w.postFfn2, w.postFfn, self.eps, self.layerScalar)
        return hidden


def small_decoder(layers: int = 2, d: int = 256, requests: int = 2, pages: int = 64, seed: int = 1, selected: Optional[Selection] = None,
                  **attention) -> tuple:
    """(CacheBook, layers) with random weights, for a demonstration or a test."""
    from . import workload

    shape = {"heads": 8, "kvHeads": 2, "headDim": 64, "pageTokens": 16, **attention}
    moe = HotpathContext(layers=layers, experts=16, d=d, f=128, sharedF=192, topK=8, maxTokens=512)
    att = AttentionContext(maxRequests=requests, maxTokens=512, **shape)
    book = CacheBook(att, requests, pages, pages)
    gen = torch.Generator(device=att.device).manual_seed(seed)
    draw = lambda rows, cols: (torch.randn((rows, cols), device=att.device, generator=gen) / cols ** 0.5).bfloat16()  # noqa: E731
    table = att.ropeTable(pages * att.pageTokens, rotaryDim=att.headDim)
    stack: List[DecoderLayer] = []
    for i in range(layers):
        workload.load_layer(moe, i, workload.make_layer(seed, i, experts=16, d=d, f=128, sharedF=192, topK=8, router_bias="normal"))
        norms = [(1 + 0.1 * torch.randn(d, device=att.device, generator=gen)).bfloat16() for _ in range(6)]
        weights = LayerWeights(draw((att.heads + 2 * att.kvHeads) * att.headDim, d), draw(d, att.heads * att.headDim), *norms)
        # every second layer sees a window and the first tokens
        stack.append(DecoderLayer(moe, att, i, weights, table, pages, window=32 if i % 2 else 0, sinks=4 if i % 2 else 0,
                                  selected=None if i % 2 else selected))
    return book, stack


def _run(book: CacheBook, stack: Sequence[DecoderLayer], steps: Sequence[tuple]):
    device = book.attention.device
    for what, want in steps:
        rows = sum(max(0, b - a) for a, b in zip(book.lengths, want))
        hidden = torch.randn((rows, stack[0].moe.d), device=device).bfloat16()
        step = book.step(want)
        for layer in stack:
            layer.forward(hidden, step)
        torch.cuda.synchronize()
        print(f"{what}: {rows} rows, lengths {want}, {int(book.freeCount)} pages free" + (f", |hidden| {hidden.float().norm(dim=1).mean():.1f}" if rows else ""))


def main():
    book, stack = small_decoder()
    _run(book, stack, [("prompts", [70, 33]), ("a block of eight rows", [78, 41]), ("five of them taken back", [73, 36]), ("a token each", [74, 37]),
                       ("one request ends", [75, 0])])
    print("error flag:", book.attention.info().deviceErrorFlag)
    book, stack = small_decoder(requests=4, selected=Selection(blocks=3))
    _run(book, stack, [("one prompt", [300, 0, 0, 0])])
    shared = book.share(0, [1, 2, 3], 300)
    print(f"three requests go on from its first {shared} tokens")
    _run(book, stack, [("their questions", [300, shared + 20, shared + 33, shared + 5]), ("a token each", [301, shared + 21, shared + 34, shared + 6]),
                       ("they end", [301, 0, 0, 0]), ("and their prompt", [0, 0, 0, 0])])
    print("error flag:", book.attention.info().deviceErrorFlag)


if __name__ == "__main__":
    main()
