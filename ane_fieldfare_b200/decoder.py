"""A decoder layer and its cache, put together from this package's operators the way a serving loop uses them:

    norm -> QKV product -> [rotary positions, INT4 cache, attention] -> output product -> fused setup -> router,
    shared FFN, routed experts -> combine -> fused tail

`CacheBook` keeps the requests' lengths, block tables and free pages on the GPU; `DecoderLayer` is one layer's forward over the
rows of a step, be they single tokens, blocks that are verified, prompts, or a mixture.  The two matrix products in front of and
behind attention are plain library products.  `python -m ane_fieldfare_b200.decoder` runs a small one: a prompt, a block
of which some rows are taken back, and single tokens.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Sequence

import torch

from .attention import AttentionContext
from .hotpath import HotpathContext, MoE, PrefillGroupedRoutedMoE, PrefillLayerGlue, PrefillMoE, PrefillRouter, PrefillSharedExpert

__all__ = ["CacheBook", "DecoderLayer", "LayerWeights", "Step"]


@dataclass
class Step:
    """What the layers need to know about the rows of a step (device tensors, and the host's bound on a request's rows)."""
    rowStart: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    lengths: torch.Tensor
    blockTable: torch.Tensor
    maxRows: int


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

    def step(self, newLengths: Sequence[int], maxRows: Optional[int] = None) -> Step:
        """Requests go to `newLengths` tokens: pages given back and taken, a row for every new token.  maxRows: a bound on
        the new tokens of one request, where it has to be the same for several steps."""
        new = list(newLengths)
        rows = [max(0, b - a) for a, b in zip(self.lengths, new)]
        device, i32, total = self.attention.device, torch.int32, sum(rows)
        after = torch.tensor(new, dtype=i32).to(device)
        step = Step(torch.empty(len(new) + 1, dtype=i32, device=device), torch.empty(total, dtype=i32, device=device),
                    torch.empty(total, dtype=i32, device=device), after, self.blockTable, max(rows + [1]) if maxRows is None else maxRows)
        self.attention.plan(self._now, after, self.blockTable, self.freePages, self.freeCount, self.freeCount, step.rowStart,
                            step.positions, step.slots)
        self.lengths, self._now = new, after
        return step


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
                 pages: int, *, window: int = 0, sinks: int = 0, interleaved: bool = False, eps: float = 1e-6, layerScalar: float = 1.0):
        self.moe, self.attention, self.layer, self.weights, self.ropeTable = moe, attention, layer, weights, ropeTable
        self.window, self.sinks, self.interleaved, self.eps, self.layerScalar = window, sinks, interleaved, eps, layerScalar
        self.cache = attention.newCache(pages)
        self._ops = (MoE(moe), PrefillRouter(moe), PrefillSharedExpert(moe), PrefillGroupedRoutedMoE(moe), PrefillMoE(moe), PrefillLayerGlue(moe))

    def attend(self, x: torch.Tensor, step: Step) -> torch.Tensor:
        """Attention of normed rows x [rows][d] over their requests' caches, theirs appended; [rows][heads][headDim]."""
        att, w = self.attention, self.weights
        qkv = (x @ w.qkv.T).unflatten(1, (-1, att.headDim))
        q, k, v = qkv.split([att.heads, att.kvHeads, att.kvHeads], dim=1)
        q = att.append(q, k, v, self.ropeTable, step.positions, step.slots, self.cache, interleaved=self.interleaved)
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


def small_decoder(layers: int = 2, d: int = 256, requests: int = 2, pages: int = 64, seed: int = 1, **attention) -> tuple:
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
        stack.append(DecoderLayer(moe, att, i, weights, table, pages, window=32 if i % 2 else 0, sinks=4 if i % 2 else 0))
    return book, stack


def main():
    book, stack = small_decoder()
    device = book.attention.device
    have = [0, 0]
    for what, want in [("prompts", [70, 33]), ("a block of eight rows", [78, 41]), ("five of them taken back", [73, 36]),
                       ("a token each", [74, 37]), ("one request ends", [75, 0])]:
        rows = sum(max(0, b - a) for a, b in zip(have, want))
        hidden = torch.randn((rows, stack[0].moe.d), device=device).bfloat16()
        step = book.step(want)
        for layer in stack:
            layer.forward(hidden, step)
        torch.cuda.synchronize()
        print(f"{what}: {rows} rows, lengths {want}, {int(book.freeCount)} pages free" + (f", |hidden| {hidden.float().norm(dim=1).mean():.1f}" if rows else ""))
        have = want
    print("error flag:", book.attention.info().deviceErrorFlag)


if __name__ == "__main__":
    main()
