"""Attention over a paged INT4 key/value cache, over the C ABI (`ff_attention_*`, `ff_cache_*`, `ff_rope*`): the half
of a layer in front of `hotpath.PrefillLayerGlue.encodePostAttnSetupBlock`.

A step of a server or a decode loop is four calls on one stream, none of which waits for the GPU or reads from it:
`plan` turns the requests' lengths into pages, positions and slots; `append` rotates queries and keys and quantizes
keys and values into the cache (once per layer); `attend` is the attention over what is cached (once per layer).

The cache's memory is the caller's: `newCache(pages)` per layer, uint8 [pages][kvHeads][bytes of a block]; its layout
stands in include/fieldfare_cuda.h.  Lengths, tables, positions and slots are int32 CUDA tensors.  Wrong shapes, types or
devices raise `ValueError`, what the library refuses raises `FieldfareError`; what a kernel finds in its data (no free
page, a page outside the cache) stands in `info().deviceErrorFlag`.  A result that a call with `stream` allocates belongs to that
stream, as torch counts it: to use it on another, wait for the stream, and `record_stream` it there.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import binding
from .binding import FFAttentionConfig, FFRope, FFRopeConfig, FieldfareError, call
from .hotpath import _stream

__all__ = ["AttentionContext", "FieldfareError", "NO_SLOT"]

NO_SLOT = -1  # as int32; also a table entry without a page

_WORD = 0xFFFFFFFF  # (ctypes would cut what is more without a word)

_SCALING = {"none": 0, "linear": 1, "byParts": 2}


class AttentionContext:
    """Owns one FFAttention: the kernels' scratch for one shape of attention."""

    def __init__(self, *, heads: int, kvHeads: int, headDim: int, pageTokens: int = 64, maxRequests: int = 64,
                 maxTokens: int = 4096, device: int = 0):
        lib = binding.load()
        self.config = FFAttentionConfig(heads, kvHeads, headDim, pageTokens, maxRequests, maxTokens)
        err = ctypes.c_char_p()
        self._handle = lib.ff_attention_create(device, ctypes.byref(self.config), ctypes.byref(err))
        if not self._handle:
            raise FieldfareError(err.value.decode() if err.value else "ff_attention_create failed")
        self.device, self._ordinal = torch.device("cuda", device), device
        self.heads, self.kvHeads, self.headDim, self.pageTokens = heads, kvHeads, headDim, pageTokens
        self.maxRequests, self.maxTokens = maxRequests, maxTokens
        self.pageBytes = lib.ff_cache_page_bytes(ctypes.byref(self.config))

    @property
    def handle(self):
        if not self._handle:
            raise FieldfareError("attention handle was destroyed")
        return self._handle

    def close(self):
        if getattr(self, "_handle", None):
            binding.load().ff_attention_destroy(self._handle)
            self._handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def info(self) -> binding.FFAttentionInfo:
        return binding.load().ff_attention_get_info(self.handle)

    def resetDeviceError(self):
        call("ff_attention_reset_device_error", self.handle)

    # -- arguments ---------------------------------------------------------------------------------

    def _new(self, shape: tuple, dtype: torch.dtype, stream) -> torch.Tensor:
        """Memory for a result, of the stream that writes it: the current stream may still use what it has freed."""
        if stream is None:
            return torch.empty(shape, dtype=dtype, device=self.device)
        with torch.cuda.stream(stream):
            return torch.empty(shape, dtype=dtype, device=self.device)

    # (A step of small calls is bound by the host: `get_device` and `is` cost a fifth of comparing torch.device objects, one
    # look at shape and strides a third of four.)

    def _ints(self, names: str, *tensors: torch.Tensor):
        """Refuses what is not a contiguous int32 tensor on the device."""
        i32, ordinal = torch.int32, self._ordinal
        for t in tensors:
            if t.dtype is not i32 or t.get_device() != ordinal or not t.is_contiguous():
                what = next(name for name, u in zip(names.split(), tensors) if u is t)
                raise ValueError(f"{what} must be a contiguous int32 tensor on {self.device}")

    def _heads(self, t: torch.Tensor, heads: int, tokens: int, what: str) -> tuple:
        """(pointer, elements between rows) of bf16 [tokens][heads][headDim], the heads of a row side by side."""
        dim = self.headDim
        if t.dtype is not torch.bfloat16 or t.get_device() != self._ordinal:
            raise ValueError(f"{what} must be bf16 on {self.device}")
        if t.shape != (tokens, heads, dim):
            raise ValueError(f"{what} must be [{tokens}][{heads}][{dim}]")
        row, head, value = t.stride()
        if tokens and (value != 1 or (head != dim and heads > 1)):
            raise ValueError(f"{what} must have the heads of a row side by side")
        if tokens < 2:
            return t.data_ptr(), heads * dim
        if row > _WORD:
            raise ValueError(f"rows of {what} must be less than 2^32 elements apart")
        return t.data_ptr(), row

    def _cache(self, pages: torch.Tensor) -> tuple:
        count = pages.shape[0] if pages.dim() else 0
        if (pages.dtype is not torch.uint8 or pages.get_device() != self._ordinal or not pages.is_contiguous()
                or pages.numel() != count * self.pageBytes):
            raise ValueError(f"a cache is contiguous uint8 [pages][kvHeads][...] with {self.pageBytes} bytes a page on {self.device}")
        return pages.data_ptr(), count

    def _rope(self, table: Optional[torch.Tensor], interleaved: bool) -> FFRope:
        if table is None:
            return FFRope(None, 0, 0, int(interleaved))
        shape = table.shape
        if table.dtype is not torch.float32 or table.get_device() != self._ordinal or not table.is_contiguous() or len(shape) != 3 or shape[2] != 2:
            raise ValueError(f"a rotary table is fp32 [positions][rotaryDim/2][2] on {self.device}")
        return FFRope(table.data_ptr(), shape[0], 2 * shape[1], int(interleaved))

    # -- the cache ---------------------------------------------------------------------------------

    def newCache(self, pages: int) -> torch.Tensor:
        """Memory of one layer's cache."""
        return torch.zeros((pages, self.kvHeads, self.pageBytes // self.kvHeads), dtype=torch.uint8, device=self.device)

    def plan(self, oldLengths: torch.Tensor, newLengths: torch.Tensor, blockTable: torch.Tensor, freePages: torch.Tensor,
             freeCount: torch.Tensor, freeCountOut: torch.Tensor, rowStart: torch.Tensor, positions: torch.Tensor,
             slots: torch.Tensor, stream=None):
        """Request r goes from oldLengths[r] to newLengths[r] tokens: pages given back and taken (blockTable [requests]
        [pages], the stack freePages with freeCount [1] entries; freeCountOut may be freeCount), and a row for every new
        token: rowStart [requests + 1], positions and slots [rows]."""
        requests, rows = oldLengths.numel(), slots.numel()
        shape = blockTable.shape
        if newLengths.numel() != requests or len(shape) != 2 or shape[0] != requests or rowStart.numel() != requests + 1:
            raise ValueError("lengths, blockTable and rowStart must agree on the number of requests")
        if positions.numel() != rows or freeCount.numel() != 1 or freeCountOut.numel() != 1:
            raise ValueError("one position and one slot per row; one word for the stack's height")
        self._ints("oldLengths newLengths blockTable freePages freeCount freeCountOut rowStart positions slots", oldLengths, newLengths,
                   blockTable, freePages, freeCount, freeCountOut, rowStart, positions, slots)
        call("ff_cache_plan", self.handle, oldLengths.data_ptr(), newLengths.data_ptr(), requests, blockTable.data_ptr(), shape[1],
             freePages.data_ptr(), freePages.numel(), freeCount.data_ptr(), freeCountOut.data_ptr(), rowStart.data_ptr(),
             positions.data_ptr(), slots.data_ptr(), rows, _stream(stream))

    def ropeTable(self, positions: int, *, base: float = 10000.0, rotaryDim: Optional[int] = None, scaling: str = "none",
                  factor: float = 1.0, lowTurns: float = 1.0, highTurns: float = 4.0, originalContext: float = 8192.0,
                  amplitude: float = 1.0, stream=None) -> torch.Tensor:
        """Cosines and sines fp32 [positions][rotaryDim/2][2]; `scaling` "none", "linear" or "byParts"."""
        if scaling not in _SCALING:
            raise ValueError(f"scaling must be one of {sorted(_SCALING)}")
        rotary = self.headDim if rotaryDim is None else rotaryDim
        config = FFRopeConfig(base, rotary, _SCALING[scaling], factor, lowTurns, highTurns, originalContext, amplitude)
        table = self._new((positions, max(0, rotary) // 2, 2), torch.float32, stream)
        call("ff_rope_table", self.handle, ctypes.byref(config), table.data_ptr(), positions, _stream(stream))
        return table

    def rope(self, x: torch.Tensor, table: Optional[torch.Tensor], positions: torch.Tensor, y: Optional[torch.Tensor] = None,
             *, interleaved: bool = False, stream=None) -> torch.Tensor:
        """Rotated heads of x [tokens][any heads][headDim] (table None: as they are); y may be x."""
        if x.dim() != 3 or positions.numel() != x.shape[0]:
            raise ValueError("x must be [tokens][heads][headDim], with one position per row")
        tokens, heads = x.shape[:2]
        if y is None:
            y = self._new((tokens, heads, self.headDim), torch.bfloat16, stream)
        rope = self._rope(table, interleaved)
        self._ints("positions", positions)
        call("ff_rope", self.handle, *self._heads(x, heads, tokens, "x"), ctypes.byref(rope), positions.data_ptr(), heads, tokens,
             *self._heads(y, heads, tokens, "y"), _stream(stream))
        return y

    def append(self, q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, table: Optional[torch.Tensor],
               positions: torch.Tensor, slots: torch.Tensor, pages: torch.Tensor, qOut: Optional[torch.Tensor] = None,
               *, interleaved: bool = False, stream=None) -> Optional[torch.Tensor]:
        """Keys rotated (table None: as they are) and values into the cache at `slots`; returns the rotated queries (qOut;
        q may be None).  q, k and v may be parts of one row (a QKV product)."""
        tokens = k.shape[0]
        if positions.numel() != tokens or slots.numel() != tokens:
            raise ValueError("one position and one slot per row")
        query, out = (None, 0), (None, 0)
        if q is not None:
            if qOut is None:
                qOut = self._new((tokens, self.heads, self.headDim), torch.bfloat16, stream)
            query, out = self._heads(q, self.heads, tokens, "q"), self._heads(qOut, self.heads, tokens, "qOut")
        rope = self._rope(table, interleaved)
        self._ints("positions slots", positions, slots)
        call("ff_cache_append", self.handle, *query, *self._heads(k, self.kvHeads, tokens, "k"), *self._heads(v, self.kvHeads, tokens, "v"),
             ctypes.byref(rope), positions.data_ptr(), slots.data_ptr(), tokens, *out, *self._cache(pages),
             _stream(stream))
        return qOut

    def read(self, pages: torch.Tensor, slots: torch.Tensor, k: Optional[torch.Tensor] = None, v: Optional[torch.Tensor] = None,
             stream=None) -> tuple:
        """(keys, values) that slots hold, bf16 [slots][kvHeads][headDim]; zeros for NO_SLOT."""
        tokens = slots.numel()
        shape = (tokens, self.kvHeads, self.headDim)
        if k is None:
            k = self._new(shape, torch.bfloat16, stream)
        if v is None:
            v = self._new(shape, torch.bfloat16, stream)
        if not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError("k and v must be contiguous")
        self._ints("slots", slots)
        call("ff_cache_read", self.handle, *self._cache(pages), slots.data_ptr(), tokens, self._heads(k, self.kvHeads, tokens, "k")[0],
             self._heads(v, self.kvHeads, tokens, "v")[0], _stream(stream))
        return k, v

    # -- attention ---------------------------------------------------------------------------------

    def attend(self, q: torch.Tensor, pages: torch.Tensor, blockTable: torch.Tensor, rowStart: torch.Tensor,
               lengths: torch.Tensor, maxRows: int, *, scale: Optional[float] = None, window: int = 0, sinks: int = 0,
               out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
        """Rows rowStart[r] .. rowStart[r + 1] - 1 of q over request r's `lengths[r]` cached keys, their own among them;
        maxRows: no request has more rows.  window 0: every key up to the row's own; otherwise the last `window` of them
        and the first `sinks`."""
        tokens, requests, shape = q.shape[0], lengths.numel(), blockTable.shape
        if rowStart.numel() != requests + 1 or len(shape) != 2 or shape[0] != requests:
            raise ValueError("lengths, blockTable and rowStart must agree on the number of requests")
        if window < 0 or sinks < 0 or maxRows < 0:
            raise ValueError("window, sinks and maxRows must not be negative")
        if window > _WORD or sinks > _WORD or maxRows > _WORD:  # (more than any request has)
            window, sinks, maxRows = min(window, _WORD), min(sinks, _WORD), min(maxRows, _WORD)
        if out is None:
            out = self._new((tokens, self.heads, self.headDim), torch.bfloat16, stream)
        self._ints("blockTable rowStart lengths", blockTable, rowStart, lengths)
        call("ff_attention", self.handle, *self._heads(q, self.heads, tokens, "q"), tokens, *self._cache(pages), blockTable.data_ptr(), shape[1],
             rowStart.data_ptr(), lengths.data_ptr(), requests, maxRows, self.headDim ** -0.5 if scale is None else scale, window, sinks,
             *self._heads(out, self.heads, tokens, "out"), _stream(stream))
        return out
