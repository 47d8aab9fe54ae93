"""Key/value cache in pages of 16-bit keys and values, for prompts, steps and drafted
trees (kt_paged_* in include/kt_cuda.h).

The reference's KVCache (Engine/kotensor/src/main/kotlin/KVCache.kt:3-59) keeps float32
keys and values in one block a sequence; here sequences of unlike lengths share a pool of
pages in bfloat16 or float16.  ``append`` rotates new queries and keys by their positions
and stores keys and values, ``attend`` runs attention of single tokens, of prompts or of
trees of drafted tokens over what is held, ``accept`` keeps the path of a tree that the
model's choices confirm.  One cache serves all layers.
"""
from __future__ import annotations

import copy
import ctypes
import math
import operator
from typing import Optional

import numpy as np

from . import _lib
from .kv8 import _rows
from .quantized import Context, raw_stream

try:
    import torch
except ImportError:  # pragma: no cover
    torch = None

COUNTER_BYTES = 4096  # of the scratch, zero before its first use
MOST_NODES = 1024     # of a drafted tree


def draft_tree(parents):
    """What ``append`` and ``attend`` need to know of drafted trees: ``parents`` is an array
    [rows] or [batch, rows] of each node's parent (smaller than its own index; -1 for
    node 0, the last token of the text).  Returns numpy int32 arrays ``depths`` of the same
    shape (nodes above each) and ``visible`` [..., rows, (rows + 31) // 32] (bit u % 32 of
    word u // 32 of row t: u is t or above it)."""
    parents = np.asarray(parents, dtype=np.int64)
    if parents.ndim not in (1, 2) or not 1 <= parents.shape[-1] <= MOST_NODES:
        raise ValueError(f"parents must be [rows] or [batch, rows] with 1..{MOST_NODES} rows, got {list(parents.shape)}")
    rows = parents.shape[-1]
    trees = parents.reshape(-1, rows)
    if (trees[:, 0] != -1).any() or (trees[:, 1:] < 0).any() or (trees >= np.arange(rows)).any():
        raise ValueError("node 0 has no parent (-1), every other one a parent before it")
    depths = np.zeros(trees.shape, np.int32)
    seen = np.zeros((*trees.shape, (rows + 31) // 32 * 32), bool)
    batch = np.arange(trees.shape[0])
    seen[:, 0, 0] = True
    for t in range(1, rows):
        depths[:, t] = depths[batch, trees[:, t]] + 1
        seen[:, t] = seen[batch, trees[:, t]]
        seen[:, t, t] = True
    visible = np.packbits(seen, axis=-1, bitorder="little").view("<i4").astype(np.int32)
    return depths.reshape(parents.shape), visible.reshape(*parents.shape, -1)


class PagedKVCache:
    """``pages`` pages of ``page`` (16, 32, 64 or 128) slots of ``kv_heads`` heads of
    ``head_dim`` (a multiple of 16 in 64..128) in each of ``layers`` layers, for ``batch``
    sequences of at most ``max_tokens`` tokens (rounded up to whole pages).

    keys, values bfloat16 or float16 [layers, pages, kv_heads, page, head_dim]
    table        int32 [batch, max_tokens / page]: the page of each run of slots, -1 for none
    lengths      int32 [batch], tokens held by each sequence
    status       int32 [1], not 0 once a token had no page

    ``reserve`` and ``release`` hand out the pool's pages; a program may fill ``table`` with
    page numbers of its own instead (shared prefixes).  ``append`` and ``attend`` of every
    layer work at the same ``lengths``; ``advance`` moves on after the last layer.  Calls
    run on the current stream of the cache's device and share one scratch buffer: order
    them on one stream.  A slot that a call writes must be one sequence's alone, and there
    once (shared pages hold tokens that all who share them keep).  A cache, or a view, whose
    calls were captured has to outlive the graph.
    """

    def __init__(self, layers: int, batch: int, kv_heads: int, head_dim: int, pages: int, max_tokens: int, page: int = 64,
                 dtype=None, device: Optional[int] = None):
        dtype = torch.bfloat16 if dtype is None else dtype
        if layers < 1 or kv_heads < 1 or pages < 1 or max_tokens < 1:
            raise ValueError("layers, kv_heads, pages and max_tokens must be positive")
        if not 1 <= batch <= 32767:
            raise ValueError(f"batch must be in 1..32767, got {batch}")
        if head_dim < 64 or head_dim > 128 or head_dim % 16:
            raise ValueError(f"head_dim must be a multiple of 16 in 64..128, got {head_dim}")
        if page not in (16, 32, 64, 128):
            raise ValueError(f"page must be 16, 32, 64 or 128, got {page}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"dtype must be bfloat16 or float16, got {dtype}")
        if max_tokens > 1 << 30 or pages * kv_heads * page > (1 << 31) - 1:
            raise ValueError("at most 2^30 tokens a sequence and 2^31 - 1 rows in a layer's pool")
        self.layers, self.batch, self.kv_heads, self.head_dim = layers, batch, kv_heads, head_dim
        self.pages, self.page, self.dtype = pages, page, dtype
        width = -(-max_tokens // page)
        self.capacity = width * page
        self.ctx = Context.get(device)
        dev = self.device = torch.device("cuda", self.ctx.device)
        self.keys = torch.zeros(layers, pages, kv_heads, page, head_dim, dtype=dtype, device=dev)
        self.values = torch.zeros_like(self.keys)
        self.table = torch.full((batch, width), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self._status = self.status.data_ptr()
        self._lib = lib = _lib.load()
        self._append, self._attention, self._accept = lib.kt_paged_append, lib.kt_paged_attention, lib.kt_paged_accept
        self.scratch = torch.empty(lib.kt_paged_scratch_bytes(self.ctx.handle), dtype=torch.uint8, device=dev)
        self.scratch[:COUNTER_BYTES].zero_()
        self._scratch = self.scratch.data_ptr()
        self._scale = 1.0 / math.sqrt(head_dim)
        self._types = {dtype: _lib.KT_BF16 if dtype is torch.bfloat16 else _lib.KT_FP16, torch.float32: _lib.KT_FP32}
        self._free = list(range(pages - 1, -1, -1))
        self._own = [[] for _ in range(batch)]
        self._first = 0  # of the whole cache's sequences, for a view
        self._results = {}  # of accept, by rows
        self._describe()

    def _describe(self) -> None:
        self._cache = _lib.KtPagedCache(self.keys.data_ptr(), self.values.data_ptr(), self.table.data_ptr(),
                                        self.lengths.data_ptr(), self.layers, self.batch, self.kv_heads, self.head_dim,
                                        self.pages, self.page, self.table.shape[1], self.table.shape[1],
                                        self._types[self.dtype])
        self._ref = ctypes.byref(self._cache)

    def sequences(self, begin: int, end: int) -> "PagedKVCache":
        """A view of sequences begin..end-1: the same buffers, pool and scratch."""
        if not 0 <= begin < end <= self.batch:
            raise ValueError(f"sequences {begin}..{end} of {self.batch}")
        view = copy.copy(self)
        view.batch, view._first = end - begin, self._first + begin
        view.table, view.lengths, view._results = self.table[begin:end], self.lengths[begin:end], {}
        view._describe()
        return view

    # -- pages
    @property
    def free_pages(self) -> int:
        """Pages that ``reserve`` can still hand out."""
        return len(self._free)

    def reserve(self, sequence, tokens: int) -> None:
        """Pages for the first ``tokens`` slots of a sequence, or of each of several (those they
        have stay).  Where the pool has too few, nobody gets any."""
        try:
            sequences = [operator.index(sequence)]
        except TypeError:
            sequences = list(dict.fromkeys(sequence))
        owns = [self._pages_of(q) for q in sequences]
        if not 0 <= tokens <= self.capacity:
            raise ValueError(f"{tokens} tokens do not fit a sequence of {self.capacity}")
        pages = -(-tokens // self.page)
        n = sum(max(0, pages - len(own)) for own in owns)
        if n > len(self._free):
            raise ValueError(f"{n} pages wanted, {len(self._free)} are free")
        for q, own in zip(sequences, owns):
            more = pages - len(own)
            if more > 0:
                new = self._free[:-more - 1:-1]
                self.table[q, len(own):pages] = torch.tensor(new, dtype=torch.int32, device=self.device)
                del self._free[-more:]
                own += new

    def release(self, sequence: int) -> None:
        """Empties a sequence; its pages may be handed out again to calls that come after
        this one on the stream."""
        own = self._pages_of(sequence)
        self._free += reversed(own)
        own.clear()
        self.table[sequence].fill_(-1)
        self.lengths[sequence].zero_()

    def _pages_of(self, sequence: int) -> list:
        if not 0 <= sequence < self.batch:
            raise ValueError(f"sequence {sequence} of {self.batch}")
        return self._own[self._first + sequence]

    def reset(self) -> None:
        """Empties every sequence; pages stay with the sequences that have them."""
        self.lengths.zero_()
        self.status.zero_()

    # -- calls
    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} of {self.layers}")
        return layer

    def _ints(self, name: str, x, shape):
        """Pointer of a contiguous int32 array on the device, or None."""
        if x is None:
            return None
        if x.get_device() != self.ctx.device or x.dtype is not torch.int32 or x.shape != shape or not x.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor of shape {list(shape)} on {self.device}, got "
                             f"{str(x.dtype).replace('torch.', '')} {list(x.shape)} on {x.device}")
        return x.data_ptr()

    def _result(self, name: str, x, rows: int, width: int, dtypes):
        if x.get_device() != self.ctx.device or x.dtype not in dtypes or x.shape != (rows, width) or not x.is_contiguous():
            raise ValueError(f"{name} must be a contiguous tensor of shape [{rows}, {width}] of the cache's type on "
                             f"{self.device}, got {str(x.dtype).replace('torch.', '')} {list(x.shape)} on {x.device}")
        return x.data_ptr()

    def append(self, layer: int, q, k, v, inv_freq, rows_per_seq: int = 1, counts=None, depths=None, out=None):
        """Row b * rows_per_seq + t of float32 ``q`` [batch * rows_per_seq, heads * head_dim]
        (or None), ``k`` and ``v`` [batch * rows_per_seq, kv_heads * head_dim] is the token in
        slot lengths[b] + t, at position lengths[b] + ``depths``[b, t] (int32 [batch,
        rows_per_seq]; t unless given).  Queries and keys are rotated by angles position *
        ``inv_freq`` (float32 [head_dim / 2]); keys and values are stored, the queries returned in
        the cache's type (``out``).  ``counts`` (int32 [batch]): only the first counts[b] rows
        of a sequence are tokens.  Tokens without a page are dropped and set ``status``."""
        rows, device = self.batch * rows_per_seq, self.ctx.device
        qp = qs = heads = None
        if q is not None:
            heads = q.shape[1] // self.head_dim if q.dim() == 2 else 0
            qp, qs = _rows("q", q, rows, heads * self.head_dim, device)
            if out is None:
                out = torch.empty((rows, heads * self.head_dim), dtype=self.dtype, device=self.device)
            to = self._result("out", out, rows, heads * self.head_dim, (self.dtype,))
        elif out is not None:
            raise ValueError("out is for queries")
        width = self.kv_heads * self.head_dim
        kp, ks = _rows("k", k, rows, width, device)
        vp, vs = _rows("v", v, rows, width, device)
        if inv_freq.get_device() != device or inv_freq.dtype is not torch.float32 or inv_freq.numel() != self.head_dim // 2 or \
                not inv_freq.is_contiguous():
            raise ValueError(f"inv_freq must be a contiguous float32 tensor of {self.head_dim // 2} elements on {self.device}")
        _lib.check(self._append(self.ctx.handle, self._ref, self._layer(layer), qp, kp, vp, qs or 0, ks, vs, heads or 0,
                                inv_freq.data_ptr(), rows_per_seq, self._ints("counts", counts, (self.batch,)),
                                self._ints("depths", depths, (self.batch, rows_per_seq)), None if q is None else to,
                                self._status, raw_stream(device)))
        return out

    def attend(self, layer: int, q, heads: int, rows_per_seq: int = 1, counts=None, visible=None,
               scale: Optional[float] = None, out=None):
        """Attention of row t of every sequence over slots 0..lengths[b]-1 and the call's tokens
        (``append`` of the same rows comes first) up to itself, or those whose bits are set in
        ``visible`` (int32 [batch, rows_per_seq, (rows_per_seq + 31) // 32], ``draft_tree``).  ``q``
        [batch * rows_per_seq, heads * head_dim] of the cache's type; the result has its
        type, or ``out``'s (the cache's or float32; ``q`` itself where its rows have no gaps).
        ``scale`` is 1 / sqrt(head_dim) unless given.  Rows that see nothing, or are no tokens
        by ``counts``, give zeros."""
        rows, width, device = self.batch * rows_per_seq, heads * self.head_dim, self.ctx.device
        if q.dtype is not self.dtype or q.get_device() != device or q.shape != (rows, width):
            raise ValueError(f"q must be a {str(self.dtype).replace('torch.', '')} tensor of shape [{rows}, {width}] on "
                             f"{self.device}, got {str(q.dtype).replace('torch.', '')} {list(q.shape)} on {q.device}")
        stride, column = q.stride()
        if column != 1 or (rows > 1 and stride < width):
            raise ValueError("q must have contiguous rows that do not overlap")
        if out is None:
            out = torch.empty((rows, width), dtype=self.dtype, device=self.device)
        to = self._result("out", out, rows, width, self._types)
        _lib.check(self._attention(self.ctx.handle, self._ref, self._layer(layer), q.data_ptr(), stride if stride > width else width,
                                   to, self._types[out.dtype], rows_per_seq, self._ints("counts", counts, (self.batch,)),
                                   self._ints("visible", visible, (self.batch, rows_per_seq, (rows_per_seq + 31) // 32)), heads,
                                   self._scale if scale is None else scale, self._scratch, raw_stream(device)))
        return out

    def accept(self, tokens, parents, choices, counts=None, accepted=None, taken=None):
        """The path of each drafted tree that the model's ``choices`` confirm: from node 0 on, the
        lowest child whose token is its parent's choice (``tokens``, ``parents``, ``choices`` int32
        [batch, rows], the rows of the last ``append``; ``counts``: nodes of each tree).  Moves
        the path's keys and values of every layer to the slots behind the text and returns
        ``accepted`` (int32 [batch, rows]: the choices along the path, then -1) and ``taken``
        (int32 [batch]: the path's nodes), by which ``advance(rows, counts=taken)`` moves on:
        those given (no memory that the call reads), or buffers of this object that its next call
        with as many rows overwrites."""
        rows = tokens.shape[1] if tokens.dim() == 2 else 0
        shape = (self.batch, rows)
        given = (self._ints("tokens", tokens, shape), self._ints("parents", parents, shape), self._ints("choices", choices, shape),
                 rows, self._ints("counts", counts, (self.batch,)))
        if rows < 1:
            raise ValueError("a drafted tree has a node at least")
        if accepted is None or taken is None:
            mine = self._results.get(rows)
            if mine is None:
                mine = self._results[rows] = (torch.empty(shape, dtype=torch.int32, device=self.device),
                                              torch.empty(self.batch, dtype=torch.int32, device=self.device))
            accepted, taken = mine[0] if accepted is None else accepted, mine[1] if taken is None else taken
        _lib.check(self._accept(self.ctx.handle, self._ref, *given, self._ints("accepted", accepted, shape),
                                self._ints("taken", taken, (self.batch,)), self._status, raw_stream(self.ctx.device)))
        return accepted, taken

    def advance(self, rows: int = 1, counts=None) -> None:
        """lengths[b] += rows, or counts[b] between 0 and rows; at most the capacity."""
        _lib.check(self._lib.kt_kv8_advance(self.ctx.handle, self.lengths.data_ptr(), self.batch, rows,
                                            self._ints("counts", counts, (self.batch,)), self.capacity, raw_stream(self.ctx.device)))
