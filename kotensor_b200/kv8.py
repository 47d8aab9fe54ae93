"""Key/value cache in 8 bits for decoding, with eviction by accumulated attention
weight (kt_kv8_* in include/kt_cuda.h).

The reference's KVCache (Engine/kotensor/src/main/kotlin/KVCache.kt:3-59) keeps
float32 keys and values; this cache keeps signed bytes with one float32 scale for
every ``block`` slots of a head, a quarter of the memory and of the bytes a decode
step reads.  ``store`` quantizes new tokens, ``attend`` runs attention over what is
held (one query row per sequence while decoding, a block of rows for a prompt) and
can add up the weight each slot received, ``evict`` prunes every head to the slots
that received most.  One cache serves all layers; sequences may hold different
numbers of tokens (``lengths``, on the device).
"""
from __future__ import annotations

import copy
import ctypes
import math
from typing import Optional

from . import _lib
from .quantized import Context, raw_stream

try:
    import torch
except ImportError:  # pragma: no cover
    torch = None


def _rows(name: str, x, rows: int, width: int, device: int):
    """Pointer and row stride of float32 rows on the device (rows may lie apart, as
    in a fused q|k|v projection)."""
    if x.dtype is not torch.float32 or x.get_device() != device or x.shape != (rows, width):
        raise ValueError(f"{name} must be a float32 tensor of shape [{rows}, {width}] on cuda:{device}, got "
                         f"{str(x.dtype).replace('torch.', '')} {list(x.shape)} on {x.device}")
    stride, column = x.stride()
    if column != 1 or (rows > 1 and stride < width):
        raise ValueError(f"{name} must have contiguous rows that do not overlap")
    return x.data_ptr(), stride if stride > width else width


def _zeroed(need: int, device):
    """Scratch whose counters, at its front, are zero as its first use needs them."""
    buffer = torch.empty(need, dtype=torch.uint8, device=device)
    buffer[:4096].zero_()
    return buffer


class _Scratch:
    """Scratch that grows with the calls that use it.  A buffer that is outgrown is freed
    once the stream is past its last use, unless a captured graph refers to it, or all
    are to stay."""

    def __init__(self, device, stays: bool):
        self.buffer = self.graphs = torch.empty(0, dtype=torch.uint8, device=device)
        self.stays, self.captured, self.kept = stays, stays, []
        self.at = {}  # pointer for the (rows_per_seq, heads) of earlier calls

    def of(self, sizes, need: int) -> int:
        """Pointer to at least `need` bytes."""
        capturing = torch.cuda.is_current_stream_capturing()
        if need > self.buffer.numel():
            if capturing:
                return self.of_graph(need)
            if self.captured:
                self.kept.append(self.buffer)
            else:
                self.at.clear()
                if self.buffer.numel():
                    self.buffer.record_stream(torch.cuda.current_stream(self.buffer.device))
            self.buffer, self.captured = _zeroed(need, self.buffer.device), self.stays
        self.captured = self.captured or capturing
        self.at[sizes] = self.buffer.data_ptr()
        return self.at[sizes]

    def of_graph(self, need: int) -> int:
        """A buffer made while a graph is captured would be zeroed by its replays, not for a
        call before them: it serves graphs alone, zeroed at each use."""
        if need > self.graphs.numel():
            self.kept.append(self.graphs)
            self.graphs = _zeroed(need, self.buffer.device)
        else:
            self.graphs[:4096].zero_()
        return self.graphs.data_ptr()


class KVCache8:
    """An 8-bit cache of ``layers`` layers, ``batch`` sequences and ``kv_heads``
    heads of ``head_dim`` (a multiple of 16 up to 128), ``capacity`` slots each
    (rounded up to whole blocks); ``block`` (16, 32 or 64) slots share a scale.
    ``track_weights`` keeps the accumulated attention weights that ``evict`` needs.

    k_codes, v_codes   int8    [layers, batch, kv_heads, capacity, head_dim]
    k_scales, v_scales float32 [layers, batch, kv_heads, capacity / block]
    k_tail, v_tail     float32 [layers, batch, kv_heads, block, head_dim]
    weights            float32 [layers, batch, kv_heads, capacity], or None
    lengths            int32   [batch], tokens held by each sequence

    ``store`` and ``attend`` of every layer work at the same ``lengths``;
    ``advance`` moves on after the last layer.  Calls run on the current stream of
    the cache's device and share one scratch buffer: order them on one stream.
    """

    def __init__(self, layers: int, batch: int, kv_heads: int, head_dim: int, capacity: int, block: int = 64,
                 track_weights: bool = False, device: Optional[int] = None):
        if layers < 1 or kv_heads < 1 or capacity < 1:
            raise ValueError("layers, kv_heads and capacity must be positive")
        if not 1 <= batch <= 32767:
            raise ValueError(f"batch must be in 1..32767, got {batch}")
        if head_dim < 16 or head_dim > 128 or head_dim % 16:
            raise ValueError(f"head_dim must be a multiple of 16 in 16..128, got {head_dim}")
        if block not in (16, 32, 64):
            raise ValueError(f"block must be 16, 32 or 64, got {block}")
        self.layers, self.batch, self.kv_heads, self.head_dim, self.block = layers, batch, kv_heads, head_dim, block
        self.capacity = capacity = -(-capacity // block) * block
        self.ctx = Context.get(device)
        dev = self.device = torch.device("cuda", self.ctx.device)
        shape = (layers, batch, kv_heads)
        self.k_codes = torch.zeros(*shape, capacity, head_dim, dtype=torch.int8, device=dev)
        self.v_codes = torch.zeros_like(self.k_codes)
        self.k_scales = torch.zeros(*shape, capacity // block, dtype=torch.float32, device=dev)
        self.v_scales = torch.zeros_like(self.k_scales)
        self.k_tail = torch.zeros(*shape, block, head_dim, dtype=torch.float32, device=dev)
        self.v_tail = torch.zeros_like(self.k_tail)
        self.weights = torch.zeros(*shape, capacity, dtype=torch.float32, device=dev) if track_weights else None
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self._status = self.status.data_ptr()
        self._new_scratch()
        lib = _lib.load()
        self._lib, self._store, self._attention = lib, lib.kt_kv8_store, lib.kt_kv8_attention
        self._scale = 1.0 / math.sqrt(head_dim)
        self._describe()

    def _describe(self) -> None:
        """The C descriptor of every layer."""
        buffers = (self.k_codes, self.v_codes, self.k_scales, self.v_scales, self.k_tail, self.v_tail, self.weights)
        self._layer = []
        for l in range(self.layers):
            s = _lib.KtKv8Cache(*(None if t is None else t[l].data_ptr() for t in buffers), self.lengths.data_ptr(),
                                self.batch, self.kv_heads, self.head_dim, self.capacity, self.block)
            self._layer.append((s, ctypes.byref(s)))

    def sequences(self, begin: int, end: int) -> "KVCache8":
        """A view of sequences begin..end-1: the same buffers, its own scratch."""
        if not 0 <= begin < end <= self.batch:
            raise ValueError(f"sequences {begin}..{end} of {self.batch}")
        view = copy.copy(self)
        view.batch, view.lengths = end - begin, self.lengths[begin:end]
        for name in ("k_codes", "v_codes", "k_scales", "v_scales", "k_tail", "v_tail", "weights"):
            t = getattr(self, name)
            setattr(view, name, None if t is None else t[:, begin:end])
        view._new_scratch()
        view._describe()
        return view

    def _cache(self, layer: int):
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} of {self.layers}")
        return self._layer[layer][1]

    def _counts(self, counts):
        if counts is None:
            return None
        if counts.get_device() != self.ctx.device or counts.dtype != torch.int32 or counts.shape != (self.batch,) or \
                not counts.is_contiguous():
            raise ValueError(f"counts must be a contiguous int32 tensor of {self.batch} elements on {self.device}")
        return counts.data_ptr()

    def _new_scratch(self) -> None:
        self._steps, self._prompts = _Scratch(self.device, stays=True), _Scratch(self.device, stays=False)

    def _scratch_of(self, rows_per_seq: int, heads: int):
        """Scratch of this call's sizes.  Calls that need no more than a single-token step,
        whose size only the heads change, share the steps': it stays where it is through
        prompts of any length, so that these short calls need not ask for a capture (0.4 of
        2 rows' 5.6 us)."""
        sizes = rows_per_seq, heads
        at = self._steps.at.get(sizes)
        if at is not None:
            return at
        at = self._prompts.at.get(sizes)
        if at is not None and (self._prompts.captured or not torch._C._cuda_isCurrentStreamCapturing()):
            return at
        step, need = (self._lib.kt_kv8_scratch_bytes(self.batch, rows, heads, self.kv_heads, self.head_dim, self.capacity,
                                                     self.weights is not None) for rows in (1, rows_per_seq))
        return (self._steps if need <= step else self._prompts).of(sizes, need)

    def store(self, layer: int, k, v, rows_per_seq: int = 1, counts=None) -> None:
        """Row b * rows_per_seq + t of ``k`` and ``v`` ([batch * rows_per_seq, kv_heads *
        head_dim], keys already rotated) into slot lengths[b] + t.  ``counts`` (int32
        [batch]): only the first counts[b] rows of a sequence are tokens.  Tokens past
        the capacity are dropped and set ``status``."""
        rows, width = self.batch * rows_per_seq, self.kv_heads * self.head_dim
        kp, ks = _rows("k", k, rows, width, self.ctx.device)
        vp, vs = _rows("v", v, rows, width, self.ctx.device)
        _lib.check(self._store(self.ctx.handle, self._cache(layer), kp, vp, ks, vs, rows_per_seq, self._counts(counts),
                               self._status, raw_stream(self.ctx.device)))

    def attend(self, layer: int, q, heads: int, rows_per_seq: int = 1, scale: Optional[float] = None, out=None,
               counts=None, accumulate: bool = False):
        """Attention of row t of every sequence over slots 0..lengths[b] + t (``store`` of
        the same rows comes first): ``q`` and the result are [batch * rows_per_seq,
        heads * head_dim]; ``scale`` is 1 / sqrt(head_dim) unless given.
        ``accumulate`` adds the attention weights to ``weights``."""
        rows, width = self.batch * rows_per_seq, heads * self.head_dim
        qp, qs = _rows("q", q, rows, width, self.ctx.device)
        if out is None:
            out = q.new_empty((rows, width))
        elif out.get_device() != self.ctx.device or out.dtype != torch.float32 or tuple(out.shape) != (rows, width) or \
                not out.is_contiguous():
            raise ValueError(f"out must be a contiguous float32 tensor of shape [{rows}, {width}] on {self.device}")
        scratch = self._scratch_of(rows_per_seq, heads) if rows_per_seq > 0 and heads > 0 else None
        _lib.check(self._attention(self.ctx.handle, self._cache(layer), qp, qs, out.data_ptr(), rows_per_seq,
                                   self._counts(counts), heads, self._scale if scale is None else scale, accumulate,
                                   scratch, raw_stream(self.ctx.device)))
        return out

    def advance(self, rows: Optional[int] = None, counts=None, limit: Optional[int] = None) -> None:
        """lengths[b] += what ``store`` of the same ``rows`` (1 unless given) and ``counts`` added:
        rows, or counts[b] between 0 and rows (the capacity unless given); at most ``limit``
        (the capacity unless given)."""
        if rows is None:
            rows = 1 if counts is None else self.capacity
        _lib.check(self._lib.kt_kv8_advance(self.ctx.handle, self.lengths.data_ptr(), self.batch, rows,
                                            self._counts(counts), self.capacity if limit is None else limit,
                                            raw_stream(self.ctx.device)))

    def evict_layer(self, layer: int, keep: int, recent: int) -> None:
        """Prunes one layer's sequences of more than ``keep`` tokens to the ``recent`` last
        ones and the others of largest accumulated weight, each head for itself;
        ``lengths`` stays (see ``evict``)."""
        _lib.check(self._lib.kt_kv8_evict(self.ctx.handle, self._cache(layer), keep, recent, self._scratch_of(1, self.kv_heads),
                                          raw_stream(self.ctx.device)))

    def evict(self, keep: int, recent: int) -> None:
        """``evict_layer`` on every layer, then lengths[b] = min(lengths[b], keep)."""
        for layer in range(self.layers):
            self.evict_layer(layer, keep, recent)
        self.advance(0, limit=keep)

    def reset(self) -> None:
        """Empties every sequence."""
        self.lengths.zero_()
        self.status.zero_()
