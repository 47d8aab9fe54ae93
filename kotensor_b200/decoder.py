"""Device-resident greedy decode step: Transformer.decode
(Engine/kotensor/src/main/kotlin/Transformer.kt:141-154) with every layer
(TransformerBlock.decodeInto, TransformerBlock.kt:40-47; Attention.decodeInto,
Attention.kt:207-239; SwiGLU.forwardInto, SwiGLU.kt:19-25) on the GPU: the
projections are the quantized matmul (kt_qmatmul, with QuantizedLinear's bias),
the rest are the decode kernels of libkt_cuda.so (kt_rmsnorm, kt_rope,
kt_kv_store, kt_attention_decode, kt_silu_mul, kt_add, kt_argmax, the
quantized / tied embedding lookups).  The token id and position live on the
device, so one step is captured into a CUDA graph and replayed per token with
no host work between tokens.  The KV cache has the reference's layout
(KVCache.kt:3-59): fp32 [layers][kvHeads][maxSeq][headDim].
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Optional

import numpy as np

from . import _lib
from .quantized import Context, MatMul, QuantizedTensor

try:
    import torch
except ImportError:  # pragma: no cover
    torch = None


@dataclass
class DecoderConfig:
    """Transformer(vocabularySize, dimension, numLayers, numHeads, hiddenDimension,
    numKeyValueHeads, normEps, ropeTheta, ropeScaling, quantization), Transformer.kt:3-14."""
    vocab: int
    dim: int
    layers: int
    heads: int
    kv_heads: int
    hidden: int
    eps: float = 1e-6
    rope_theta: float = 10000.0
    rope_scaling: Optional[tuple] = None  # RoPEScaling(factor, low, high, originalMaxPositions)
    bits: int = 4
    group_size: int = 64
    tied: bool = False        # Transformer.tieEmbeddingToHead (Transformer.kt:380-386)
    qkv_bias: bool = False

    @property
    def head_dim(self) -> int:
        return self.dim // self.heads


def rope_inv_freq(head_dim: int, base: float, scaling: Optional[tuple]) -> np.ndarray:
    """RoPE.invFreq (RoPE.kt:39-42) and RoPEScaling.scale (RoPE.kt:15-27) in float32."""
    half = head_dim // 2
    out = np.empty(half, np.float32)
    for i in range(half):
        raw = np.float32(1.0) / np.float32(math.pow(float(np.float32(base)),
                                                    float(np.float32(2 * i) / np.float32(head_dim))))
        if scaling is not None:
            factor, low, high = np.float32(scaling[0]), np.float32(scaling[1]), np.float32(scaling[2])
            orig = np.float32(int(scaling[3]))
            wl = np.float32(2.0 * math.pi / float(raw))
            if wl < orig / high:
                pass
            elif wl > orig / low:
                raw = raw / factor
            else:
                smooth = (orig / wl - low) / (high - low)
                raw = (np.float32(1.0) - smooth) * raw / factor + smooth * raw
        out[i] = np.float32(raw)
    return out


def tensor_parallel_plan(cfg: DecoderConfig, parts: int, rank: int) -> dict:
    """Rank ``rank``'s share of a decoder split over ``parts`` ranks: query and
    key/value heads (contiguous blocks), the columns [q0, q1) of the query
    projection (= the rows of the output projection), [k0, k1) of the key and
    value projections, the block [h0, h1) of whole groups of the hidden width
    (gate / up columns, down-projection rows) and the lm head's vocabulary
    columns [v0, v1).  Requires heads and kv_heads divisible by ``parts`` and
    the output projection's rows to split on group boundaries."""
    from .parallel import COLUMNS, ROWS, shard_bounds
    if parts < 1 or not 0 <= rank < parts:
        raise ValueError(f"rank {rank} of {parts}")
    if cfg.heads % parts or cfg.kv_heads % parts:
        raise ValueError(f"{cfg.heads} query / {cfg.kv_heads} key-value heads do not split over {parts} ranks")
    hd, g = cfg.head_dim, cfg.group_size
    heads, kv = cfg.heads // parts, cfg.kv_heads // parts
    q0, q1 = rank * heads * hd, (rank + 1) * heads * hd
    k0, k1 = rank * kv * hd, (rank + 1) * kv * hd
    if parts > 1 and (q0 % g or (q1 % g and q1 != cfg.dim)):
        raise ValueError(f"{q1 - q0} output-projection rows per rank is not a multiple of the group size {g}")
    hidden = shard_bounds(ROWS, cfg.hidden, g, parts, rank) if parts > 1 else (0, cfg.hidden)
    vocab = shard_bounds(COLUMNS, cfg.vocab, g, parts, rank) if parts > 1 else (0, cfg.vocab)
    return {"heads": heads, "kv_heads": kv, "q": (q0, q1), "kv": (k0, k1), "hidden": hidden, "vocab": vocab}


def _upload(w) -> QuantizedTensor:
    """A QuantizedTensor, or host arrays in the reference layout (objects with
    qdata / scales / zeros / rows / columns / bits / group_size)."""
    if isinstance(w, QuantizedTensor):
        return w
    return QuantizedTensor.from_arrays(w.qdata, w.scales, w.zeros, (w.rows, w.columns), w.bits, w.group_size)


class _Rows:
    """Activation buffers for a block of rows (one decode step, or a prefill)."""


class DeviceDecoder:
    """Greedy decoding of one sequence with weights, KV cache and buffers in HBM.

    ``max_block_rows`` (65,535, the row kernels' grid limit) bounds the rows of
    one prefill block; a batch with more prompt rows is prefilled in blocks of
    whole sequences.

    ``weights``: ``embedding`` ([vocab x dim], None when tied), ``layers`` (a list
    of dicts with wq wk wv wo wg wu wd, their biases bq bk bv bo bg bu bd and the
    RMSNorm weights norm1 norm2), ``final_norm``, ``head`` ([dim x vocab]),
    ``head_bias``.  ``batch`` sequences decode together (one KV cache each, the
    same position): every matmul of a step runs at m = batch.

    ``comm`` (a parallel.Comm over P ranks, one process per GPU, every rank
    building the decoder from the same weights): tensor parallelism
    (``tensor_parallel_plan``).  Rank r keeps its block of query heads and of
    key/value heads -- the q|k|v projection column-parallel over them,
    attention and its KV cache local -- the output projection row-parallel over
    the same rows, the gate|up projection column-parallel and the down
    projection row-parallel over one block of whole groups of the hidden width,
    and the lm head column-parallel over the vocabulary with the greedy argmax
    taken across shards (argmaxOfLastToken's rule, Transformer.kt:255-266).
    The two row-parallel products of a layer end in the only exchange: an
    all-reduce of [batch x dim] partial sums (fused into the m = 1 GEMV over
    peer memory, else NCCL), after which every rank holds the whole residual
    stream.

    ``kv_bits`` 16: keys and values in a PagedKVCache (``cache``) of ``kv_dtype`` (bfloat16
    unless given), half the fp32 cache's memory: ``kv_pages`` pages (enough for every
    sequence unless given) of ``kv_page`` positions, which sequences receive as they grow.
    ``generate_drafted`` then checks several drafted tokens in one pass.

    ``kv_bits`` 8: keys and values in a KVCache8 (``cache``) with a scale for every
    ``kv_block`` positions of a head, a quarter of the fp32 cache's memory and of the
    bytes a step's attention reads.  ``kv_weights`` also accumulates the attention
    weight every slot receives, by which ``evict`` prunes the cache.  ``penalize``
    puts penalties, biases and a grammar mask between the logits and the greedy
    choice."""

    max_block_rows = 65535

    def __init__(self, cfg: DecoderConfig, weights, max_seq: int, device: Optional[int] = None, batch: int = 1,
                 comm=None, kv_bits: int = 32, kv_block: int = 64, kv_weights: bool = False, kv_page: int = 64,
                 kv_pages: Optional[int] = None, kv_dtype=None):
        if kv_bits not in (8, 16, 32):
            raise ValueError(f"kv_bits must be 8, 16 or 32, got {kv_bits}")
        if kv_weights and kv_bits != 8:
            raise ValueError("attention weights are kept by the 8-bit cache only")
        self.cfg = cfg
        self.max_seq = max_seq
        self.ctx = Context.get(device)
        dev = torch.device("cuda", self.ctx.device)
        f32 = dict(dtype=torch.float32, device=dev)

        def vec(a):
            if isinstance(a, torch.Tensor):
                return a.detach().to(device=dev, dtype=torch.float32).reshape(-1).contiguous()
            return torch.as_tensor(np.ascontiguousarray(a, dtype=np.float32).reshape(-1)).to(dev)

        from .parallel import COLUMNS, ROWS, concat_columns, slice_weight
        self.comm = comm
        P = comm.world if comm is not None else 1
        plan = tensor_parallel_plan(cfg, P, comm.rank if comm is not None else 0)
        self.parts = P
        self.heads_local, self.kv_local = plan["heads"], plan["kv_heads"]
        q0, q1 = plan["q"]
        k0, k1 = plan["kv"]
        h0, h1 = plan["hidden"]
        v0, v1 = plan["vocab"]
        self.q_width, self.kv_width = q1 - q0, k1 - k0
        self.hidden_local, self.vocab_begin, self.vocab_local = h1 - h0, v0, v1 - v0

        def cols(w, b, e):
            return w if P == 1 else slice_weight(w, COLUMNS, b, e)

        self.layers = []
        for L in weights.layers:
            d = {k: (_upload(v) if k.startswith("w") else vec(v)) for k, v in L.items()}
            # q|k|v and gate|up as one matmul each: per-column quantization makes
            # the fused weight's columns exactly the separate weights' columns
            # (and a rank's column shard exactly those columns of the weight)
            d["wqkv"] = concat_columns([cols(d["wq"], q0, q1), cols(d["wk"], k0, k1), cols(d["wv"], k0, k1)])
            d["bqkv"] = torch.cat([d["bq"][q0:q1], d["bk"][k0:k1], d["bv"][k0:k1]])
            d["wgu"] = concat_columns([cols(d["wg"], h0, h1), cols(d["wu"], h0, h1)])
            d["bgu"] = torch.cat([d["bg"][h0:h1], d["bu"][h0:h1]])
            if P > 1:  # row-parallel: this rank's rows; the bias is added once, after the exchange
                d["wo"] = slice_weight(d["wo"], ROWS, q0, q1)
                d["wd"] = slice_weight(d["wd"], ROWS, h0, h1)
            for k in ("wq", "wk", "wv", "wg", "wu", "bq", "bk", "bv", "bg", "bu"):
                del d[k]
            self.layers.append(d)
        full_head = _upload(weights.head)
        self.head = cols(full_head, v0, v1)
        self.head_bias = vec(weights.head_bias)[v0:v1].contiguous()
        # tied embeddings look tokens up in the whole head (any column may be asked for)
        self.lookup_head = full_head if cfg.tied else None
        self.embedding = None if cfg.tied else _upload(weights.embedding)
        self.final_norm = vec(weights.final_norm)
        if batch < 1:
            raise ValueError(f"batch must be positive, got {batch}")
        self.batch = batch
        # one KV cache per sequence, each in the reference's layout [L][kvH][maxSeq][hd]
        # (this rank's key/value heads under tensor parallelism)
        self.cache = self.keys = self.values = None
        self.paged = kv_bits == 16
        if kv_bits == 8:
            from .kv8 import KVCache8
            self.cache = KVCache8(cfg.layers, batch, self.kv_local, cfg.head_dim, max_seq, kv_block, kv_weights, self.ctx.device)
            self.cache._scratch_of(1, self.heads_local)  # what a captured step needs
        elif kv_bits == 16:
            from .paged import PagedKVCache
            if kv_pages is None:
                kv_pages = batch * -(-max_seq // kv_page)
            self.cache = PagedKVCache(cfg.layers, batch, self.kv_local, cfg.head_dim, kv_pages, max_seq, kv_page, kv_dtype,
                                      self.ctx.device)
        else:
            self.keys = torch.zeros((batch, cfg.layers, self.kv_local, max_seq, cfg.head_dim), **f32)
            self.values = torch.zeros_like(self.keys)
        self.cache_stride = cfg.layers * self.kv_local * max_seq * cfg.head_dim
        self.inv_freq = vec(rope_inv_freq(cfg.head_dim, cfg.rope_theta, cfg.rope_scaling))
        self.token = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.next_token = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.position = torch.zeros(1, dtype=torch.int32, device=dev)  # shared: sequences advance together
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)
        self.logits = torch.empty((batch, self.vocab_local), **f32)  # this rank's vocabulary columns
        self._head_in = torch.empty((batch, cfg.dim), **f32)
        self._head_xn = torch.empty((batch, cfg.dim), **f32)
        self._last_rows = torch.empty(batch, dtype=torch.int32, device=dev)
        self._step_bufs = self._buffers(batch, tokens=self.token)
        self._prefill_bufs = None  # prefill buffers, allocated on first use
        self.length = 0    # tokens processed
        self._evicted = 0  # of them, no longer in the cache
        self._penal = None
        self._text, self._prompt_end = [], 0  # int32 [batch, n] of each call, tokens up to the last prompt's end
        self.scale = float(np.float32(1.0) / np.float32(math.sqrt(float(cfg.head_dim))))
        self._graph = None
        self._drafts = None  # buffers and graph of generate_drafted's passes
        self.passes = 0      # of its last call
        g_ = self.heads_local // self.kv_local
        self._fused_attention = g_ <= 8 and cfg.head_dim in (64, 128) and max_seq <= 16384
        if P > 1:
            self._warm_exchanges()

    # -- helpers
    @staticmethod
    def _p(t) -> ctypes.c_void_p:
        return ctypes.c_void_p(t.data_ptr())

    def _stream(self) -> ctypes.c_void_p:
        return ctypes.c_void_p(torch.cuda.current_stream(self.ctx.device).cuda_stream)

    @property
    def held(self) -> int:
        """Positions in the cache (fewer than ``length`` after an eviction)."""
        return self.length - self._evicted

    def reset(self) -> None:
        self.length = self._evicted = 0
        self._text, self._prompt_end = [], 0
        self.position.zero_()
        if self.cache is not None:
            self.cache.reset()
        if self._penal is not None:
            self._lay_out(self._history[:, :0], 0)

    def _buffers(self, rows: int, tokens=None) -> "_Rows":
        cfg = self.cfg
        dev = self.position.device
        f32 = dict(dtype=torch.float32, device=dev)
        kv = cfg.kv_heads * cfg.head_dim
        b = _Rows()
        b.rows = rows
        b.x = torch.empty((rows, cfg.dim), **f32)
        b.normed = torch.empty((rows, cfg.dim), **f32)
        b.qkv = torch.empty((rows, self.q_width + 2 * self.kv_width), **f32)
        b.ctx = torch.empty((rows, self.q_width), **f32)
        b.gu = torch.empty((rows, 2 * self.hidden_local), **f32)
        b.act = torch.empty((rows, self.hidden_local), **f32)
        # rotated queries in the paged cache's type
        b.q16 = torch.empty((rows, self.q_width), dtype=self.cache.dtype, device=dev) if self.paged else None
        b.tokens = tokens if tokens is not None else torch.empty(rows, dtype=torch.int32, device=dev)
        # attention scratch; zero-filled: its tail holds the fused kernel's merge counters
        # (the 8-bit cache has its own)
        b.scores = None if self.cache is not None else torch.zeros(
            _lib.load().kt_attention_scratch_floats(rows, self.heads_local, cfg.head_dim, self.max_seq), **f32)
        return b

    def _row_parallel(self, x, w, out, rows: int, bias, accumulate: bool = True) -> None:
        """out[rows x dim] (+)= x . W + bias (the residual add of
        TransformerBlock.decodeInto): the local product, or under tensor
        parallelism this rank's rows of W and the all-reduce of the partials."""
        if self.comm is None:
            MatMul.multiply_quantized(x, w, out, rows, accumulate=accumulate, bias=bias)
        else:
            from .parallel import matmul_row_parallel
            matmul_row_parallel(self.comm, x, w, out, rows, accumulate=accumulate, bias=bias)

    def _warm_exchanges(self) -> None:
        """Collective (every rank, at construction): each row-parallel shard
        agrees its exchange once at m = batch (the fused peer-memory GEMV at
        m = 1 is set up and agreed on its first call, and the agreement
        synchronizes the stream, which a CUDA graph capture cannot), and the
        communicator's scratch grows to the step's size, so a captured step
        neither sets up nor allocates."""
        dev = self.position.device
        m = self.batch
        x_o = torch.zeros((m, self.q_width), dtype=torch.float32, device=dev)
        x_d = torch.zeros((m, self.hidden_local), dtype=torch.float32, device=dev)
        out = torch.empty((m, self.cfg.dim), dtype=torch.float32, device=dev)
        for L in self.layers:
            self._row_parallel(x_o, L["wo"], out, m, None, accumulate=False)
            self._row_parallel(x_d, L["wd"], out, m, None, accumulate=False)
        from .parallel import argmax_column_parallel
        self.logits.zero_()
        argmax_column_parallel(self.comm, self.logits, self.vocab_begin, self.next_token)
        torch.cuda.current_stream(self.ctx.device).synchronize()

    def gather_logits(self):
        """The whole [batch x vocab] logits on every rank (an all-gather of the
        ranks' vocabulary columns; the logits themselves when not sharded)."""
        if self.comm is None:
            return self.logits
        from .parallel import allgather_columns
        if self.cfg.vocab % self.parts:
            raise ValueError("the vocabulary does not split evenly: gather the shards with their offsets")
        full = torch.empty((self.batch, self.cfg.vocab), dtype=torch.float32, device=self.logits.device)
        allgather_columns(self.comm, self.logits, full, self.batch)
        return full

    def _reserve(self, positions: int) -> None:
        """Pages of the paged cache for so many positions of every sequence, or of none."""
        if self.paged:
            self.cache.reserve(range(self.batch), min(positions, self.cache.capacity))

    def _layers(self, b: "_Rows", rows: int, rows_per_seq: int, seq0: int = 0, counts=None, depths=None, visible=None) -> None:
        """Embedding lookup of b.tokens[:rows] through every block; leaves the
        residual rows in b.x (the head applies the final norm).  Row r is
        sequence seq0 + r / rows_per_seq at position *position + r %
        rows_per_seq (one sequence's prompt, or one token of each of `rows`
        sequences).  Per layer: norm1 + q|k|v, RoPE / cache / attention, the
        output projection added to the residual, norm2 + gate|up + SiLU * up,
        the down projection added to the residual -- five launches at batch 1,
        where the GEMV applies each norm while staging its input row and forms
        silu(gate) * up in its epilogue.  With a paged cache the rows of a sequence may be a
        drafted tree (``counts``, ``depths``, ``visible`` as PagedKVCache takes them)."""
        L_ = _lib.load()
        cfg, h = self.cfg, self.ctx.handle
        s, p = self._stream(), self._p
        if self.cache is None:
            keys = ctypes.c_void_p(self.keys.data_ptr() + seq0 * self.cache_stride * self.keys.element_size())
            values = ctypes.c_void_p(self.values.data_ptr() + seq0 * self.cache_stride * self.values.element_size())
        else:
            n = rows // rows_per_seq
            cache = self.cache if n == self.batch else self.cache.sequences(seq0, seq0 + n)
        hd, kvh = cfg.head_dim, self.kv_local
        kv = self.kv_width
        if cfg.tied:
            _lib.check(L_.kt_dequantize_column(h, self.lookup_head.handle, p(b.tokens), rows, p(b.x), p(self.status),
                                               s))
        else:
            _lib.check(L_.kt_dequantize_rows(h, self.embedding.handle, p(b.tokens), rows, p(b.x), p(self.status), s))
        for l, L in enumerate(self.layers):
            _lib.check(L_.kt_rmsnorm_qmatmul(h, L["wqkv"].handle, p(b.x), p(L["norm1"]), cfg.eps, p(b.normed),
                                             p(b.qkv), rows, 0, p(L["bqkv"]), s))
            if self.paged:
                q, k, v = b.qkv[:rows].split([self.q_width, kv, kv], 1)
                q = cache.append(l, q, k, v, self.inv_freq, rows_per_seq, counts, depths, out=b.q16[:rows])
                cache.attend(l, q, self.heads_local, rows_per_seq, counts, visible, self.scale, out=b.ctx[:rows])
            elif self.cache is not None:
                _lib.check(L_.kt_rope_seqs(h, p(b.qkv), rows, self.q_width, kvh, hd, p(self.inv_freq), p(self.position),
                                           rows_per_seq, s))
                q, k, v = b.qkv[:rows].split([self.q_width, kv, kv], 1)
                cache.store(l, k, v, rows_per_seq)
                cache.attend(l, q, self.heads_local, rows_per_seq, self.scale, out=b.ctx[:rows],
                             accumulate=cache.weights is not None)
            elif rows_per_seq == 1 and self._fused_attention and rows <= (16 if cfg.head_dim == 128 else 8):
                # one token per sequence: RoPE, cache store, attention and merge in one launch
                # (measured slower than the separate kernels once more sequences share a
                # step: beyond 16 at head_dim 128, beyond 8 at 64)
                _lib.check(L_.kt_attention_rope_decode(h, p(b.qkv), rows, self.q_width, self.heads_local, kvh, hd,
                                                       p(self.inv_freq), keys, values, p(b.ctx), p(b.scores),
                                                       self.max_seq, l, self.scale, p(self.position),
                                                       self.cache_stride, s))
            else:
                _lib.check(L_.kt_rope_kv_seqs(h, p(b.qkv), rows, self.q_width, kvh, hd, p(self.inv_freq), keys,
                                              values, self.max_seq, l, p(self.position), rows_per_seq,
                                              self.cache_stride, s))
                _lib.check(L_.kt_attention_seqs(h, p(b.qkv), keys, values, p(b.ctx), p(b.scores), rows,
                                                self.q_width + 2 * kv, self.heads_local, kvh, hd, self.max_seq, l,
                                                self.scale, p(self.position), rows_per_seq, self.cache_stride, s))
            self._row_parallel(b.ctx[:rows], L["wo"], b.x[:rows], rows, L["bo"])  # x += attention output
            _lib.check(L_.kt_rmsnorm_qmatmul_swiglu(h, L["wgu"].handle, p(b.x), p(L["norm2"]), cfg.eps,
                                                    p(b.normed), p(b.gu), p(b.act), rows, p(L["bgu"]), s))
            self._row_parallel(b.act[:rows], L["wd"], b.x[:rows], rows, L["bd"])  # x += feed-forward output

    def _head(self, x_rows, advance: int) -> None:
        """The final norm and the head on `batch` residual rows, greedy argmax
        per row, position += advance."""
        L_ = _lib.load()
        h, s, p = self.ctx.handle, self._stream(), self._p
        _lib.check(L_.kt_rmsnorm_qmatmul(h, self.head.handle, p(x_rows), p(self.final_norm), self.cfg.eps,
                                         p(self._head_xn), p(self.logits), self.batch, 0, p(self.head_bias), s))
        if self._penal is not None:  # penalties, biases, mask and the choice in one pass
            self._processor(self.logits, tokens=self._history, lengths=self._history_lengths,
                            prompt_lengths=self._prompt_lengths, next_token=self.next_token, **self._penal)
        elif self.comm is None:
            _lib.check(L_.kt_argmax(h, p(self.logits), self.batch, self.cfg.vocab, p(self.next_token), s))
        else:  # every rank's best column, merged across ranks: the same token everywhere
            from .parallel import argmax_column_parallel
            argmax_column_parallel(self.comm, self.logits, self.vocab_begin, self.next_token)
        _lib.check(L_.kt_increment(h, p(self.position), advance, s))
        if self.cache is not None:
            self.cache.advance(advance)
        self.token.copy_(self.next_token)

    def _launch_step(self, remember: bool = True) -> None:
        """One decode step on the current stream: reads self.token and
        self.position, writes self.logits and self.next_token, advances
        the position and feeds the next tokens back."""
        b = self._step_bufs
        if self._penal is not None and remember:  # the step's tokens join the history
            column, forgotten, length, after = self._places.index_select(0, self._place)[0].split(1)
            self._history.scatter_(1, forgotten.expand(self.batch, 1), -1)
            self._history.scatter_(1, column.expand(self.batch, 1), self.token[:, None])
            self._history_lengths.copy_(length.expand(self.batch))
            self._place.copy_(after)
        self._layers(b, self.batch, 1)
        self._head(b.x, 1)

    def _result(self):
        return self.logits[0] if self.batch == 1 else self.logits

    def prefill(self, prompts):
        """Transformer.prefill (Transformer.kt:99-132) for every sequence: each
        prompt (a list of token ids; one per sequence, equal lengths) runs as one
        block of rows through every layer (the matmuls at m = batch x T on the
        tensor-core GEMM, causal attention over each sequence's cache); returns
        the last tokens' logits and leaves their greedy successors in
        next_token / token."""
        if len(prompts) > 0 and not isinstance(prompts[0], (list, tuple, np.ndarray)):
            prompts = [prompts]
        if len(prompts) != self.batch:
            raise ValueError(f"{len(prompts)} prompts for a batch of {self.batch}")
        T = len(prompts[0])
        if T == 0:
            raise ValueError("Prompt cannot be empty")
        if any(len(pr) != T for pr in prompts):
            raise ValueError("prompts of one batch must have equal lengths")
        if any(not 0 <= t < self.cfg.vocab for pr in prompts for t in pr):
            raise ValueError("token out of vocab bounds")
        if self.held + T > self.max_seq:
            raise ValueError(f"KV cache full: {self.held} + {T} positions exceed maxSequenceLength {self.max_seq}")
        if T > self.max_block_rows:
            raise ValueError(f"{T} prompt tokens exceed {self.max_block_rows} rows of one prefill block")
        self._reserve(self.held + T)
        # whole sequences per block: a block holds at most max_block_rows rows (the
        # kernels' grid rows); larger batches are prefilled in several blocks
        per = min(self.batch, self.max_block_rows // T)
        if self._prefill_bufs is None or self._prefill_bufs.rows < per * T:
            self._prefill_bufs = self._buffers(per * T)
        if self.comm is not None:
            # a larger block may replace the communicator's scratch that a
            # captured step refers to: capture again before the next replay
            self._graph = None
        b = self._prefill_bufs
        flat = torch.tensor([t for pr in prompts for t in pr], dtype=torch.int32)
        if self._penal is not None:
            self._append_prompt(flat.view(self.batch, T))
        L_ = _lib.load()
        for s0 in range(0, self.batch, per):
            s1 = min(self.batch, s0 + per)
            rows = (s1 - s0) * T
            b.tokens[:rows].copy_(flat[s0 * T:s1 * T])
            self._layers(b, rows, T, seq0=s0)
            # the head only on each sequence's last row
            self._last_rows[:s1 - s0].copy_(torch.tensor([q * T + T - 1 for q in range(s1 - s0)], dtype=torch.int32))
            dst = ctypes.c_void_p(self._head_in.data_ptr() + s0 * self.cfg.dim * self._head_in.element_size())
            _lib.check(L_.kt_gather_rows(self.ctx.handle, self._p(b.x), self._p(self._last_rows), s1 - s0,
                                         self.cfg.dim, dst, self._stream()))
        self._head(self._head_in, T)
        self.length += T
        self._text.append(flat.view(self.batch, T).numpy())
        self._prompt_end = sum(t.shape[1] for t in self._text)
        return self._result()

    def step(self, tokens):
        """Transformer.decode(token) for every sequence (an int when batch == 1):
        the logits of this step (device tensor)."""
        return self._step(tokens)

    def _step(self, tokens, remember: bool = True):
        tokens = [tokens] if isinstance(tokens, (int, np.integer)) else list(tokens)
        if len(tokens) != self.batch:
            raise ValueError(f"{len(tokens)} tokens for a batch of {self.batch}")
        for t in tokens:
            if not 0 <= t < self.cfg.vocab:
                raise ValueError(f"{t} out of vocab bounds {self.cfg.vocab}")
        if self.held >= self.max_seq:
            raise ValueError(f"KV cache full: maxSequenceLength {self.max_seq}")
        self._reserve(self.held + 1)
        self.token.copy_(torch.tensor(tokens, dtype=torch.int32))
        self._launch_step(remember)
        self.length += 1
        self._text.append(np.array(tokens, dtype=np.int32)[:, None])
        return self._result()

    def capture(self) -> None:
        """Records one step (from the current self.token / self.position) into a CUDA graph."""
        torch.cuda.synchronize()
        self._graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self._graph):
            self._launch_step()

    def _check_room(self, prompt: int, max_tokens: int) -> None:
        """Refuses a generation that does not fit: nothing checks the replays of the
        captured step, and the last token chosen is not processed."""
        if prompt + max_tokens > self.max_seq:
            raise ValueError("prompt + max_tokens exceed max_seq")
        if self.held + prompt + max_tokens - 1 > self.max_seq:
            raise ValueError(f"KV cache full: {self.held} + {prompt} + {max_tokens - 1} positions exceed maxSequenceLength "
                             f"{self.max_seq}")
        self._reserve(self.held + prompt + max_tokens - 1)

    def _check_dropped(self) -> None:
        """An error if the 8-bit or paged cache, until ``reset``, had no room for a token it was given."""
        if self.cache is not None and int(self.cache.status.item()) != 0:
            raise ValueError("KV cache full: tokens were dropped")

    def generate(self, prompt: list[int], max_tokens: int) -> list[int]:
        """Greedy continuation of one sequence (batch 1): the prompt fed step by
        step (eager), then ``max_tokens`` replays of the captured step."""
        if self.batch != 1:
            raise ValueError("generate is for batch 1; use generate_batch")
        self._check_room(len(prompt), max_tokens)
        if any(not 0 <= t < self.cfg.vocab for t in prompt):
            raise ValueError("token out of vocab bounds")
        if self._penal is not None and len(prompt) > 0:
            self._append_prompt(torch.tensor([list(prompt)], dtype=torch.int32))
        for t in prompt:
            self._step(t, remember=False)
        if len(prompt) > 0:
            self._prompt_end = sum(t.shape[1] for t in self._text)
        out = [int(self.next_token[0].item())]
        if self._graph is None:
            self.capture()  # captures the position reached after the prompt
        for _ in range(max_tokens - 1):
            self._graph.replay()
            self.length += 1
            self._text.append(np.array([out[-1:]], dtype=np.int32))
            out.append(int(self.next_token[0].item()))
        self._check_dropped()
        return out

    def generate_batch(self, prompts, max_tokens: int, keep: Optional[int] = None, recent: int = 0) -> list:
        """Greedy continuation of every sequence: the prompts prefilled as blocks,
        then ``max_tokens`` - 1 replays of the captured batched step.  With ``keep``
        the cache is pruned to ``keep`` positions (``evict``) after the prompts and
        whenever it is full, so the text may outgrow it."""
        if keep is not None:
            self._check_evict(keep, recent)
            if not keep < self.max_seq:
                raise ValueError(f"keep must be below max_seq {self.max_seq}, got {keep}")
        else:
            self._check_room(len(prompts[0]), max_tokens)
        self.prefill(prompts)
        out = [self.next_token.cpu().tolist()]
        if keep is not None:
            self.evict(keep, recent)
        if self._graph is None:
            self.capture()
        for _ in range(max_tokens - 1):
            if keep is not None and self.held >= self.max_seq:
                self.evict(keep, recent)
            self._graph.replay()
            self.length += 1
            self._text.append(np.array(out[-1], dtype=np.int32)[:, None])
            out.append(self.next_token.cpu().tolist())
        self._check_dropped()
        return [[row[q] for row in out] for q in range(self.batch)]

    def generate_drafted(self, prompts, max_tokens: int, nodes: int = 16, draft=None) -> list:
        """Greedy continuation of every sequence, several tokens a pass (``kv_bits`` 16): the
        tokens that may follow each text are drafted as a tree of at most ``nodes`` nodes,
        its first the text's last token; one pass over the model gives the choice after each
        node, and the path that the choices confirm is kept (PagedKVCache.accept).  The
        choices are those of the model on the tokens before them, so drafts change how
        many passes a text takes and not what it says, but for choices within the
        difference of the matmul kernels (m = batch x nodes instead of m = batch).

        ``draft``: a function of a text (a list of token ids) that returns lists of tokens
        that may follow it, the likeliest first; drafts.look_up unless given.  ``passes``
        counts the passes of the last call."""
        from .drafts import grow, look_up
        from .paged import MOST_NODES
        if not self.paged:
            raise ValueError("drafted tokens need kv_bits 16")
        if self.comm is not None or self._penal is not None:
            raise ValueError("drafted tokens need the whole logits and the plain choice: no tensor parallelism, no penalties")
        if len(prompts) > 0 and not isinstance(prompts[0], (list, tuple, np.ndarray)):
            prompts = [prompts]
        if not 1 <= nodes <= MOST_NODES or self.batch * nodes > self.max_block_rows:
            raise ValueError(f"nodes must be in 1..{MOST_NODES} with at most {self.max_block_rows} rows in all, got {nodes}")
        if max_tokens < 1:
            raise ValueError(f"max_tokens must be positive, got {max_tokens}")
        draft = draft or look_up
        begin = self.length
        self._check_room(len(prompts[0]), max_tokens)
        self.prefill(prompts)
        known = np.concatenate(self._text, 1)
        texts = [known[q].tolist() for q in range(self.batch)]
        out = [[t] for t in self.next_token.tolist()]
        end = begin + len(prompts[0]) + max_tokens - 1  # positions held by every sequence at the end
        if self._drafts is None or self._drafts.rows_per_seq != nodes:
            self._drafts = self._draft_buffers(nodes)
        d = self._drafts
        self.passes = 0
        try:
            while any(len(o) < max_tokens for o in out):
                trees = []
                for text, o in zip(texts, out):
                    room = min(nodes, max_tokens - len(o))  # every node may be accepted; its position is within `end`
                    trees.append(grow(o[-1] if room > 0 else 0, draft(text + o) if room > 1 else [], room, self.cfg.vocab))
                accepted, taken = self._pass(d, trees)
                self.passes += 1
                for o, tokens, n in zip(out, accepted, taken):
                    o += tokens[:n]
            self._check_dropped()
        except BaseException:
            self.cache.lengths.fill_(self.length)  # as the prompts left it
            raise
        self.position.fill_(end)  # (as the lengths are: no tree had more nodes than tokens to come)
        self.length = end
        chosen = np.array(out, dtype=np.int32)
        self._text.append(chosen[:, :-1])
        self.next_token.copy_(torch.from_numpy(chosen[:, -1].copy()))
        self.token.copy_(self.next_token)
        return chosen.tolist()

    def _draft_buffers(self, nodes: int) -> "_Rows":
        dev, batch, rows = self.position.device, self.batch, self.batch * nodes
        d = _Rows()
        d.rows_per_seq, d.graph, d.warm = nodes, None, False
        words = (nodes + 31) // 32
        # tokens, parents, depths, visible words and counts of a pass, copied in one piece
        sizes = [rows, rows, rows, rows * words, batch]
        d.host = torch.zeros(sum(sizes), dtype=torch.int32, pin_memory=True)
        d.device = torch.zeros(sum(sizes), dtype=torch.int32, device=dev)
        d.fields, d.given = (x.split(sizes) for x in (d.host, d.device))
        tokens, parents, depths, visible, d.counts = d.given
        d.parents, d.depths = parents.view(batch, nodes), depths.view(batch, nodes)
        d.visible = visible.view(batch, nodes, words)
        d.tokens = tokens.view(batch, nodes)
        d.b = self._buffers(rows, tokens=tokens)
        f32 = dict(dtype=torch.float32, device=dev)
        d.normed, d.logits = torch.empty((rows, self.cfg.dim), **f32), torch.empty((rows, self.cfg.vocab), **f32)
        d.choices = torch.zeros((batch, nodes), dtype=torch.int32, device=dev)
        d.result = torch.zeros(rows + batch, dtype=torch.int32, device=dev)
        d.accepted, d.taken = d.result[:rows].view(batch, nodes), d.result[rows:]
        return d

    def _pass(self, d: "_Rows", trees):
        """One pass over drafted trees ((tokens, parents) of each sequence): accepted tokens and
        how many, as lists."""
        from .paged import draft_tree
        nodes, words = d.rows_per_seq, (d.rows_per_seq + 31) // 32
        tokens, parents, depths, visible, counts = (x.numpy() for x in d.fields)
        shape = (self.batch, nodes)
        tokens, parents, depths = tokens.reshape(shape), parents.reshape(shape), depths.reshape(shape)
        tokens[:], parents[:], depths[:], visible[:] = 0, -1, 0, 0
        visible = visible.reshape(*shape, words)
        for q, (t, p) in enumerate(trees):
            n = counts[q] = len(t)
            if n > 0:
                tokens[q, :n], parents[q, :n] = t, p
                depths[q, :n], seen = draft_tree(p)
                visible[q, :n, :seen.shape[1]] = seen
        d.device.copy_(d.host, non_blocking=True)
        if not d.warm:  # (a text of one pass is not worth a graph)
            self._launch_pass(d)
            d.warm = True
        else:
            if d.graph is None:
                torch.cuda.synchronize()
                d.graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(d.graph):
                    self._launch_pass(d)
            d.graph.replay()
        result = d.result.tolist()
        accepted = result[:self.batch * nodes]
        return [accepted[q * nodes:(q + 1) * nodes] for q in range(self.batch)], result[self.batch * nodes:]

    def _launch_pass(self, d: "_Rows") -> None:
        L_ = _lib.load()
        h, s, p, rows = self.ctx.handle, self._stream(), self._p, self.batch * d.rows_per_seq
        self._layers(d.b, rows, d.rows_per_seq, counts=d.counts, depths=d.depths, visible=d.visible)
        _lib.check(L_.kt_rmsnorm_qmatmul(h, self.head.handle, p(d.b.x), p(self.final_norm), self.cfg.eps, p(d.normed),
                                         p(d.logits), rows, 0, p(self.head_bias), s))
        _lib.check(L_.kt_argmax(h, p(d.logits), rows, self.cfg.vocab, p(d.choices), s))
        self.cache.accept(d.tokens, d.parents, d.choices, d.counts, d.accepted, d.taken)
        self.cache.advance(d.rows_per_seq, counts=d.taken)

    # -- the 8-bit cache and the choice of tokens
    def _check_evict(self, keep: int, recent: int) -> None:
        if self.cache is None or self.paged or self.cache.weights is None:
            raise ValueError("eviction needs kv_bits 8 and kv_weights")
        if keep < 1 or not 0 <= recent <= keep:
            raise ValueError(f"eviction needs 0 <= recent <= keep and 1 <= keep, got {recent} and {keep}")

    def evict(self, keep: int, recent: int) -> None:
        """Prunes the cache to ``keep`` positions: in every layer each key/value head keeps
        its ``recent`` last ones and those of the others that received most attention
        (KVCache8.evict).  Positions of later tokens go on from ``length``."""
        self._check_evict(keep, recent)
        if self.held > keep:
            self.cache.evict(keep, recent)
            self._evicted = self.length - keep

    def penalize(self, repetition=None, frequency=None, presence=None, bias_ids=None, bias_values=None, bias_counts=None,
                 allowed=None, history: Optional[int] = None) -> None:
        """From the next step on the logits go through a LogitsProcessor: penalties (a
        number, or one for each sequence) for the tokens of prompt and answer, those
        processed so far (prefill, step, generate) among them, sparse biases and a mask
        of allowed tokens (device tensors as LogitsProcessor takes them; the mask's
        contents may change between steps).  Of each text the last ``history`` tokens
        are remembered (max_seq unless given); a further call changes what is given and
        keeps them.  No arguments: plain argmax again."""
        self._graph = None  # a captured step has the old choice
        given = dict(repetition=repetition, frequency=frequency, presence=presence, bias_ids=bias_ids,
                     bias_values=bias_values, bias_counts=bias_counts, allowed=allowed)
        given = {k: v for k, v in given.items() if v is not None}
        if not given:
            self._penal = None
            return
        if self.comm is not None:
            raise ValueError("penalties need the whole logits: not under tensor parallelism")
        from .logits import LogitsProcessor
        dev = self.position.device
        for k in ("repetition", "frequency", "presence"):
            if k in given:
                x = torch.as_tensor(given[k], dtype=torch.float32, device=dev)
                if x.numel() not in (1, self.batch):
                    raise ValueError(f"{k} must be a number or one for each of {self.batch} sequences")
                given[k] = x.reshape(-1).expand(self.batch).contiguous()
        self._processor = LogitsProcessor(self.batch, self.cfg.vocab, self.ctx.device)
        room = history or self.max_seq
        if self._penal is not None:
            text, prompt = self._remembered()
        else:
            text = np.concatenate([np.empty((self.batch, 0), np.int32), *self._text], 1)
            text, prompt = torch.from_numpy(text), self._prompt_end
        before = text.shape[1]
        text = text[:, -room:]
        prompt = max(0, prompt - (before - text.shape[1]))
        i64 = dict(dtype=torch.int64, device=dev)
        self._history = torch.empty((self.batch, 2 * room), dtype=torch.int32, device=dev)
        self._history_lengths = torch.zeros(self.batch, dtype=torch.int32, device=dev)
        self._prompt_lengths = torch.zeros(self.batch, dtype=torch.int32, device=dev)
        self._place, self._places = torch.zeros(1, **i64), torch.zeros((2 * room, 4), **i64)
        self._lay_out(text, prompt)
        self._penal = given

    # The tokens that penalties see: the last `room` of each text, in 2 * room columns.  Token m of a
    # text is in column m until the columns 0..room-1 are full.  Then the columns are taken round and
    # round, the oldest token first, but that an answer's token must not lie ahead of the prompt's end
    # (_prompt_lengths): it takes column m + room where the prompt's token m is forgotten (-1: no token).
    # _places has, for every place m in 0..2*room-1, its column, the one forgotten, the columns in use
    # after it and the place after it, so that a captured step needs no host.
    def _lay_out(self, text, prompt: int) -> None:
        """The history is `text` [batch, at most room tokens], of which the first `prompt` are the prompt's."""
        text = text.to(self._history.device, copy=True)
        n, room = text.shape[1], self._history.shape[1] // 2
        self._history.fill_(-1)
        self._history[:, :n] = text
        self._history_lengths.fill_(n)
        self._prompt_lengths.fill_(prompt)
        self._place.fill_(n)
        m = torch.arange(2 * room, device=text.device)
        full, again = m >= room, m - room
        self._places.copy_(torch.stack([torch.where(full & (again >= prompt), again, m), torch.where(full, again, m),
                                        torch.where(full, room + prompt, m + 1), torch.where(m + 1 < 2 * room, m + 1, room)], 1))

    def _remembered(self):
        """The history in the texts' order, and how many of its tokens are the prompt's."""
        room, place = self._history.shape[1] // 2, int(self._place.item())
        first, again = self._history[:, :room], self._history[:, room:]
        prompt = int((first[0, :int(self._prompt_lengths[0].item())] >= 0).sum().item())
        text = torch.where(first >= 0, first, again)
        return (text[:, :place] if place < room else text.roll(room - place, 1)), prompt

    def _append_prompt(self, prompts) -> None:
        """Prompt tokens [batch, n] into the history; what is there so far counts as prompt."""
        room = self._history.shape[1] // 2
        text = torch.cat([self._remembered()[0], prompts.to(self._history.device)], 1)[:, -room:]
        self._lay_out(text, text.shape[1])

    # -- files (Transformer.saveQuantized / loadQuantized, Transformer.kt:402-471)
    def save_quantized(self, path) -> None:
        """Transformer.saveQuantized: the reference's file, byte for byte, written
        from HBM (q|k|v and gate|up are split back into their projections)."""
        from .parallel import COLUMNS, slice_weight
        if self.comm is not None:
            raise ValueError("save_quantized needs the whole model: save from an unsharded decoder")
        from .safetensors import SafeTensorsEntry, quantized_entries, save_entries
        cfg = self.cfg
        kv = cfg.kv_heads * cfg.head_dim
        meta = quantized_metadata(cfg)
        entries, keep = [], []

        def f32(name, t, n):
            entries.append(SafeTensorsEntry(name, "F32", [1, n], t.contiguous()))

        for l, L in enumerate(self.layers):
            f32(f"block.{l}.norm1.weight", L["norm1"], cfg.dim)
            f32(f"block.{l}.norm2.weight", L["norm2"], cfg.dim)
        f32("finalNorm.weight", self.final_norm, cfg.dim)
        q_cols = [(0, cfg.dim), (cfg.dim, cfg.dim + kv), (cfg.dim + kv, cfg.dim + 2 * kv)]
        g_cols = [(0, cfg.hidden), (cfg.hidden, 2 * cfg.hidden)]
        projections = []
        for l, L in enumerate(self.layers):
            parts = {}
            for key, (b, e) in zip(("wq", "wk", "wv"), q_cols):
                parts[key] = (slice_weight(L["wqkv"], COLUMNS, b, e), L["bqkv"][b:e])
            parts["wo"] = (L["wo"], L["bo"])
            for key, (b, e) in zip(("wg", "wu"), g_cols):
                parts[key] = (slice_weight(L["wgu"], COLUMNS, b, e), L["bgu"][b:e])
            parts["wd"] = (L["wd"], L["bd"])
            for suffix, key in PROJECTION_NAMES:
                projections.append((f"block.{l}.{suffix}",) + parts[key])
        projections.append(("lmHead", self.head, self.head_bias))
        for name, w, b in projections:
            f32(f"{name}.bias", b, w.columns)
        quantized = ([] if cfg.tied else [("embedding", self.embedding)]) + [(n, w) for n, w, _ in projections]
        for name, w in quantized:
            entries += quantized_entries(name, w)
            keep.append(w)  # the slices stay alive until the file is written
        save_entries(path, entries, meta)

    @staticmethod
    def load_quantized(path, max_seq: int, device: Optional[int] = None, **options) -> "DeviceDecoder":
        """Transformer.loadQuantized: a decoder whose weights go from the file
        straight into HBM; ``options`` are the constructor's (batch, kv_bits, ...)."""
        cfg, weights = load_quantized_weights(path, device)
        return DeviceDecoder(cfg, weights, max_seq, device, **options)


# (file name suffix, decoder weight key) in Transformer.namedProjections order (Transformer.kt:268-282)
PROJECTION_NAMES = [("attention.wQ", "wq"), ("attention.wK", "wk"), ("attention.wV", "wv"),
                    ("attention.wOut", "wo"), ("ffn.wGate", "wg"), ("ffn.wUp", "wu"), ("ffn.wDown", "wd")]


def quantized_metadata(cfg: DecoderConfig) -> dict:
    """The kotensor.* metadata of Transformer.saveQuantized (Transformer.kt:403-419)."""
    from .safetensors import java_float_string as js
    meta = {
        "kotensor.vocabularySize": str(cfg.vocab),
        "kotensor.dimension": str(cfg.dim),
        "kotensor.numLayers": str(cfg.layers),
        "kotensor.numHeads": str(cfg.heads),
        "kotensor.hiddenDimension": str(cfg.hidden),
        "kotensor.numKeyValueHeads": str(cfg.kv_heads),
        "kotensor.normEps": js(cfg.eps),
        "kotensor.ropeTheta": js(cfg.rope_theta),
    }
    if cfg.rope_scaling is not None:
        f, lo, hi, orig = cfg.rope_scaling
        meta["kotensor.ropeScaling"] = f"{js(f)},{js(lo)},{js(hi)},{int(orig)}"
    meta["kotensor.quantization.bits"] = str(cfg.bits)
    meta["kotensor.quantization.groupSize"] = str(cfg.group_size)
    if cfg.tied:
        meta["kotensor.tiedEmbedding"] = "true"
    return meta


class LoadedWeights:
    """Device weights read from a file, in DeviceDecoder's ``weights`` shape."""

    def __init__(self):
        self.embedding = None
        self.layers = []
        self.final_norm = None
        self.head = None
        self.head_bias = None


def load_quantized_weights(path, device: Optional[int] = None):
    """(config, weights) of a file written by Transformer.saveQuantized
    (Transformer.loadQuantized, Transformer.kt:433-471), weights in HBM."""
    from .quantized import Quantization
    from .safetensors import SafeTensorsFile
    with SafeTensorsFile(path) as f:
        meta = f.metadata

        def value(key):
            if key not in meta:
                raise ValueError(f"{path} has no {key} metadata; was it written by saveQuantized?")
            return meta[key]

        scaling = None
        if "kotensor.ropeScaling" in meta:
            p = meta["kotensor.ropeScaling"].split(",")
            scaling = (float(np.float32(p[0])), float(np.float32(p[1])), float(np.float32(p[2])), int(p[3]))
        q = Quantization(int(value("kotensor.quantization.bits")), int(value("kotensor.quantization.groupSize")))
        cfg = DecoderConfig(vocab=int(value("kotensor.vocabularySize")), dim=int(value("kotensor.dimension")),
                            layers=int(value("kotensor.numLayers")), heads=int(value("kotensor.numHeads")),
                            kv_heads=int(value("kotensor.numKeyValueHeads")),
                            hidden=int(value("kotensor.hiddenDimension")),
                            eps=float(np.float32(value("kotensor.normEps"))),
                            rope_theta=float(np.float32(value("kotensor.ropeTheta"))), rope_scaling=scaling,
                            bits=q.bits, group_size=q.group_size, tied=meta.get("kotensor.tiedEmbedding") == "true")
        kv = cfg.kv_heads * cfg.head_dim
        shapes = {"wq": (cfg.dim, cfg.dim), "wk": (cfg.dim, kv), "wv": (cfg.dim, kv), "wo": (cfg.dim, cfg.dim),
                  "wg": (cfg.dim, cfg.hidden), "wu": (cfg.dim, cfg.hidden), "wd": (cfg.hidden, cfg.dim)}

        def param(name):
            if name not in f:
                raise ValueError(f"{path} is missing {name}")
            return f.load(name, device).reshape(-1)

        w = LoadedWeights()
        for l in range(cfg.layers):
            L = {"norm1": param(f"block.{l}.norm1.weight"), "norm2": param(f"block.{l}.norm2.weight")}
            for suffix, key in PROJECTION_NAMES:
                name = f"block.{l}.{suffix}"
                L["b" + key[1]] = param(f"{name}.bias")
                L[key] = f.load_quantized(name, q, *shapes[key], device=device)
            w.layers.append(L)
        w.final_norm = param("finalNorm.weight")
        w.head_bias = param("lmHead.bias")
        w.head = f.load_quantized("lmHead", q, cfg.dim, cfg.vocab, device=device)
        if not cfg.tied:
            w.embedding = f.load_quantized("embedding", q, cfg.vocab, cfg.dim, device=device)
        torch.cuda.current_stream(w.head.device).synchronize()  # the file's staging buffers are released on close
    return cfg, w
