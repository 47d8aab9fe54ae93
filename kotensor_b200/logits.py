"""Logits before the choice of a token: penalties for repeated tokens, biases and
grammar masks, with the greedy choice in the same pass (kt_logits_process in
include/kt_cuda.h; the choice is argmaxOfLastToken,
Engine/kotensor/src/main/kotlin/Transformer.kt:255-266)."""
from __future__ import annotations

import ctypes

from . import _lib
from .quantized import Context, _stream_of

try:
    import torch
except ImportError:  # pragma: no cover
    torch = None


def _per_row(name: str, x, rows: int, dtype, width=None):
    """Pointer of a per-request device array: [rows], or [rows, >= width] with contiguous rows."""
    if x is None:
        return None
    if not x.is_cuda or x.dtype != dtype:
        raise ValueError(f"{name} must be a CUDA tensor of {str(dtype).replace('torch.', '')}")
    if width is None:
        if x.shape != (rows,) or not x.is_contiguous():
            raise ValueError(f"{name} must be a contiguous tensor of {rows} elements, got {list(x.shape)}")
    elif x.dim() != 2 or x.shape[0] != rows or x.shape[1] < width or (x.shape[1] > 1 and x.stride(1) != 1):
        raise ValueError(f"{name} must be [{rows}, at least {width}] with contiguous rows, got {list(x.shape)}")
    return x.data_ptr()


class LogitsProcessor:
    """Processes [rows, vocab] float32 logits; one object per stream (it holds the
    buffer the greedy choice is merged in)."""

    def __init__(self, rows: int, vocab: int, device=None):
        if rows < 1 or vocab < 1:
            raise ValueError(f"rows and vocab must be positive, got {rows} and {vocab}")
        self.rows, self.vocab = rows, vocab
        self.ctx = Context.get(device)
        dev = torch.device("cuda", self.ctx.device)
        self._scratch = torch.zeros(16 * rows, dtype=torch.uint8, device=dev)
        self.next_token = torch.zeros(rows, dtype=torch.int32, device=dev)
        self._lib = _lib.load()

    def __call__(self, logits, out=None, tokens=None, lengths=None, prompt_lengths=None, repetition=None,
                 frequency=None, presence=None, bias_ids=None, bias_values=None, bias_counts=None, allowed=None,
                 next_token=None):
        """For token id i of a row, in this order:
          repetition: x / repetition if x > 0, else x * repetition, for i among the row's tokens;
          frequency, presence: x - frequency * n - presence for i that occurs n > 0
            times from index prompt_lengths[row] on;
          biases: x + bias_values of every entry of bias_ids that is i;
          allowed: -inf where bit i % 32 of word i / 32 is 0.
        ``tokens`` int32 [rows, n] of which the first lengths[row] count; the penalties
        float32 [rows]; ``bias_ids`` int32 / ``bias_values`` float32 [rows, e] of which the
        first bias_counts[row] count; ``allowed`` int32 words.  Writes ``out`` (the logits
        themselves unless given) and returns the greedy choice of each row (int32)."""
        rows, vocab = self.rows, self.vocab
        if not logits.is_cuda or logits.dtype != torch.float32 or tuple(logits.shape) != (rows, vocab) or \
                (vocab > 1 and logits.stride(1) != 1):
            raise ValueError(f"logits must be a float32 CUDA tensor of shape [{rows}, {vocab}] with contiguous rows")
        if out is None:
            out = logits
        elif not out.is_cuda or out.dtype != torch.float32 or tuple(out.shape) != (rows, vocab) or \
                (vocab > 1 and out.stride(1) != 1):
            raise ValueError(f"out must be a float32 CUDA tensor of shape [{rows}, {vocab}] with contiguous rows")
        if tokens is not None and lengths is None:
            raise ValueError("tokens need lengths")
        if tokens is None and not (repetition is None and frequency is None and presence is None):
            raise ValueError("penalties need tokens")
        if (bias_ids is None) != (bias_values is None):
            raise ValueError("bias_ids and bias_values come together")
        if bias_ids is not None and bias_ids.shape != bias_values.shape:
            raise ValueError("bias_ids and bias_values must have the same shape")
        if next_token is None:
            next_token = self.next_token
        i32, f32 = torch.int32, torch.float32
        if bias_ids is not None and bias_ids.stride() != bias_values.stride():
            raise ValueError("bias_ids and bias_values must have the same strides")
        a = _lib.KtLogitsArgs(
            logits.data_ptr(), out.data_ptr(), logits.stride(0), out.stride(0), rows, vocab,
            _per_row("tokens", tokens, rows, i32, 0), _per_row("lengths", lengths, rows, i32),
            _per_row("prompt_lengths", prompt_lengths, rows, i32), 0 if tokens is None else tokens.stride(0),
            0 if tokens is None else tokens.shape[1],
            _per_row("repetition", repetition, rows, f32), _per_row("frequency", frequency, rows, f32),
            _per_row("presence", presence, rows, f32), 0 if bias_ids is None else bias_ids.shape[1],
            _per_row("bias_ids", bias_ids, rows, i32, 0),
            _per_row("bias_values", bias_values, rows, f32, 0), _per_row("bias_counts", bias_counts, rows, i32),
            0 if bias_ids is None else bias_ids.stride(0), _per_row("allowed", allowed, rows, i32, (vocab + 31) // 32),
            0 if allowed is None else allowed.stride(0), _per_row("next_token", next_token, rows, i32),
            self._scratch.data_ptr())
        _lib.check(self._lib.kt_logits_process(self.ctx.handle, ctypes.byref(a), _stream_of(logits)))
        return next_token
