"""Logits before the choice of a token: penalties for repeated tokens, biases and
grammar masks, with the greedy choice in the same pass (kt_logits_process in
include/kt_cuda.h; the choice is argmaxOfLastToken,
Engine/kotensor/src/main/kotlin/Transformer.kt:255-266)."""
from __future__ import annotations

import ctypes
import struct

from . import _lib
from .quantized import Context, raw_stream

try:
    import torch
except ImportError:  # pragma: no cover
    torch = None


_PACK = struct.Struct("@PPqqiiPPPqiPPPiPPPqPqPP")
assert _PACK.size == ctypes.sizeof(_lib.KtLogitsArgs)


def _one(name: str, x, rows: int, dtype, device: int):
    """Pointer of a device array with one element for each row."""
    if x is None:
        return 0
    if x.dtype is not dtype or x.get_device() != device or x.dim() != 1 or x.numel() != rows or not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor of {rows} {str(dtype).replace('torch.', '')} on cuda:{device}, got "
                         f"{str(x.dtype).replace('torch.', '')} {list(x.shape)} on {x.device}")
    return x.data_ptr()


def _list(name: str, x, rows: int, dtype, device: int, least: int = 0):
    """Pointer, row stride and width of a device array [rows, at least `least`] with contiguous rows
    (the stride of a single row says nothing: its width)."""
    if x.dtype is not dtype or x.get_device() != device or x.dim() != 2 or x.shape[0] != rows or x.shape[1] < least or \
            (x.stride(1) != 1 and x.shape[1] > 1):
        raise ValueError(f"{name} must be a tensor of {str(dtype).replace('torch.', '')}, [{rows}, at least {least}] with "
                         f"contiguous rows, on cuda:{device}, got {str(x.dtype).replace('torch.', '')} {list(x.shape)} on {x.device}")
    width = x.shape[1]
    return x.data_ptr(), x.stride(0) if rows > 1 else width, width


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
        self._process = _lib.load().kt_logits_process
        self._scratch_ptr = self._scratch.data_ptr()
        self._args = _lib.KtLogitsArgs()  # filled anew by every call
        self._args_ref = ctypes.byref(self._args)

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
        themselves unless given) and returns the greedy choice of each row: ``next_token``
        (int32 [rows]), or a buffer of this object that its next call overwrites."""
        rows, vocab, device = self.rows, self.vocab, self.ctx.device
        f32, i32 = torch.float32, torch.int32
        token_p = lengths_p = prompt_p = repetition_p = frequency_p = presence_p = 0
        token_stride = token_width = bias_p = value_p = count_p = bias_stride = bias_width = allowed_p = allowed_stride = 0
        for name, x in (("logits", logits), ("out", out)):
            if x is not None and (x.dtype is not f32 or x.get_device() != device or x.shape != (rows, vocab) or
                                  (x.stride(1) != 1 and vocab > 1)):
                raise ValueError(f"{name} must be a float32 tensor of shape [{rows}, {vocab}] with contiguous rows on "
                                 f"cuda:{device}")
        if out is None:
            out = logits
        if tokens is not None:
            if lengths is None:
                raise ValueError("tokens need lengths")
            token_p, token_stride, token_width = _list("tokens", tokens, rows, i32, device)
            lengths_p = _one("lengths", lengths, rows, i32, device)
            prompt_p = _one("prompt_lengths", prompt_lengths, rows, i32, device)
            repetition_p = _one("repetition", repetition, rows, f32, device)
            frequency_p = _one("frequency", frequency, rows, f32, device)
            presence_p = _one("presence", presence, rows, f32, device)
        elif not (repetition is None and frequency is None and presence is None):
            raise ValueError("penalties need tokens")
        if (bias_ids is None) != (bias_values is None):
            raise ValueError("bias_ids and bias_values come together")
        if bias_ids is not None:
            bias_p, bias_stride, bias_width = _list("bias_ids", bias_ids, rows, i32, device)
            value_p, *same = _list("bias_values", bias_values, rows, f32, device)
            if same != [bias_stride, bias_width]:
                raise ValueError("bias_ids and bias_values must have the same shape and strides")
            count_p = _one("bias_counts", bias_counts, rows, i32, device)
        if allowed is not None:
            allowed_p, allowed_stride, _ = _list("allowed", allowed, rows, i32, device, (vocab + 31) // 32)
        if next_token is None:
            next_token = self.next_token
        x_stride, y_stride = (logits.stride(0), out.stride(0)) if rows > 1 else (vocab, vocab)
        # kt_logits_args, field by field (a ctypes structure takes twice as long to fill)
        _PACK.pack_into(self._args, 0, logits.data_ptr(), out.data_ptr(), x_stride, y_stride, rows, vocab,
                        token_p, lengths_p, prompt_p, token_stride, token_width, repetition_p, frequency_p, presence_p,
                        bias_width, bias_p, value_p, count_p, bias_stride, allowed_p, allowed_stride,
                        _one("next_token", next_token, rows, i32, device), self._scratch_ptr)
        _lib.check(self._process(self.ctx.handle, self._args_ref, raw_stream(self.ctx.device)))
        return next_token
