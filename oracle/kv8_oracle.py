"""Restatement in numpy of the 8-bit key/value cache and the logit processing: the
quantisation bit for bit (float32 steps), everything else in 64 bits."""
import numpy as np

F = np.float32


def quantise(x):
    """(codes, scale) of one block of float32 values."""
    bits = np.abs(x).astype(F)
    if not np.isfinite(bits).all():
        return np.zeros(x.shape, np.int8), F(np.nan)
    a = bits.max() if bits.size else F(0)
    if a < F(2.0 ** -100):
        return np.zeros(x.shape, np.int8), F(0)
    inverse = F(F(1.0) / a) * F(127.0)
    codes = np.clip(np.rint(x * inverse), -127, 127).astype(np.int8)
    return codes, a * (F(1.0) / F(127.0))


class Cache:
    """One layer, every buffer as the device keeps it."""

    def __init__(self, batch, kv_heads, head_dim, capacity, block, lengths):
        self.b, self.h, self.d, self.cap, self.block = batch, kv_heads, head_dim, capacity, block
        self.codes = {n: np.zeros((batch, kv_heads, capacity, head_dim), np.int8) for n in "kv"}
        self.scales = {n: np.zeros((batch, kv_heads, capacity // block), F) for n in "kv"}
        self.tail = {n: np.zeros((batch, kv_heads, block, head_dim), F) for n in "kv"}
        self.weights = np.zeros((batch, kv_heads, capacity), F)
        self.lengths = np.array(lengths, np.int32)

    def store(self, k, v, rows, counts=None):
        """k, v [batch * rows, kv_heads * head_dim]; True if tokens were dropped."""
        dropped = False
        for b in range(self.b):
            n = rows if counts is None else max(0, min(rows, int(counts[b])))
            held = int(self.lengths[b])
            if held + n > self.cap:
                n, dropped = self.cap - held, True
            if n == 0:
                continue
            inside, first = held % self.block, held // self.block
            for name, x in (("k", k), ("v", v)):
                new = x.reshape(self.b, rows, self.h, self.d)[b, :n].transpose(1, 0, 2)
                for h in range(self.h):
                    y = np.concatenate([self.tail[name][b, h, :inside], new[h]])
                    for i in range(0, len(y), self.block):
                        part = y[i:i + self.block]
                        codes, scale = quantise(part)
                        at = first * self.block + i
                        self.codes[name][b, h, at:at + len(part)] = codes
                        self.scales[name][b, h, at // self.block] = scale
                    left = (held + n) % self.block
                    if left:
                        self.tail[name][b, h, :left] = y[-left:]
            self.weights[b, :, held:held + n] = 0
        return dropped

    def values(self, name, b, h, n):
        """The values of slots 0..n-1, in 64 bits."""
        s = np.repeat(self.scales[name][b, h].astype(np.float64), self.block)[:n]
        return self.codes[name][b, h, :n].astype(np.float64) * s[:, None]

    def attend(self, q, heads, rows, scale, counts=None):
        """(context, weight received by each slot, largest sum of |scale q k| terms, largest |v|)."""
        group = heads // self.h
        q = q.astype(np.float64).reshape(self.b, rows, heads, self.d)
        out = np.zeros((self.b, rows, heads, self.d))
        weights = np.zeros((self.b, self.h, self.cap))
        size = top = 0.0
        for b in range(self.b):
            m = rows if counts is None else max(0, min(rows, int(counts[b])))
            for h in range(self.h):
                n = min(int(self.lengths[b]) + m, self.cap)
                k, v = self.values("k", b, h, n), self.values("v", b, h, n)
                top = max(top, np.abs(v).max(initial=0))
                for t in range(m):
                    seen = min(int(self.lengths[b]) + t + 1, self.cap)
                    for g in range(group):
                        x = q[b, t, h * group + g]
                        size = max(size, scale * (np.abs(k[:seen]) @ np.abs(x)).max(initial=0))
                        s = scale * (k[:seen] @ x)
                        p = np.exp(s - s.max())
                        p /= p.sum()
                        out[b, t, h * group + g] = p @ v[:seen]
                        weights[b, h, :seen] += p
        return out.reshape(self.b * rows, heads * self.d), weights, size, top

    def kept(self, b, h, keep, recent):
        """Slots that eviction keeps, in order."""
        n = int(self.lengths[b])
        w = self.weights[b, h, :n - recent]
        w = np.where(np.isnan(w), np.inf, w.astype(np.float64))
        nan_first = np.where(np.isnan(self.weights[b, h, :n - recent]), 0, 1)
        order = np.lexsort((np.arange(len(w)), -w, nan_first))[:keep - recent]
        return np.concatenate([np.sort(order), np.arange(n - recent, n)]).astype(np.int64)

    def evict(self, keep, recent):
        for b in range(self.b):
            if self.lengths[b] <= keep:
                continue
            for h in range(self.h):
                at = self.kept(b, h, keep, recent)
                for name in "kv":
                    x = self.codes[name][b, h, at].astype(F) * self.scales[name][b, h, at // self.block][:, None]
                    for i in range(0, keep, self.block):
                        part = x[i:i + self.block]
                        codes, scale = quantise(part)
                        self.codes[name][b, h, i:i + len(part)] = codes
                        self.scales[name][b, h, i // self.block] = scale
                    left = keep % self.block
                    if left:
                        self.tail[name][b, h, :left] = x[-left:]
                self.weights[b, h, :keep] = self.weights[b, h, at].copy()


def process_logits(logits, tokens=None, lengths=None, prompt_lengths=None, repetition=None, frequency=None, presence=None,
                   bias_ids=None, bias_values=None, bias_counts=None, allowed=None):
    """(logits, next token) of [rows, vocab], in 64 bits."""
    y = logits.astype(np.float64)
    rows, n = y.shape
    best = np.zeros(rows, np.int32)
    for r in range(rows):
        if tokens is not None:
            line = tokens[r, :max(0, min(int(lengths[r]), tokens.shape[1]))]
            prompt = 0 if prompt_lengths is None else max(0, int(prompt_lengths[r]))
            for i in {int(t) for t in line if 0 <= t < n}:
                if repetition is not None:
                    y[r, i] = y[r, i] / float(repetition[r]) if y[r, i] > 0 else y[r, i] * float(repetition[r])
            answer = [int(t) for t in line[prompt:] if 0 <= t < n]
            for i in set(answer):
                y[r, i] -= (float(frequency[r]) if frequency is not None else 0.0) * answer.count(i)
                y[r, i] -= float(presence[r]) if presence is not None else 0.0
        if bias_ids is not None:
            e = bias_ids.shape[1] if bias_counts is None else max(0, min(int(bias_counts[r]), bias_ids.shape[1]))
            for i, x in zip(bias_ids[r, :e], bias_values[r, :e]):
                if 0 <= i < n:
                    y[r, i] += float(x)
        if allowed is not None:
            bit = (allowed[r].view(np.uint32)[np.arange(n) // 32] >> (np.arange(n) % 32).astype(np.uint32)) & 1
            y[r, bit == 0] = -np.inf
        seen = np.where(np.isnan(y[r]), -np.inf, y[r])
        best[r] = int(seen.argmax()) if seen.max() > -1e9 else 0
    return y, best
