"""The paged 16-bit key/value cache in plain torch on the CPU, in 64 bits: rotation and
store, attention with its masks, and the accepted path of a drafted tree.  What
tests/test_paged_gpu.py compares with; the definitions are those of include/kt_cuda.h."""
import math

import torch


def slots(table, b, n, page, pages):
    """[(page, slot in it)] of the first n slots of sequence b; None where there is no page."""
    found = []
    for s in range(n):
        p = int(table[b, s // page]) if s // page < table.shape[1] else -1
        found.append((p, s % page) if 0 <= p < pages else None)
    return found


def tokens_of(counts, lengths, b, rows, capacity):
    """(tokens held, rows of the call that are tokens)."""
    held = min(max(int(lengths[b]), 0), capacity)
    n = rows if counts is None else min(max(int(counts[b]), 0), rows)
    return held, min(n, capacity - held)


def rotate(x, positions, inv_freq):
    """x [n, heads, d] in 64 bits, pairs (i, i + d / 2) turned by position * inv_freq."""
    angle = positions.double()[:, None, None] * inv_freq.double()
    cos, sin = torch.cos(angle), torch.sin(angle)
    low, high = x.double().chunk(2, -1)
    return torch.cat([low * cos - high * sin, low * sin + high * cos], -1)


def attend(keys, values, table, lengths, q, heads, rows, counts=None, visible=None, scale=None):
    """(out, magnitude) float64 [batch * rows, heads, d] of one layer's keys and values
    [pages, kv_heads, page, d]: the attention, and the same with |values|, by which
    roundings are counted.  Slots without a page are seen by no row."""
    pages, kv, page, d = keys.shape
    batch, capacity = table.shape[0], table.shape[1] * page
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    group = heads // kv
    out = torch.zeros(batch, rows, heads, d, dtype=torch.float64)
    size = torch.zeros_like(out)
    spread = torch.zeros(batch, rows, heads, 1, dtype=torch.float64)
    q = q.reshape(batch, rows, heads, d).double()
    for b in range(batch):
        held, n = tokens_of(counts, lengths, b, rows, capacity)
        where = slots(table, b, held + n, page, pages)
        for t in range(n):
            seen = []
            for s, place in enumerate(where):
                u = s - held
                sees = u < 0 or (u <= t if visible is None else bool(int(visible[b, t, u // 32]) >> (u % 32) & 1))
                if sees and place is not None:
                    seen.append(place)
            if not seen:
                continue
            p, i = torch.tensor(seen).T
            for h in range(kv):
                k, v = keys[p, h, i].double(), values[p, h, i].double()
                lines = slice(h * group, (h + 1) * group)
                w = torch.softmax(q[b, t, lines] @ k.T * scale, -1)
                out[b, t, lines] = w @ v
                size[b, t, lines] = w @ v.abs()
                spread[b, t, lines] = (q[b, t, lines].abs() @ k.abs().T).amax(-1, keepdim=True) * abs(scale)
    flat = lambda x: x.reshape(batch * rows, heads, -1)  # noqa: E731
    return flat(out), flat(size), flat(spread)


def path(tokens, parents, choices, n):
    """Nodes of the accepted path of one tree of n nodes."""
    if n == 0:
        return []
    nodes = [0]
    while True:
        at = nodes[-1]
        below = [u for u in range(at + 1, n) if int(parents[u]) == at and int(tokens[u]) == int(choices[at])]
        if not below:
            return nodes
        nodes.append(below[0])
