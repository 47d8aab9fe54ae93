"""Tokens that may follow a text, and their tree, for DeviceDecoder.generate_drafted (on the
host; no reference counterpart)."""
from __future__ import annotations

import numpy as np


def look_up(text, most: int = 4, depth: int = 8, longest: int = 3) -> list:
    """What followed the text's last tokens earlier in it: up to ``most`` continuations of up
    to ``depth`` tokens, those after the longest match (of at most ``longest`` tokens) and
    the latest first."""
    text = np.asarray(text)
    found = []
    for n in range(min(longest, len(text) - 1), 0, -1):
        windows = np.lib.stride_tricks.sliding_window_view(text[:-1], n)
        for at in np.nonzero((windows == text[-n:]).all(1))[0][::-1]:
            after = text[at + n:at + n + depth].tolist()
            if after not in found:
                found.append(after)
            if len(found) == most:
                return found
    return found


def grow(last: int, chains, nodes: int, vocab: int):
    """(tokens, parents) of a tree of at most ``nodes`` nodes from ``last``, the text's last
    token, along every chain in turn; equal beginnings share their nodes, and a token
    outside 0..vocab-1 ends its chain.  Empty lists where ``nodes`` is 0."""
    if nodes < 1:
        return [], []
    tokens, parents, children = [int(last)], [-1], {}
    for chain in chains:
        at = 0
        for token in chain:
            token = int(token)
            if not 0 <= token < vocab:
                break
            child = children.get((at, token))
            if child is None:
                if len(tokens) == nodes:
                    break
                child = children[at, token] = len(tokens)
                tokens.append(token)
                parents.append(at)
            at = child
    return tokens, parents
