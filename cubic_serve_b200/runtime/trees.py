"""Trees of drafted tokens: their masks, and several continuations of one text as one tree.

Node 0 is the request's last token; node ``j > 0`` is a draft that follows ``parents[j] < j``.  What follows the same tokens is drafted once.
"""
from __future__ import annotations

import numpy as np


def tree_masks(parents, words: int | None = None) -> np.ndarray:
    """Ancestors and self of every node as 32-bit words (uint32 ``[n, words]``, bit ``j % 32`` of word ``j / 32`` = node j), the
    ``masks`` of ``ops.kernels.tree_attention``."""
    n = len(parents)
    words = max(1, -(-n // 32)) if words is None else words
    if n > 32 * words:
        raise ValueError(f"{n} nodes do not fit {words} words")
    out = np.zeros((n, words), dtype=np.uint32)
    for j, p in enumerate(parents):
        if j and not 0 <= p < j:
            raise ValueError("a node follows an earlier one")
        if j:
            out[j] = out[p]
        out[j, j >> 5] |= np.uint32(1 << (j & 31))
    return out


def tree_depths(parents) -> np.ndarray:
    """Distance of every node from node 0 (int32): its position is the request's next one plus this."""
    out = np.zeros(len(parents), dtype=np.int32)
    for j in range(1, len(parents)):
        out[j] = out[parents[j]] + 1
    return out


def merge_drafts(drafts, most: int) -> tuple[list[int], list[int]]:
    """Several continuations of a text (lists of tokens, the likeliest first) as one tree of up to ``most`` drafts: ``(tokens,
    parents)`` of the nodes behind node 0, whose own place (token 0, parent -1) is the first entry of both."""
    tokens, parents, child = [0], [-1], {}
    for d in drafts:
        at = 0
        for t in d:
            nxt = child.get((at, int(t)))
            if nxt is None:
                if len(tokens) > most:
                    break
                nxt = child[at, int(t)] = len(tokens)
                tokens.append(int(t))
                parents.append(at)
            at = nxt
    return tokens, parents
