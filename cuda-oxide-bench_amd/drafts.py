"""Drafted tokens that form a tree: what ops.gqa_kv8_tree and ops.qk_norm_rope take of it, on the host.

A tree is the list of its tokens' parents, each an earlier token's number or -1: a token that follows the
sequence itself.  A verified step takes the tokens of one sequence in that order.
"""
from __future__ import annotations

from operator import index

import torch


def _checked(parents) -> list[int]:
    parents = [index(p) for p in parents]
    for i, p in enumerate(parents):
        if not -1 <= p < i:
            raise ValueError(f"token {i}'s parent ({p}) must be an earlier token or -1")
    return parents


def masks(parents, words: int | None = None) -> torch.Tensor:
    """[tokens, words] int64 on the host: each token's ancestors and itself, bit j % 64 of word j // 64 for token j.
    words: how many (the most of a call's trees, up to 16), as few as hold the tokens without it."""
    parents = _checked(parents)
    need = max(1, -(-len(parents) // 64))
    words = need if words is None else index(words)
    if not need <= words <= 16:
        raise ValueError(f"{len(parents)} tokens need {need} words, up to 16 (got {words})")
    rows: list[int] = []
    for i, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else 0) | 1 << i)
    signed = [[(r >> 64 * w & (1 << 64) - 1) - ((r >> 64 * w + 63 & 1) << 64) for w in range(words)] for r in rows]
    return torch.tensor(signed, dtype=torch.int64).reshape(len(rows), words)


def depths(parents) -> torch.Tensor:
    """[tokens] int32 on the host: how many ancestors each token has.  Its position is the sequence's length before
    the drafted tokens and that."""
    out: list[int] = []
    for p in _checked(parents):
        out.append(out[p] + 1 if p >= 0 else 0)
    return torch.tensor(out, dtype=torch.int32)
