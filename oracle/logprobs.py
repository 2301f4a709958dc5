"""Oracle of log probabilities, entropy and top alternatives (test infrastructure only), in 64 bits, a row at a time.

No counterpart in the reference, which ends at attention and products.  Pinned in
tests/test_oracle_serving.py."""
from __future__ import annotations

import math

import torch


def token_logprobs(logits, tokens, top):
    """(logprobs, entropy, ids, top_logprobs, spread): tokens a list of lists; spread [T] = sum p (x - max)^2, what a
    bound on the entropy's roundings needs."""
    logits = logits.detach().cpu().double()
    T, V = logits.shape
    n = len(tokens[0]) if T else 0
    lp = torch.full((T, n), math.nan, dtype=torch.float64)
    entropy = torch.full((T,), math.nan, dtype=torch.float64)
    ids = torch.full((T, top), -1, dtype=torch.int32)
    best = torch.full((T, top), math.nan, dtype=torch.float64)
    spread = torch.zeros(T, dtype=torch.float64)
    for t, x in enumerate(logits):
        m = x.max()
        if x.isnan().any() or m.abs() == math.inf:
            continue
        y = x - m
        log_s = torch.exp(y).sum().log()
        log_p = y - log_s
        p = torch.exp(log_p)
        seen = p > 0
        entropy[t] = -(p[seen] * log_p[seen]).sum()
        spread[t] = (p[seen] * y[seen] ** 2).sum()
        for i, v in enumerate(tokens[t]):
            if 0 <= v < V:
                lp[t, i] = log_p[v]
        order = sorted(range(V), key=x.neg().tolist().__getitem__)[:top] if top else []  # stable: ties by the lowest id
        ids[t] = torch.tensor(order, dtype=torch.int32)
        best[t] = log_p[order] if order else best[t]
    return lp, entropy, ids, best, spread
