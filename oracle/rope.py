"""Oracle of the norm and rotation of heads (test infrastructure only), in 64 bits, a pair at a time.

No counterpart in the reference, whose attention takes rotated queries and keys.  Pinned in
tests/test_oracle_serving.py."""
from __future__ import annotations

import torch


def norm_rope(x, w, table, positions, eps, neighbours=False):
    """(out, weight) [T, heads, d]: the normed and turned heads, and |a cos| + |b sin| of each value (what a bound
    on the device's roundings needs).  Tokens whose position is no row of the table are NaN."""
    x, w, table = x.detach().cpu().double(), w.detach().cpu().double(), table.detach().cpu().double()
    half = table.shape[1] // 2
    there = torch.tensor([0 <= p < table.shape[0] for p in positions])
    at = table[torch.tensor([p if 0 <= p < table.shape[0] else 0 for p in positions])]
    y = x / torch.sqrt((x ** 2).mean(2, keepdim=True) + eps) * w
    out, weight = y.clone(), y.abs()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + half)
        c, s = at[:, None, i], at[:, None, half + i]
        out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
        weight[..., a] = (y[..., a] * c).abs() + (y[..., b] * s).abs()
        weight[..., b] = (y[..., b] * c).abs() + (y[..., a] * s).abs()
    out[~there] = float("nan")
    return out, weight
