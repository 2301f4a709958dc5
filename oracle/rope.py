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
    out = torch.full(x.shape, float("nan"), dtype=torch.float64)
    weight = torch.zeros_like(x)
    for t, p in enumerate(positions):
        if not 0 <= p < table.shape[0]:
            continue
        y = x[t] / torch.sqrt((x[t] ** 2).mean(1, keepdim=True) + eps) * w
        out[t], weight[t] = y, y.abs()
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + half)
            c, s = table[p, i], table[p, half + i]
            out[t, :, a], out[t, :, b] = y[:, a] * c - y[:, b] * s, y[:, b] * c + y[:, a] * s
            weight[t, :, a] = (y[:, a] * c).abs() + (y[:, b] * s).abs()
            weight[t, :, b] = (y[:, b] * c).abs() + (y[:, a] * s).abs()
    return out, weight
