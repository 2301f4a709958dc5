"""Oracle of the paged 8-bit cache and the attention over it (test infrastructure
only): plain loops over sequences, pages and heads, in 64 bits.

No counterpart in the reference, whose caches are 16-bit.  Pinned in
tests/test_oracle_kv8.py."""
from __future__ import annotations

import math

import torch

LEAST = 2.0 ** -32


def scale_for(most: float) -> float:
    """The smallest power of two s, at least 2^-32, with most <= 448 s."""
    s = LEAST
    while most > 448 * s:
        s *= 2
    return s


def nearest_e4m3(x: torch.Tensor) -> torch.Tensor:
    """The e4m3 value nearest to each x (float64, |x| <= 448), ties to the even code."""
    mag = x.abs().clamp_min(2.0 ** -6)
    step = torch.exp2(torch.floor(torch.log2(mag)) - 3)
    return torch.round(x / step) * step


class Cache:
    """Values of codes in float64 (NaN where a code is NaN), and their scales."""

    def __init__(self, k, v, k_scale, v_scale):
        """From the tensors of a KV8Cache (copied)."""
        self.k = k.detach().cpu().float().double()
        self.v = v.detach().cpu().float().double().transpose(2, 3).contiguous()  # [pages, n_kv, page, d] here
        self.ks, self.vs = k_scale.detach().cpu().double(), v_scale.detach().cpu().double()
        self.pages, self.n_kv, self.page, self.d = self.k.shape

    def append(self, k, v, table, lens, cu):
        """New rows into the cache; table [B][..], lens [B], cu [B + 1] plain lists."""
        for b in range(len(lens)):
            n = cu[b + 1] - cu[b]
            start = lens[b] - n
            rows = {start + i: cu[b] + i for i in range(n) if start + i >= 0}
            for j in sorted({t // self.page for t in rows}):
                p = table[b][j]
                if not 0 <= p < self.pages:
                    continue
                new = [t for t in rows if t // self.page == j]
                lo = min(new) - j * self.page
                for x, code, scale in ((k, self.k, self.ks), (v, self.v, self.vs)):
                    x = x.detach().cpu().double()
                    for h in range(self.n_kv):
                        y = x[[rows[t] for t in new], h]
                        fin = torch.isfinite(y)
                        s = scale_for(float(y[fin].abs().max()) if fin.any() else 0.0)
                        if lo > 0:
                            old = float(scale[p, h])
                            s = max(s, old)
                            kept = code[p, h, :lo]
                            code[p, h, :lo] = torch.where(kept.isnan(), kept, nearest_e4m3(kept * (old / s)))
                        z = torch.where(fin, nearest_e4m3(torch.where(fin, y, torch.zeros_like(y)) / s),
                                        torch.full_like(y, math.nan))
                        for t, row in zip(new, z):
                            code[p, h, t - j * self.page] = row
                        scale[p, h] = s

    def tokens(self, b, h, n, table):
        """(K, V [n, d], present [n]): tokens of an unknown page are absent."""
        k, v = torch.zeros((n, self.d), dtype=torch.float64), torch.zeros((n, self.d), dtype=torch.float64)
        present = torch.zeros(n, dtype=torch.bool)
        for t in range(n):
            j = t // self.page
            p = table[b][j] if j < len(table[b]) else -1
            if 0 <= p < self.pages:
                k[t] = self.k[p, h, t % self.page] * self.ks[p, h]
                v[t] = self.v[p, h, t % self.page] * self.vs[p, h]
                present[t] = True
        return k, v, present

    def attend(self, q, table, lens, cu, causal=True, scale=None, seen=None):
        """(out, weight, score) [T, n_q, d] / [T, n_q]: the attention, the sum of
        p |v| for each output, and the largest sum of |scale q k| of a row (what a bound on the
        device's roundings needs).  Rows of no sequence are NaN.  seen(b, i): which of the tokens
        0 .. lens[b] - 1 the i-th row of sequence b sees, instead of the causal mask."""
        q = q.detach().cpu().double()
        T, n_q, d = q.shape
        scale = 1 / math.sqrt(d) if scale is None else scale
        out = torch.full((T, n_q, d), math.nan, dtype=torch.float64)
        weight, score = torch.zeros((T, n_q, d), dtype=torch.float64), torch.zeros((T, n_q), dtype=torch.float64)
        for b in range(len(lens)):
            n = cu[b + 1] - cu[b]
            if not n:
                continue
            for h in range(self.n_kv):
                k, v, present = self.tokens(b, h, lens[b], table)
                for i in range(n):
                    see = present.clone()
                    if seen is not None:
                        see &= seen(b, i)
                    elif causal:
                        see[max(lens[b] - n + i + 1, 0):] = False
                    r = cu[b] + i
                    for j in range(h * (n_q // self.n_kv), (h + 1) * (n_q // self.n_kv)):
                        if not see.any():
                            out[r, j] = 0
                            continue
                        p = torch.softmax((k[see] @ q[r, j]) * scale, 0)
                        out[r, j] = p @ v[see]
                        weight[r, j] = p @ v[see].abs()
                        score[r, j] = ((k[see].abs() @ q[r, j].abs()) * abs(scale)).max()
        return out, weight, score
