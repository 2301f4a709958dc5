"""Int8 oracle (test infrastructure only): quantisation with a scale per row, and
the product with a scale per token and channel, in 64 bits.

No counterpart in the reference.  Pinned in tests/test_oracle_int8.py."""
from __future__ import annotations

import torch


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [M,K] (16-bit) -> (q [M,K] int8, scale [M] fp32): scale = max |row| / 127 in
    fp32 (1 for a zero row, NaN for one with an infinity or a NaN), q = the quotient's
    nearest integer, ties to even."""
    x = x.detach().cpu()
    finite = torch.isfinite(x).all(1)
    xf = torch.where(finite[:, None], x, torch.zeros_like(x)).float()
    amax = xf.abs().amax(1)
    scale = torch.where(amax > 0, amax / 127, torch.ones_like(amax))
    q = torch.round(xf.double() / scale.double()[:, None]).to(torch.int8)
    return q, torch.where(finite, scale, torch.full_like(scale, float("nan")))


def product(a: torch.Tensor, sa: torch.Tensor, w: torch.Tensor, sw: torch.Tensor) -> torch.Tensor:
    """[M,N] float64: (a . w^T) sa sw (products of int8 sum exactly in float64)."""
    c = a.detach().cpu().double() @ w.detach().cpu().double().t()
    return c * sa.detach().cpu().double()[:, None] * sw.detach().cpu().double()
