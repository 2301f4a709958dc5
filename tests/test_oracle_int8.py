"""The int8 oracle against brute force and closed forms."""
from __future__ import annotations

from fractions import Fraction

import torch

from oracle import int8


def test_codes_are_the_nearest_integers():
    x = (torch.randn((6, 40), generator=torch.Generator().manual_seed(1)) * 3).to(torch.bfloat16)
    q, s = int8.quantize_rows(x)
    for m in range(6):
        assert s[m] == x[m].float().abs().max() / 127
        for k in range(40):
            exact = Fraction(float(x[m, k])) / Fraction(float(s[m]))
            assert round(exact) == int(q[m, k])  # Fraction rounds half to even


def test_special_rows():
    x = torch.zeros((4, 16), dtype=torch.float16)
    x[1, 3], x[2, 0] = float("inf"), float("nan")
    x[3, :3] = torch.tensor([127.0, 0.5, 1.5])
    q, s = int8.quantize_rows(x)
    assert s[0] == 1 and s[1:3].isnan().all() and s[3] == 1
    assert not q[:3].any() and q[3, :3].tolist() == [127, 0, 2]


def test_product_is_exact():
    g = torch.Generator().manual_seed(2)
    a = torch.randint(-128, 128, (3, 64), generator=g, dtype=torch.int32)
    w = torch.randint(-128, 128, (5, 64), generator=g, dtype=torch.int32)
    c = int8.product(a.to(torch.int8), torch.ones(3), w.to(torch.int8), torch.full((5,), 0.5))
    assert torch.equal(c, (a @ w.t()).double() / 2)
