"""Pins of the oracles of the norm and rotation of heads and of log probabilities."""
from __future__ import annotations

import math

import torch

from oracle import logprobs, rope


def test_norm_rope_by_hand():
    """A quarter turn moves the first half into the second; the norm makes the mean square one."""
    x = torch.zeros((1, 1, 16))
    x[0, 0, :8] = 3.0
    table = torch.cat([torch.zeros((2, 8)), torch.ones((2, 8))], 1)
    out, weight = rope.norm_rope(x, torch.full((16,), 0.5), table, [1], 0.0)
    assert torch.allclose(out[0, 0, 8:], torch.full((8,), 0.5 * math.sqrt(2), dtype=torch.float64))
    assert torch.equal(out[0, 0, :8], torch.zeros(8, dtype=torch.float64)) and torch.equal(weight, out.abs())
    x = torch.zeros((1, 1, 16))
    x[0, 0, ::2] = 1.0
    out, _ = rope.norm_rope(x, torch.ones(16), table, [0], 0.0, neighbours=True)
    assert torch.allclose(out[0, 0, 1::2], torch.full((8,), math.sqrt(2), dtype=torch.float64))
    assert bool(rope.norm_rope(x, torch.ones(16), table, [2], 0.0)[0].isnan().all())


def test_norm_rope_keeps_products_of_equal_distance():
    """q . k depends on the difference of the positions alone, and channels behind the rotation on neither."""
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn((1, 1, 48), generator=g), torch.randn((1, 1, 48), generator=g)
    angle = torch.arange(64.0, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(0, 32, 2) / 32)
    table = torch.cat([angle.cos(), angle.sin()], 1)
    for neighbours in (False, True):
        dots = []
        for a, b in ((9, 4), (30, 25), (63, 58)):
            x, _ = rope.norm_rope(q, torch.ones(48), table, [a], 1e-6, neighbours)
            y, _ = rope.norm_rope(k, torch.ones(48), table, [b], 1e-6, neighbours)
            dots.append(float((x * y).sum()))
            plain, _ = rope.norm_rope(q, torch.ones(48), table, [0], 1e-6, neighbours)
            assert torch.equal(x[..., 32:], plain[..., 32:])
        assert max(dots) - min(dots) < 1e-12


def test_logprobs_by_hand():
    x = torch.tensor([[0.0, math.log(3), -math.inf, math.log(4)], [1.0, 1.0, 1.0, 1.0], [0.0, math.nan, 0.0, 0.0],
                      [math.inf, 0.0, 0.0, 0.0], [-math.inf] * 4], dtype=torch.float64)
    lp, h, ids, best, _ = logprobs.token_logprobs(x, [[3, -1], [0, 4], [0, 1], [0, 1], [0, 1]], 4)
    assert torch.allclose(lp[0, 0], torch.tensor(math.log(0.5), dtype=torch.float64)) and lp[0, 1].isnan()
    assert torch.allclose(h[:2], torch.tensor([-(0.125 * math.log(0.125) + 0.375 * math.log(0.375) + 0.5 * math.log(0.5)),
                                               math.log(4)], dtype=torch.float64))
    assert ids.tolist() == [[3, 1, 0, 2], [0, 1, 2, 3], [-1] * 4, [-1] * 4, [-1] * 4]
    assert best[0, 3] == -math.inf and bool(h[2:].isnan().all()) and bool(best[2:].isnan().all())


def test_logprobs_against_torch():
    x = torch.randn((3, 1000), generator=torch.Generator().manual_seed(2), dtype=torch.float64) * 5
    lp, h, ids, best, _ = logprobs.token_logprobs(x, [[5], [0], [999]], 7)
    want = torch.log_softmax(x, 1)
    assert torch.allclose(lp[:, 0], want[range(3), [5, 0, 999]], rtol=1e-13)
    assert torch.allclose(h, torch.distributions.Categorical(logits=x).entropy(), rtol=1e-12)
    assert torch.equal(ids.long(), want.topk(7).indices) and torch.allclose(best, want.topk(7).values, rtol=1e-13)
