"""Masks and depths of drafted trees, on the host."""
from __future__ import annotations

import random

import pytest
import torch

from conftest import import_submodule

drafts = import_submodule("drafts")


def test_masks_and_depths():
    parents = [-1, 0, 0, 2, -1, 4]
    m = drafts.masks(parents)
    assert m.dtype == torch.int64 and m.tolist() == [[1], [0b11], [0b101], [0b1101], [0b10000], [0b110000]]
    assert drafts.depths(parents).tolist() == [0, 1, 1, 2, 0, 1]
    assert drafts.masks([], 2).shape == (0, 2) and drafts.depths([]).shape == (0,)
    assert drafts.masks([-1], 3).tolist() == [[1, 0, 0]]


def test_many_words():
    rng = random.Random(1)
    n = 200
    parents = [rng.randint(max(-1, i - 5), i - 1) for i in range(n)]
    m = drafts.masks(parents)
    assert m.shape == (n, 4)
    for i in range(n):
        seen = {i}
        while parents[min(seen)] >= 0:
            seen.add(parents[min(seen)])
        assert {j for j in range(256) if m[i, j // 64].item() >> j % 64 & 1} == seen
        assert drafts.depths(parents)[i] == len(seen) - 1


def test_refusals():
    for parents in ([0], [-1, 1], [-2], [-1, 0.5]):
        with pytest.raises((ValueError, TypeError)):
            drafts.masks(parents)
        with pytest.raises((ValueError, TypeError)):
            drafts.depths(parents)
    with pytest.raises(ValueError):
        drafts.masks([-1] * 65, 1)
    with pytest.raises(ValueError):
        drafts.masks([-1] * 1025)
    with pytest.raises(ValueError):
        drafts.masks([-1], 17)
