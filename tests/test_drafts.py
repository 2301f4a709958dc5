"""Masks and depths of drafted trees, on the host."""
from __future__ import annotations

import random

import pytest
import torch

from conftest import import_submodule
from oracle import kv8 as oracle

drafts = import_submodule("drafts")
kv_pages = import_submodule("kv_pages")


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


@pytest.mark.parametrize("before", [1, 20, 30, 32, 48])
@pytest.mark.parametrize("forked", [False, True])
def test_rejected_drafts_and_the_page_they_shared(before, forked):
    """Loud drafts that are rejected: on a fork they leave nothing behind, and the cache holds what it would hold had
    the accepted tokens alone been appended; without one the page that they began on keeps their scale."""
    page, news, kept = 16, 20, [0, 2, 5]

    def values(n, seed):
        return torch.randn((n, 2, 64), generator=torch.Generator().manual_seed(seed)).bfloat16()

    def append(cache, seq, k, v):
        table, lens = pool.table([seq])
        cache.append(k, v, table.tolist(), lens.tolist(), [0, len(k)])

    def copy(cache, pairs):
        for a, b in pairs:
            for x in (cache.k, cache.v, cache.ks, cache.vs):
                x[b] = x[a]

    def held(cache, seq):
        table, lens = pool.table([seq])
        return [x for h in range(2) for x in cache.tokens(0, h, int(lens), table.tolist())[:2]]

    f8, ones = torch.float8_e4m3fn, torch.ones((9, 2))
    cache, plain = (oracle.Cache(torch.zeros((9, 2, page, 64)).to(f8), torch.zeros((9, 2, 64, page)).to(f8), ones, ones)
                    for _ in range(2))
    pool = kv_pages.KVPages(9, page)
    k, v = values(before, 1), values(before, 2)
    a = pool.new()
    pool.extend(a, before)
    append(cache, a, k, v)
    dk, dv = values(news, 3), values(news, 4)
    dk[1] *= 200
    dv[4] *= 100
    trunk = pool.fork(a) if forked else None
    copy(cache, pool.extend(a, news))
    append(cache, a, dk, dv)
    if forked:
        pool.free(a)
        a = trunk
    else:
        pool.truncate(a, before)
    copy(cache, pool.extend(a, len(kept)))
    append(cache, a, dk[kept], dv[kept])

    got = held(cache, a)
    pool = kv_pages.KVPages(9, page)
    b = pool.new()
    pool.extend(b, before)
    append(plain, b, k, v)
    pool.extend(b, len(kept))
    append(plain, b, dk[kept], dv[kept])
    same = all(torch.equal(x, y) for x, y in zip(got, held(plain, b)))
    assert same if forked or before % page == 0 else not same
