"""Windows and trees over 128 channels on pages of 64 tokens and more, whose kernels look a tile's one page up for all of it:
pages out of view, pages that are none, masks of all kinds and NaN codes, in every kernel form, and with split keys."""
from __future__ import annotations

import random

import pytest
import torch

from conftest import announce
from oracle import kv8 as oracle
from test_gpu_kv8 import BF16, F16, bound, filled, i32, prefix, randn, tables
from test_gpu_kv8_masks import (compare, crowd, in_tree, in_window, random_masks, run_tree, run_window, words_of)

pytestmark = pytest.mark.gpu

D = 128


def give_back(cache, table, lens, news, window, sinks, junk):
    """Junk for the pages that no row sees: a number that is no page, or a page (the cache's last) of NaN."""
    page, bad = cache.page, cache.pages - 1
    cache.k_scale[bad], cache.v_scale[bad] = float("nan"), 0.0
    cache.k.view(torch.uint8)[bad] = 0x7F
    cache.v.view(torch.uint8)[bad] = 0xFF
    given = 0
    for b, (len_, n) in enumerate(zip(lens, news)):
        for j in range(-(-len_ // page)):
            if j * page >= sinks and (j + 1) * page <= len_ - n - window + 1:
                table[b][j] = bad if junk == "page" else junk
                given += 1
    return given


def spoil(cache, table, places, k_at=()):
    """NaN codes of V at these (sequence, token), of K where named."""
    for b, t in places:
        p = table[b][t // cache.page]
        if t >= 0 and 0 <= p < cache.pages - 1:
            cache.v.view(torch.uint8)[p, 0, (7 * t) % D, t % cache.page] = 0x7F if t % 2 else 0xFF
            if (b, t) in k_at:
                cache.k.view(torch.uint8)[p, 0, t % cache.page, 5] = 0x7F


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("group,n", [(1, 1), (4, 3), (4, 13), (4, 70), (1, 200)])
@pytest.mark.parametrize("page", [64, 128])
def test_window_pages_out_of_view(ops, dtype, group, n, page):
    """As in the narrow form's test: pages given back, NaN codes beside the window, inside it and among the sinks."""
    announce(f"wide window out of view group{group} n{n} page{page} {dtype}")
    window, sinks = 150, 20
    lens, news = [700, 640], [n, n]
    for junk in (-1, 2 ** 30, "page"):
        cache = filled(ops, 30, 1, D, page, 10)
        table = tables(lens, page, 29, 11)
        assert give_back(cache, table, lens, news, window, sinks, junk)
        last = (0, lens[0] - 1 - n // 3)
        spoil(cache, table, [(0, lens[0] - window - 3), (0, lens[0] - window - n // 2), last, (0, sinks), (0, sinks - 1),
                             (1, lens[1] - 1)], [last])
        q = randn((2 * n, group, D), 12, dtype)
        run_window(ops, cache, q, table, lens, news, window, sinks, scale=0.02)


@pytest.mark.parametrize("page", [64, 128])
def test_window_bad_numbers(ops, page):
    """Pages in view that are none, fewer tokens than rows, lengths past the table, a negative scale, rows of no sequence."""
    announce(f"wide window bad numbers page{page}")
    cache = filled(ops, 9, 1, D, page, 16)
    table = [[0, 1, 2], [3, -9, 4], [5, 6, 7]]
    lens, news = [3 * page, 3 * page - 3, 30], [2, 130, 60]
    cu = [1 + c for c in prefix(news)]
    qkv = randn((cu[-1] + 2, 6 * D), 17, BF16)
    q = qkv[:, :4 * D].unflatten(1, (4, D))
    oc = oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)
    for window, sinks in ((9, 2), (page + 5, 0), (100, page + 3)):
        exp, weight, score = oc.attend(q, table, lens, cu, scale=-0.05, seen=in_window(lens, news, window, sinks))
        for empty, max_kv in ((0, None), (120, 1000), (600, 300)):
            t, l, n = crowd(table, [2 ** 31 - 1, *lens[1:]], news, empty, page) if empty else (table, [2 ** 31 - 1, *lens[1:]], news)
            if empty:  # as wide as the sequences are long, or the first one's length is another
                t = [r[:3] for r in t]
            out = torch.full(q.shape, 7.0, dtype=BF16, device="cuda")
            ops.gqa_kv8_window(qkv.cuda()[:, :4 * D].unflatten(1, (4, D)), cache, i32(t), i32(l), window, sinks,
                               i32([1 + c for c in prefix(n)]), 130, max_kv, scale=-0.05, out=out)
            got = out.cpu().double()
            assert bool((got[0] == 7).all()) and bool((got[-2:] == 7).all())
            rows = slice(1, cu[-1])
            assert bool(((got - exp).abs()[rows] <= bound(exp, weight, score, lens, D, BF16, cache.v_scale)[rows]).all())


@pytest.mark.parametrize("group,n", [(2, 5), (4, 13), (4, 60), (1, 300)])
@pytest.mark.parametrize("page", [64, 128])
def test_tree_masks(ops, group, n, page):
    """As in the narrow form's test: masks of nothing, of everything, of later tokens, of bits past the drafted tokens; fewer words than
    drafted tokens and more; NaN codes among the drafted tokens and before them."""
    announce(f"wide tree masks group{group} n{n} page{page}")
    lens, news = [n, n + 77, n + 130], [n, n, n]
    rng = random.Random(4)
    masks = [[rng.choice([0, (1 << n) - 1, 1 << n - 1, 1 << i, -1 % (1 << 1024), rng.getrandbits(n)]) for i in range(n)]
             for _ in news]
    cache = filled(ops, sum(-(-m // page) for m in lens) + 2, 1, D, page, 26)
    table = tables(lens, page, cache.pages - 1, 27)
    q = randn((sum(news), group, D), 28, BF16)
    for words in sorted({1, -(-n // 64), 16}):
        run_tree(ops, cache, q, table, lens, news, masks, words, scale=0.02)
    middle = [(b, lens[b] - n + n // 2) for b in range(3)]
    spoil(cache, table, [*middle, *((b, lens[b] - n + j) for b in range(3) for j in (0, n - 1)), (2, lens[2] - n - 1)], middle)
    run_tree(ops, cache, q, table, lens, news, masks, 16, scale=0.02)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("page", [64, 128])
def test_tree_bad_numbers(ops, dtype, page):
    """Fewer tokens than drafted rows, pages that are none, a negative scale."""
    announce(f"wide tree bad numbers page{page} {dtype}")
    n = 90
    cache = filled(ops, 10, 1, D, page, 32)
    table, lens, news = [[0, 1, 2], [3, -9, 4], [5, 6, 7]], [2 * page + 40, 2 * page + 45, 26], [n, n, n]
    masks = random_masks(random.Random(5), news)
    q = randn((3 * n, 4, D), 33, dtype)
    run_tree(ops, cache, q, table, lens, news, masks, scale=-0.05)


@pytest.mark.parametrize("page", [64, 128])
def test_split_keys_of_tiles(ops, page):
    """Split keys in the tile kernel with NaN codes on both sides of what rows see, and pages given back."""
    announce(f"wide split tiles page{page}")
    lens, news, empty = [5000, 3001, 90], [64, 33, 1], 137
    cache = filled(ops, sum(-(-n // page) for n in lens) + 2, 1, D, page, 60)
    table = tables(lens, page, cache.pages - 1, 61)
    q = randn((sum(news), 4, D), 62, BF16)
    masks = random_masks(random.Random(9), news)
    spoil(cache, table, [(0, 5000 - 30), (0, 5000 - 64), (1, 3001 - 20), (0, 5000 - 2500 - 40), (1, 99), (1, 700)], [(1, 3001 - 20)])

    def wide(table):
        t, l, n = crowd(table, lens, news, empty, page)
        return i32(t), i32(l), i32(prefix(n))

    t, l, cu = wide(table)
    assert ops.gqa_kv8_tree_workspace_bytes(140, 98, 64, 5000, 4, 1, D) > 0
    oc = oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)
    out = torch.full(q.shape, float("nan"), dtype=BF16, device="cuda")
    ops.gqa_kv8_tree(q.cuda(), cache, t, l, words_of(masks, 1), cu, 64, 5000, 0.02, out)
    compare(cache, oc, q, table, lens, news, in_tree(lens, news, masks), [out], 0.02)
    window, sinks = 2500, 100
    assert ops.gqa_kv8_window_workspace_bytes(140, 98, 64, 5000, 4, 1, D, window, sinks) > 0
    for junk in (-1, "page"):
        given = [list(r) for r in table]
        assert give_back(cache, given, lens, news, window, sinks, junk)
        t, l, cu = wide(given)
        oc = oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)
        out = torch.full(q.shape, float("nan"), dtype=BF16, device="cuda")
        ops.gqa_kv8_window(q.cuda(), cache, t, l, window, sinks, cu, 64, 5000, 0.02, out)
        compare(cache, oc, q, given, lens, news, in_window(lens, news, window, sinks), [out], 0.02)


@pytest.mark.parametrize("page", [64, 128])
def test_split_keys_of_blocks_of_32(ops, page):
    """Few KV heads, long sequences, 52 rows: blocks of 32 rows side by side whose keys are split."""
    announce(f"wide split blocks page{page}")
    lens, news, n_kv = [8300, 3000, 20], [13, 9, 13], 8
    cache = filled(ops, sum(-(-n // page) for n in lens) + 2, n_kv, D, page, 70)
    table = tables(lens, page, cache.pages - 1, 71)
    q = randn((sum(news), 4 * n_kv, D), 72, BF16)
    masks = random_masks(random.Random(11), news)
    spoil(cache, table, [(0, 8300 - 6), (0, 8300 - 7010), (1, 2995), (2, 15), (0, 99)], [(1, 2995)])
    assert ops.gqa_kv8_tree_workspace_bytes(3, 35, 13, 8300, 32, 8, D) > 0
    run_tree(ops, cache, q, table, lens, news, masks, scale=0.02, max_kv=8300)
    window, sinks = 7000, 100
    assert ops.gqa_kv8_window_workspace_bytes(3, 35, 13, 8300, 32, 8, D, window, sinks) > 0
    assert give_back(cache, table, lens, news, window, sinks, "page")
    run_window(ops, cache, q, table, lens, news, window, sinks, scale=0.02, max_kv=8300)
