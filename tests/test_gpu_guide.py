"""The recipes of INTEGRATION.md for the 8-bit layer, run as they stand."""
from __future__ import annotations

import importlib

import pytest
import torch

from conftest import announce
from test_gpu_kv8 import BF16, i32, randn
from test_guide import BLOCKS

pytestmark = pytest.mark.gpu


def block(name):
    return next(code for code in BLOCKS if name in code)


def held(cache, pool, seq):
    """Keys and values of a sequence's tokens, and the scales that they lie at."""
    pages, n = list(pool.pages_of(seq)), pool.length(seq)
    at = torch.tensor(pages).cuda()
    k = cache.k.view(torch.uint8)[at].transpose(1, 2).flatten(0, 1)[:n]
    v = cache.v.view(torch.uint8)[at].permute(0, 3, 1, 2).flatten(0, 1)[:n]
    return [t.cpu() for t in (k, v, cache.k_scale[at], cache.v_scale[at])]


def test_the_guides_steps(ops):
    """Prompts, then a verified tree whose rejected drafts are far louder than the rest: the cache then holds what it would
    hold had the accepted tokens alone been appended, for the sequence and for its fork."""
    announce("the guide's steps")
    width, hidden = (32 + 2 * 8) * 128, 256
    space = {"importlib": importlib, "ops": ops, "torch": torch, "w": randn((width, hidden), 1, BF16, hidden ** -0.5).cuda(),
             "x": randn((237, hidden), 2, BF16).cuda()}
    exec(block("KVPages("), space)
    cache, pool, a, c = (space[n] for n in ("cache", "pool", "a", "c"))
    assert space["o"].shape == (237, 32, 128) and bool(space["o"].isfinite().all()) and pool.length(a) == 200
    fork = held(cache, pool, c)
    state = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    table, _ = pool.table([a])

    x = randn((6, hidden), 3, BF16)
    x[[1, 3, 4]] *= 1000.0
    norm = torch.ones(128, dtype=BF16).cuda()
    space.update(x=x.cuda(), q_norm=norm, k_norm=norm, logits=randn((6, 1000), 4, BF16).cuda(),
                 children=i32([[5, 7], [1, 2], [3, -1], [-1, -1], [-1, -1], [-1, -1]]))
    exec(block("ops.gqa_kv8_tree("), space)
    torch.cuda.synchronize()
    assert bool(space["o"].isfinite().all()) and space["ids"].shape == (6, 20)
    a = space["a"]
    assert pool.length(a) == 203 and all(torch.equal(s, t) for s, t in zip(held(cache, pool, c), fork))

    plain = ops.KV8Cache(*state)
    kept, k, v = space["kept"], space["k"], space["v"]
    ops.kv8_append(k[kept], v[kept], plain, table.cuda(), i32([203]), i32([0, 3]), 3)
    at = table[0].long().cuda()
    want = (plain.k.view(torch.uint8)[at].transpose(1, 2).flatten(0, 1)[:203],
            plain.v.view(torch.uint8)[at].permute(0, 3, 1, 2).flatten(0, 1)[:203], plain.k_scale[at], plain.v_scale[at])
    for got, exp in zip(held(cache, pool, a), want):
        assert torch.equal(got, exp.cpu())
