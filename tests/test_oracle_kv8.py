"""The oracle of the 8-bit cache against torch's e4m3, closed forms and the dense attention oracle."""
from __future__ import annotations

import math

import torch

from oracle import kv8
from oracle.gqa import gqa_naive


def empty(pages, n_kv, page, d):
    f8 = torch.float8_e4m3fn
    return kv8.Cache(torch.zeros((pages, n_kv, page, d)).to(f8), torch.zeros((pages, n_kv, d, page)).to(f8),
                     torch.ones((pages, n_kv)), torch.ones((pages, n_kv)))


def test_nearest_is_torchs_cast():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().double()
    fin = codes[codes.isfinite()]
    assert torch.equal(kv8.nearest_e4m3(fin), fin)
    x = torch.cat([torch.randn(20000, generator=torch.Generator().manual_seed(1)) * 100, (fin[:-1] + fin[1:]).float() / 2])
    x = x[x.abs() <= 448]
    assert torch.equal(kv8.nearest_e4m3(x.double()), x.to(torch.float8_e4m3fn).double())


def test_scale():
    assert [kv8.scale_for(x) for x in (0.0, 448.0, 449.0, 1.0, 1.75, 1.7501)] == [2.0 ** -32, 1, 2, 2 ** -8, 2 ** -8, 2 ** -7]


def test_append_in_one_call_and_token_by_token():
    """The same tokens give the same values either way but for codes among the smallest, which may be rounded again."""
    k, v = (torch.randn((40, 2, 64), generator=torch.Generator().manual_seed(s)).bfloat16() for s in (1, 2))
    one, many = empty(4, 2, 16, 64), empty(4, 2, 16, 64)
    table = [[2, 0, 3]]
    one.append(k, v, table, [40], [0, 40])
    for t in range(40):
        many.append(k[t:t + 1], v[t:t + 1], table, [t + 1], [0, 1])
    assert torch.equal(one.ks, many.ks) and torch.equal(one.vs, many.vs)
    assert ((one.k - many.k).abs() <= 2.0 ** -9).all()
    for h in range(2):
        values, _, present = one.tokens(0, h, 40, table)
        assert present.all() and ((values - k[:, h].double()).abs() <= k[:, h].double().abs() / 16 + one.ks.max() / 1024).all()


def test_attention_is_the_dense_one():
    cache = empty(6, 2, 16, 64)
    k, v, q = (torch.randn((50, n, 64), generator=torch.Generator().manual_seed(n)).bfloat16() for n in (2, 2, 6))
    table = [[5, 1, 0, 2]]
    cache.append(k, v, table, [50], [0, 50])
    kk, vv = (torch.stack([cache.tokens(0, h, 50, table)[i] for h in range(2)])[None].float() for i in range(2))
    for causal in (True, False):
        want = gqa_naive(q.transpose(0, 1)[None], kk, vv, causal)[0].transpose(0, 1)
        out, weight, _ = cache.attend(q, table, [50], [0, 50], causal)
        assert (out - want).abs().max() < 1e-5 and (weight >= out.abs() - 1e-12).all()


def test_rows_that_see_nothing():
    cache = empty(2, 1, 16, 64)
    q = torch.ones((6, 1, 64))
    out, _, _ = cache.attend(q, [[0], [-1]], [2, 9], [0, 4, 5])
    assert (out[:2] == 0).all() and (out[4] == 0).all() and math.isnan(out[5, 0, 0])
