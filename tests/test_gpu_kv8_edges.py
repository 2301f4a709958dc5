"""The paged 8-bit cache on the GPU at its edges: pages without tokens, queries that are no numbers, every 16-bit value,
split launches of each kernel form, scales far apart."""
from __future__ import annotations

import pytest
import torch

from conftest import announce
from oracle import kv8 as oracle
from test_gpu_kv8 import BF16, F16, bound, check_attend, filled, i32, prefix, randn, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("news", [[1, 1], [6, 2], [70, 30]])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 16), (64, 32), (128, 32), (64, 64), (128, 64), (128, 128)])
def test_pages_of_no_token_do_not_count(ops, d, page, news, dtype):
    """Pages that the table names behind a sequence's last token, not written yet: whatever their codes and scales
    are, zeros, infinities or NaN, the outputs are bit for bit those with ordinary ones."""
    announce(f"gqa_kv8 pages behind the last token d{d} page{page} {news} {dtype}")
    lens = [max(20, news[0]), 1090]
    pages = sum(-(-n // page) for n in lens) + 9
    cache = filled(ops, pages, 2, d, page, 1)
    table = tables(lens, page, pages - 8, 2, columns=-(-lens[1] // page) + 4)
    for row in table:
        first = row.index(-1)
        row[first:] = [pages - 8 + i % 8 for i in range(len(row) - first)]
    q = randn((sum(news), 8, d), 3, dtype, 0.1).cuda()
    more = () if news == [1, 1] else (i32(prefix(news)), max(news))
    args = (q, cache, i32(table), i32(lens), *more)
    want = [ops.gqa_kv8(*args, causal=causal) for causal in (True, False)]
    assert all(bool(w.isfinite().all()) for w in want)
    cache.k.view(torch.uint8)[-8:] = 0x7F
    cache.v.view(torch.uint8)[-8:] = 0x7F
    for bad in (0.0, float("inf"), float("nan")):
        cache.k_scale[-8:] = bad
        cache.v_scale[-8:] = bad
        for causal, w in zip((True, False), want):
            assert torch.equal(ops.gqa_kv8(*args, causal=causal), w)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("news", [[1, 1, 1], [5, 3, 4], [90, 40, 70]])
def test_queries_that_are_no_numbers_and_see_nothing(ops, news, d, page, dtype):
    """Queries with a NaN or an infinity: zeros where every page of what they could see is none, NaN where one is
    there (all scores of such a query are infinite or NaN)."""
    announce(f"gqa_kv8 queries of NaN d{d} page{page} {news} {dtype}")
    lens = [500, 300, 420]
    pages = 80
    cache = filled(ops, pages, 2, d, page, 4)
    table = tables(lens, page, pages, 5)
    table[0] = [-1, pages] * (len(table[0]) // 2) + [-7] * (len(table[0]) % 2)   # none at all
    table[1][0] = -1                                                             # some
    table[2] = [-1 if page * (j + 1) <= lens[2] - news[2] // 2 else p for j, p in enumerate(table[2])]
    q = randn((sum(news), 4, d), 6, dtype, 0.1)
    for b, first in enumerate(prefix(news)[:-1]):
        q[first, 0, 3] = float("nan")
        q[first + news[b] - 1, 1, d - 1] = float("inf")
        q[first + news[b] // 2, 2, d // 2] = float("-inf")
        q[first + news[b] // 3, 3, ::7] = float("nan")
    for causal in (True, False):
        exp, _, _ = check_attend(ops, cache, q, table, lens, news, causal)
        assert bool((exp[:news[0]] == 0).all()) and bool(exp[news[0]:].isnan().any())


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_append_every_value(ops, dtype):
    """Every finite 16-bit value that fits, as keys and as values of a page with a present scale from 2^-32 to 2^127
    (one token before keeps it): the nearest code of the exact quotient, ties to even."""
    announce(f"kv8_append every value {dtype}")
    d = page = 128
    exps = [-32, -31, -20, -9, -1, 0, 1, 7, 30, 60, 119, 120, 121, 126, 127]
    bits = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16).view(dtype)
    bits = bits[bits.isfinite()]
    n_kv = -(-bits.numel() // ((page - 1) * d))
    x = torch.zeros(n_kv * (page - 1) * d, dtype=dtype)
    x[:bits.numel()] = bits
    x = x.reshape(page - 1, n_kv, d)
    cache = ops.KV8Cache.empty(len(exps), n_kv, d, page)
    scale = torch.tensor([2.0 ** e for e in exps])
    cache.k_scale.copy_(scale[:, None].expand(-1, n_kv))
    cache.v_scale.copy_(scale[:, None].expand(-1, n_kv))
    parts = [torch.where(x.double().abs() <= 448 * 2.0 ** e, x, torch.zeros_like(x)) for e in exps]
    k = torch.cat(parts).cuda()
    table, lens = i32([[b] for b in range(len(exps))]), i32([page] * len(exps))
    ops.kv8_append(k, -k, cache, table, lens, i32([b * (page - 1) for b in range(len(exps) + 1)]), page - 1)
    for got in (cache.k_scale, cache.v_scale):
        assert torch.equal(got.cpu(), scale[:, None].expand(-1, n_kv))
    for b, (e, part) in enumerate(zip(exps, parts)):
        want = oracle.nearest_e4m3(part.double() * 2.0 ** -e).transpose(0, 1)
        got = cache.k[b].cpu().float().double()[:, 1:], -cache.v[b].cpu().float().double().transpose(1, 2)[:, 1:]
        for g in got:
            assert torch.equal(g, want), f"scale 2^{e}: {int((g != want).sum())} codes"


# d, page, n_kv, group, lens, news: see test_split_launches_cover_each_kernel in test_kv8_host.py
SPLIT = [
    (128, 16, 1, 4, [600, 530], [1, 1]),
    (64, 32, 3, 1, [1200, 40], [1, 1]),
    (128, 64, 1, 7, [700, 515], [2, 1]),
    (64, 128, 2, 5, [1100, 1030], [3, 2]),
    (128, 32, 2, 8, [700, 520], [3, 4]),
    (128, 16, 1, 5, [550, 1030], [4, 5]),
    (64, 16, 2, 12, [1100, 1050], [2, 2]),
    (128, 64, 1, 7, [1030, 600], [4, 3]),
    (64, 128, 1, 10, [1300, 90], [3, 1]),
    (128, 16, 1, 3, [300, 700], [40, 90]),
    (64, 32, 2, 2, [290, 500], [130, 61]),
    (128, 128, 2, 2, [300, 500], [150, 61]),
    (64, 64, 1, 4, [300, 640], [150, 300]),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", range(len(SPLIT)))
def test_attend_split(ops, case, causal, dtype):
    """Every kernel form with its keys split: NaN codes of V among the last tokens and, without a causal mask, one
    that every row sees; codes behind the last token and pages behind the last one are NaN."""
    d, page, n_kv, group, lens, news = SPLIT[case]
    announce(f"gqa_kv8 split d{d} page{page} n_kv{n_kv} group{group} {lens} {news} causal={causal} {dtype}")
    pages = sum(-(-n // page) for n in lens) + 2
    cache = filled(ops, pages, n_kv, d, page, case)
    table = tables(lens, page, pages, case)
    v = cache.v.view(torch.uint8)
    for row, n in zip(table, lens):
        if n % page:
            cache.k.view(torch.uint8)[row[n // page], :, n % page:] = 0x7F
            v[row[n // page], :, :, n % page:] = 0xFF
        for t, c in ((n - 1, 5), (n - 2, d - 1), (n - 9, 17)) if causal else ((n // 2, 5),):
            v[row[t // page], n_kv - 1, c, t % page] = 0x7F
    q = randn((sum(news), n_kv * group, d), 100 + case, dtype, 0.02)
    check_attend(ops, cache, q, table, lens, news, causal)


@pytest.mark.parametrize("news,apart", [([1], 27), ([16], 27), ([20], 23), ([100], 23)])
def test_attend_one_token_on_a_quiet_page(ops, news, apart):
    """f16: a channel that a single token holds, whose page's scale lies 2^27 below the others' (2^23 where a KV head has
    more than 32 rows, here two a token).  The row's largest P' is put at 2^15 (2^10 or above) and scores are
    below 1/8, so the token's P' is 2^(15 - 27 - 1/2) or 2^(10 - 23 - 1/2), more than 2^-14: a normal f16, and so is the
    output.  The channel then has the relative error of any other: the roundings of P' and of the output, 2^-11 each, and
    what the fp32 steps add (2^-15 is ample)."""
    announce(f"gqa_kv8 one quiet token {news}")
    n, page, d = 100, 16, 64
    cache = filled(ops, 7, 1, d, page, 3)
    table = [[4, 0, 2, 1, 3, 6, 5]]
    loud = 2.0 ** (apart - 9)
    cache.k_scale.fill_(2.0 ** -9)
    cache.v_scale.fill_(loud)
    cache.v_scale[2] = 2.0 ** -9                       # tokens 32 .. 47
    v = cache.v.view(torch.uint8)
    v.copy_((torch.arange(v.numel()) % 4).reshape(v.shape).to(torch.uint8))    # 0 .. 3 * 2^-9
    v[:, :, 0] = 0
    v[2, :, 0, 5] = 0x7E                               # 448: 0.875 with its scale, about 0.00875 in the output
    q = randn((news[0], 2, d), 5, F16, 0.002)
    exp, _, score = oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale).attend(q, table, [n], prefix(news), False)
    assert float(score.max()) < 1 / 8 and bool((exp[..., 0] > 2.0 ** -8).all()) and bool((exp[..., 0] < 2.0 ** -6).all())
    more = {} if news == [1] else {"cu_q": i32(prefix(news)), "max_q": news[0]}
    got = ops.gqa_kv8(q.cuda(), cache, i32(table), i32([n]), causal=False, **more).cpu().double()[..., 0]
    exp = exp[..., 0]
    assert bool(((got - exp).abs() <= exp * (2 * 2.0 ** -11 + 2.0 ** -15)).all())


@pytest.mark.parametrize("news", [[1], [20], [100]])
@pytest.mark.parametrize("e", [-90, 119])
def test_attend_scales_of_any_size(ops, e, news):
    """V's scales around 2^-90 or 2^119 (bf16, whose outputs reach as far)."""
    announce(f"gqa_kv8 V scales around 2^{e} {news}")
    n, page = 700, 32
    cache = filled(ops, 24, 1, 64, page, 7)
    cache.v_scale.copy_(torch.exp2(torch.rand((24, 1), generator=torch.Generator().manual_seed(3)) + e).cuda())
    q = randn((news[0], 2, 64), 5, BF16, 0.1)
    table = tables([n], page, 24, 2)
    exp, weight, score = oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale).attend(q, table, [n], prefix(news))
    more = {} if news == [1] else {"cu_q": i32(prefix(news)), "max_q": news[0]}
    got = ops.gqa_kv8(q.cuda(), cache, i32(table), i32([n]), **more).cpu().double()
    half = 2.0 ** -8
    delta = 2.0 ** -24 * ((64 + 16) * score + 64) + 2.0 ** -21
    rel = half * 1.01 + 2 * delta[..., None] + 2 * (n + 8) * 2.0 ** -24
    # sums of P' v8 vanish below 2^-126 times the scale of the largest, as the P' do: 2^-126 of 448 a token
    assert bool(((got - exp).abs() <= weight * rel + exp.abs() * half + 2.0 ** -126 * n * 448 * 2.0 ** (e + 1)).all())


def test_copies_of_more_pages_than_one_launch_takes(ops):
    """2^22 + 3 pairs of 1 KB pages: all but some near both ends name no page and are skipped."""
    announce("kv8_copy_pages of 2^22 + 3 pairs")
    cache = filled(ops, 40, 1, 64, 16, 1)
    was = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)]
    n = 2 ** 22 + 3
    src, dst = (torch.full((n,), -1, dtype=torch.int32, device="cuda") for _ in range(2))
    for i, (a, b) in {0: (3, 20), 7: (4, 21), 2 ** 22 - 1: (5, 22), 2 ** 22: (6, 23), n - 1: (3, 24)}.items():
        src[i], dst[i] = a, b
        for t in was:
            t[b] = t[a]
    ops.kv8_copy_pages(cache, src, dst)
    for t, e in zip((cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale), was):
        assert torch.equal(t, e)


@pytest.mark.parametrize("wide", [2048, 2100, 100000])
def test_a_workspace_of_the_calls_own_hints(ops, wide):
    """A workspace of gqa_kv8_workspace_bytes' size for the hints of the call, max_kv among them, is enough, also where
    max_kv is more than the table holds."""
    announce(f"gqa_kv8 workspace of its own hints, max_kv {wide}")
    cache = filled(ops, 130, 8, 128, 64, 1)
    lens = [2048, 1900, 700, 64]
    table = tables(lens, 64, 130, 2, columns=32)
    q = randn((4, 32, 128), 3, BF16, 0.02)
    need = ops.gqa_kv8_workspace_bytes(4, 4, 1, wide, 32, 8, 128)
    assert need
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    check_attend(ops, cache, q, table, lens, [1] * 4, max_kv=wide, workspace=ws)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,page,news", [(128, 64, [3, 0, 2, 5, 1]), (64, 16, [4, 0, 3, 1, 6]), (128, 16, [7, 0, 5, 8, 2]),
                                         (64, 64, [90, 0, 40, 70, 33]), (128, 32, [90, 0, 40, 70, 33])])
def test_rows_of_none_with_split_keys(ops, d, page, news, dtype, causal):
    """Keys split over workgroups: rows before the first and behind the last sequence stay as they are, sequences of no
    rows and of no tokens, more rows than tokens, lengths past the table, pages that are none."""
    announce(f"gqa_kv8 rows of none, split keys, d{d} page{page} {news} {dtype} causal={causal}")
    lens = [1200, 900, 0, 1100, 17 if news[4] > 17 else 1]
    pages = sum(-(-n // page) for n in lens) + 2
    cache = filled(ops, pages, 2, d, page, 3)
    table = tables(lens, page, pages, 4)
    for j in range(5, 12):
        table[0][j] = -1 if j % 2 else pages
    cu = [4 + c for c in prefix(news)]
    q = randn((cu[-1] + 5, 6, d), 5, dtype, 0.05)
    oc = oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)
    exp, weight, score = oc.attend(q, table, lens, cu, causal)
    out = torch.full(q.shape, 7.0, dtype=dtype, device="cuda")
    asked = ops.gqa_kv8_workspace_bytes(5, q.shape[0], max(news), len(table[0]) * page, 6, 2, d)
    assert asked, "the keys are split"
    ops.gqa_kv8(q.cuda(), cache, i32(table), i32([2 ** 31 - 1 if n == 1200 and 1200 % page == 0 else n for n in lens]), i32(cu),
                max_q=max(news), causal=causal, out=out)
    got = out.cpu().double()
    assert bool((got[:cu[0]] == 7).all()) and bool((got[cu[-1]:] == 7).all())
    rows = slice(cu[0], cu[-1])
    limit = bound(exp, weight, score, lens, d, dtype, cache.v_scale)
    assert bool(((got - exp).abs() <= limit)[rows].all())
    assert bool((got[cu[2]:cu[3]] == 0).all())
    # ranges that begin below 0 and end past the rows: cut
    wild = [-5, *cu[1:-1], q.shape[0] + 9]
    cut = [0, *cu[1:-1], q.shape[0]]
    a, b = (ops.gqa_kv8(q.cuda(), cache, i32(table), i32(lens), i32(c), max_q=max(news) + 14, causal=causal) for c in (wild, cut))
    assert torch.equal(a, b)


def test_a_workspace_of_the_tables_width(ops):
    """max_kv past the table's width: a workspace for either serves, one that is too small for both is refused."""
    announce("gqa_kv8 max_kv past the table, workspaces")
    cache = filled(ops, 130, 8, 128, 64, 1)
    lens = [2048, 1900, 700, 64]
    table = tables(lens, 64, 130, 2, columns=32)
    q = randn((4, 32, 128), 3, BF16, 0.02)
    size = {n: ops.gqa_kv8_workspace_bytes(4, 4, 1, n, 32, 8, 128) for n in (2048, 2100, 4096)}
    assert size[2100] < size[2048]
    for hint, ws in ((2100, size[2100]), (2100, size[2048]), (4096, size[2048]), (4096, size[4096])):
        ws = torch.empty(ws, dtype=torch.uint8, device="cuda")
        check_attend(ops, cache, q, table, lens, [1] * 4, max_kv=hint, workspace=ws)
    small = torch.empty(size[2100] - 16, dtype=torch.uint8, device="cuda")
    for hint in (2048, 2100, None):
        with pytest.raises(RuntimeError, match="workspace"):
            ops.gqa_kv8(q.cuda(), cache, i32(table), i32(lens), max_kv=hint, workspace=small)
