"""The paged 8-bit cache on the GPU: append, attention, page copies, against the 64-bit oracle."""
from __future__ import annotations

import itertools

import pytest
import torch

from conftest import announce, import_submodule
from oracle import int8 as oint8
from oracle import kv8 as oracle

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def randn(shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def prefix(news):
    return [sum(news[:b]) for b in range(len(news) + 1)]


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def filled(ops, pages, n_kv, d, page, seed, spread=3.0):
    """A cache of random codes (every bit pattern but NaN) and powers of two as scales."""
    g = torch.Generator().manual_seed(seed)

    def codes(shape):
        c = torch.randint(0, 256, shape, generator=g, dtype=torch.int32).to(torch.uint8)
        c[(c & 0x7F) == 0x7F] = 0x31
        return c.cuda().view(torch.float8_e4m3fn)

    def scales():
        return torch.exp2(torch.round(torch.rand((pages, n_kv), generator=g) * spread) - 9).cuda()

    return ops.KV8Cache(codes((pages, n_kv, page, d)), codes((pages, n_kv, d, page)), scales(), scales())


def tables(lens, page, pages, seed, columns=None, unused=-1):
    """Pages of each sequence, in no order; `unused` behind a sequence's last."""
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    need = [-(-n // page) for n in lens]
    columns = columns or max(1, max(need))
    out = []
    for n in need:
        out.append([order.pop() for _ in range(n)] + [unused] * (columns - n))
    return out


def assert_cache(cache, want):
    for got, exp in ((cache.k, want.k), (cache.v, want.v.transpose(2, 3))):
        got = got.cpu().float().double()
        assert torch.equal(got.isnan(), exp.isnan())
        assert torch.equal(got.nan_to_num(), exp.nan_to_num())
    for got, exp in ((cache.k_scale, want.ks), (cache.v_scale, want.vs)):
        assert torch.equal(got.cpu().double(), exp)


def bound(out, weight, score, lens, d, dtype, vs):
    """How far an output may be off.  Roundings of P' (half a step) and of the output; the scores' fp32 sums of d
    products and the steps to the exponent (some 16 more, relative to the largest sum of |q k|, and to at most
    64 for the exponent itself), the exponential (2^-21), the two fp32 sums over the tokens.  In f16, P' below
    2^-14 is off by up to 2^-25 of 448 vs a token, and the output by 2^-25.  fp32 and bf16 have no normal numbers
    below 2^-126: an exponential below it (a weight of 10^-38 and less) may be 0, which is off by up to 2^-126 of
    448 vs a token, and so may the output."""
    half = torch.finfo(dtype).eps / 2
    delta = 2.0 ** -24 * ((d + 16) * score + 64) + 2.0 ** -21
    rel = half * 1.01 + 2 * delta[..., None] + 2 * (max(lens) + 8) * 2.0 ** -24
    least = 2.0 ** -25 if dtype == F16 else 2.0 ** -126
    floor = least * (max(lens) * 448 * float(vs.max()) + 1)
    return weight * rel + out.abs() * half + floor


def check_attend(ops, cache, q, table, lens, news, causal=True, scale=None, want=None, **hints):
    cu = prefix(news)
    oc = oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)
    exp, weight, score = want or oc.attend(q, table, lens, cu, causal, scale)
    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    more = {} if news == [1] * len(news) else {"cu_q": i32(cu), "max_q": max(max(news), 1)}
    ops.gqa_kv8(q.cuda(), cache, i32(table), i32(lens), causal=causal, scale=scale, out=out, **{**more, **hints})
    got = out.cpu().double()
    assert torch.equal(got.isnan(), exp.isnan())
    off = (got - exp).abs()
    ok = (off <= bound(exp, weight, score, lens, cache.d, q.dtype, cache.v_scale)) | exp.isnan()
    assert bool(ok.all()), f"{int((~ok).sum())} of {ok.numel()} outputs are off, by up to {float(off.nan_to_num().max())}"
    return exp, weight, score


# ---- append ---------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,page,n_kv", [(64, 16, 1), (128, 16, 3), (64, 32, 2), (128, 32, 2), (64, 64, 1), (128, 64, 8),
                                         (64, 128, 2), (128, 128, 2)])
def test_append(ops, dtype, d, page, n_kv):
    """Single tokens, chunks that begin and end inside pages or on their edges, a sequence with nothing new, one whose
    new tokens are louder than what its page holds, over a pool whose other pages stay as they are."""
    announce(f"kv8_append d{d} page{page} n_kv{n_kv} {dtype}")
    lens = [1, page, page + 1, 3 * page, 2 * page - 1, 5, 2 * page + 7, 4]
    news = [1, 1, 1, 2 * page + 3, page + 2, 0, 7, 4]
    pages = sum(-(-n // page) for n in lens) + 3
    cache = filled(ops, pages, n_kv, d, page, 1)
    want = oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)
    table, cu = tables(lens, page, pages, 2), prefix(news)
    k, v = randn((cu[-1], n_kv, d), 3, dtype), randn((cu[-1], n_kv, d), 4, dtype)
    k[cu[2]:cu[3]] *= 40
    v[cu[6]:cu[7]] *= 300
    want.append(k, v, table, lens, cu)
    ops.kv8_append(k.cuda(), v.cuda(), cache, i32(table), i32(lens), i32(cu), max(news))
    assert_cache(cache, want)


def test_append_one_by_one(ops):
    """Tokens of growing and falling magnitude, one call each, as decoding makes them: the page's scale follows the
    largest, and a page that is begun anew forgets what it held."""
    announce("kv8_append one by one")
    cache = filled(ops, 4, 2, 64, 16, 5)
    want = oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)
    table = [[2, 0, 3]]
    for t in range(40):
        k, v = randn((1, 2, 64), 2 * t, BF16, 2.0 ** (t % 7 - 3)), randn((1, 2, 64), 2 * t + 1, BF16, 1.7 ** (t % 5))
        want.append(k, v, table, [t + 1], [0, 1])
        ops.kv8_append(k.cuda(), v.cuda(), cache, i32(table), i32([t + 1]))
    assert_cache(cache, want)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_append_special_values(ops, dtype):
    """Zeros, the type's extremes and subnormals, exact ties, infinities and NaNs (which poison themselves alone)."""
    announce(f"kv8_append special values {dtype}")
    cache = filled(ops, 8, 1, 64, 16, 6)
    want = oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)
    x = torch.zeros((7, 1, 64), dtype=dtype)
    x[1] = torch.finfo(dtype).max
    x[2] = torch.finfo(dtype).smallest_normal / 4
    x[3, 0] = (torch.arange(64) + 0.5) * 0.25
    x[3, 0, 0] = 448
    x[4, 0, ::5] = float("inf")
    x[4, 0, 1::5] = float("nan")
    x[4, 0, 2::5] = 3.0
    x[5] = float("-inf")
    x[6, 0] = 448.5 if dtype == F16 else 450
    table = [[b] for b in range(7)]
    want.append(x, -x, table, [1] * 7, list(range(8)))
    ops.kv8_append(x.cuda(), (-x).cuda(), cache, i32(table), i32([1] * 7))
    assert_cache(cache, want)


def test_append_strides_hints_and_bad_numbers(ops):
    """Views of a fused projection; a max_q below the truth; more rows than tokens; lengths past the table or below
    zero; page numbers that are none; rows outside cu: nothing but what the rules name is written."""
    announce("kv8_append strides, hints, bad numbers")
    n_kv, d, page = 2, 64, 16
    cache = filled(ops, 9, n_kv, d, page, 7)
    want = oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)
    table = [[0, 1, 2], [3, 9, 4], [-7, 5, 6], [7, 8, -1]]
    news = [40, 45, 30, 5]
    cu = [2 + c for c in prefix(news)]
    qkv = randn((cu[-1] + 4, 8 * d), 8, BF16)
    k, v = qkv[:, 4 * d:6 * d].unflatten(1, (n_kv, d)), qkv[:, 6 * d:].unflatten(1, (n_kv, d))
    lens = [48, 46, 32, 2]  # the last has fewer tokens than rows
    want.append(k, v, table, lens, cu)
    qkv = qkv.cuda()
    ops.kv8_append(qkv[:, 4 * d:6 * d].unflatten(1, (n_kv, d)), qkv[:, 6 * d:].unflatten(1, (n_kv, d)), cache, i32(table),
                   i32(lens), i32(cu), max_q=1)
    assert_cache(cache, want)
    ops.kv8_append(qkv[:4, 4 * d:6 * d].unflatten(1, (n_kv, d)), qkv[:4, 6 * d:].unflatten(1, (n_kv, d)), cache, i32(table),
                   i32([-3, 0, -2 ** 31, 0]))
    assert_cache(cache, want)
    cut = [48 if n > 48 else n for n in (2 ** 31 - 1, 46, 32, 2)]
    want.append(k[:4], v[:4], table, cut, [0, 1, 2, 3, 4])
    ops.kv8_append(qkv[:4, 4 * d:6 * d].unflatten(1, (n_kv, d)), qkv[:4, 6 * d:].unflatten(1, (n_kv, d)), cache, i32(table),
                   i32([2 ** 31 - 1, 46, 32, 2]))
    assert_cache(cache, want)


def test_append_to_other_scales(ops):
    """Pages whose present scale is no power of two: it stays where it is large enough, and every code, kept or
    new, is the nearest one up to fp32's rounding of the quotient (the scale's reciprocal, the product: 2^-23 of it)."""
    announce("kv8_append to scales that are no powers of two")
    n_kv, d, page = 2, 64, 32
    for dtype, loud in itertools.product((BF16, F16), (8, 1)):
        cache = filled(ops, 6, n_kv, d, page, 9)
        s = torch.rand((2, 6, n_kv), generator=torch.Generator().manual_seed(1)) * 0.02 + 0.001
        cache.k_scale.copy_(s[0])
        cache.v_scale.copy_(s[1])
        want = oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)
        was = [want.k * s[0][:, :, None, None], want.v * s[1][:, :, None, None]]
        table, lens, cu = [[0], [1], [2], [3]], [20, 32, 9, 4], [0, 3, 10, 11, 15]
        k, v = randn((15, n_kv, d), 3, dtype), randn((15, n_kv, d), 4, dtype, loud)
        want.append(k, v, table, lens, cu)
        ops.kv8_append(k.cuda(), v.cuda(), cache, i32(table), i32(lens), i32(cu), 7)
        for code, exp, scale, exp_s, x, old in ((cache.k, want.k, cache.k_scale, want.ks, k, was[0]),
                                                (cache.v.transpose(2, 3), want.v, cache.v_scale, want.vs, v, was[1])):
            assert torch.equal(scale.cpu().double(), exp_s)
            assert bool((exp_s[3].log2().frac() == 0).all())
            if x is k or loud == 1:
                assert bool((exp_s[:3].log2().frac() != 0).any())
            for b in range(4):
                n = cu[b + 1] - cu[b]
                true = old[b].clone()
                true[:, lens[b] - n:lens[b]] = x[cu[b]:cu[b + 1]].double().transpose(0, 1)
                step = exp_s[b][:, None, None]
                err = (code[b].cpu().double() * step - true)[:, :lens[b]].abs()
                best = (exp[b] * step - true)[:, :lens[b]].abs()
                assert bool((err <= best + 2 * 2.0 ** -23 * true[:, :lens[b]].abs()).all())
                behind = torch.equal(code[b].cpu().double()[:, lens[b]:], exp[b][:, lens[b]:])
                assert behind


def test_one_row_of_any_stride(ops):
    announce("kv8 one row of any stride")
    cache, other = (filled(ops, 4, 2, 64, 16, 1) for _ in range(2))
    table, lens = i32([[2, 1]]), i32([20])
    q, k, v = (randn((1, n, 64), n, BF16, 0.1).cuda() for n in (4, 2, 2))
    ops.kv8_append(k, v, other, table, lens)
    want = ops.gqa_kv8(q, other, table, lens)
    for stride in (0, 7, 10 ** 10):
        far = [t.as_strided(t.shape, (stride, 64, 1)) for t in (q, k, v)]
        ops.kv8_append(far[1], far[2], cache, table, lens)
        assert torch.equal(cache.k.view(torch.uint8), other.k.view(torch.uint8))
        assert torch.equal(cache.v.view(torch.uint8), other.v.view(torch.uint8))
        assert torch.equal(ops.gqa_kv8(far[0], cache, table, lens), want)


def test_tables_too_large_are_refused(ops):
    announce("kv8 table of more than 2^30 tokens")
    cache = filled(ops, 4, 1, 64, 16, 1)
    q = randn((1, 1, 64), 1, BF16).cuda()
    table = torch.zeros((1, 2 ** 26 + 1), dtype=torch.int32, device="cuda")
    for call in (lambda: ops.kv8_append(q, q, cache, table, i32([5])), lambda: ops.gqa_kv8(q, cache, table, i32([5]))):
        with pytest.raises(ValueError, match="too large"):
            call()
    # the widest one, all of it the same page: as many tokens as are there count
    table = table[:, :2 ** 26].contiguous()
    assert torch.equal(ops.gqa_kv8(q, cache, table, i32([5])), ops.gqa_kv8(q, cache, i32([[0]]), i32([5])))


# ---- attention ------------------------------------------------------------
ATTEND = [
    # d, page, n_kv, group, dtype, lens, news
    (128, 64, 8, 4, BF16, [1, 64, 65, 1000, 300], [1] * 5),
    (128, 64, 1, 1, F16, [1, 2, 63, 127, 129], [1] * 5),
    (64, 16, 3, 1, F16, [17, 500, 255], [1] * 3),
    (64, 32, 2, 7, BF16, [33, 700], [1, 1]),
    (128, 128, 2, 16, F16, [129, 640, 5], [1] * 3),
    (64, 128, 1, 32, BF16, [100, 128], [1, 1]),
    (128, 16, 2, 4, BF16, [90, 300, 70], [2, 4, 3]),
    (64, 64, 2, 2, F16, [64, 513], [8, 5]),
    (128, 64, 2, 8, F16, [200, 70, 3], [4, 1, 3]),
    (128, 64, 1, 48, BF16, [150], [1]),
    (128, 64, 2, 4, BF16, [300, 130, 65, 64], [300, 67, 1, 64]),
    (64, 16, 1, 8, F16, [257, 100], [100, 100]),
    (128, 32, 2, 1, F16, [400, 33], [290, 33]),
    (64, 128, 2, 3, BF16, [500, 129], [129, 128]),
    (128, 16, 1, 7, BF16, [90, 200], [80, 37]),
    (64, 64, 3, 2, BF16, [64, 65, 1], [64, 65, 1]),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attend(ops, case, causal):
    """Pages behind a sequence's last token hold NaN codes, as do the slots behind it on its last page."""
    d, page, n_kv, group, dtype, lens, news = ATTEND[case]
    announce(f"gqa_kv8 d{d} page{page} n_kv{n_kv} group{group} {dtype} {lens} {news} causal={causal}")
    pages = sum(-(-n // page) for n in lens) + 2
    cache = filled(ops, pages, n_kv, d, page, case)
    table = tables(lens, page, pages, case, columns=max(-(-n // page) for n in lens) + 1)
    for row, n in zip(table, lens):
        if n % page:
            cache.k.view(torch.uint8)[row[n // page], :, n % page:] = 0x7F
            cache.v.view(torch.uint8)[row[n // page], :, :, n % page:] = 0xFF
    q = randn((sum(news), n_kv * group, d), 100 + case, dtype, 0.02)
    check_attend(ops, cache, q, table, lens, news, causal)


@pytest.mark.parametrize("news", [[1, 1], [5, 3], [150, 40]])
def test_attend_scales_far_apart_and_negative(ops, news):
    """Pages whose scales lie 2^20 apart (any positive numbers, no powers of two), and a negative softmax scale."""
    announce(f"gqa_kv8 scales far apart {news}")
    lens = [200, 160]
    for dtype, scale in ((BF16, None), (F16, -0.3), (F16, 0.0)):
        cache = filled(ops, 25, 2, 64, 16, 3)
        s = torch.exp2(torch.rand((2, 25, 2), generator=torch.Generator().manual_seed(4)) * 20 - 25).cuda()
        cache.v_scale.copy_(s[0])
        cache.k_scale.copy_(s[1] * 2 ** 12)
        q = randn((sum(news), 4, 64), 5, dtype, 0.1)
        check_attend(ops, cache, q, tables(lens, 16, 25, 6), lens, news, scale=scale)


@pytest.mark.parametrize("news", [[1], [20], [100]])
def test_attend_channel_on_quiet_pages(ops, news):
    """f16: a channel that only pages with a scale 2^22 below the others' hold.  Its weights P' there lie within f16's
    range, so the channel has the relative error of any other: the roundings of P' and of the output, 2^-11 each, what
    the fp32 steps add (2^-15 is ample: scores to 2, some 200 terms), and half of f16's least step, 2^-25."""
    announce(f"gqa_kv8 quiet pages {news}")
    n, page = 300, 64
    cache = filled(ops, 5, 1, 64, page, 3)
    table = [[4, 0, 2, 1, 3]]
    cache.v_scale.fill_(1.0)
    cache.k_scale.fill_(2.0 ** -9)
    cache.v_scale[2] = cache.v_scale[3] = 2.0 ** -22
    v = cache.v.view(torch.uint8)
    for p in (0, 1, 4):
        v[p, :, 0] = 0
    for p in (2, 3):
        v[p, :, 0] = 0x70 + (torch.arange(page, device="cuda") % 14).to(torch.uint8)
    q = randn((news[0], 2, 64), 5, F16, 0.2)
    exp, _, _ = oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale).attend(q, table, [n], prefix(news), False)
    more = {} if news == [1] else {"cu_q": i32(prefix(news)), "max_q": news[0]}
    got = ops.gqa_kv8(q.cuda(), cache, i32(table), i32([n]), causal=False, **more).cpu().double()[..., 0]
    exp = exp[..., 0]
    assert bool((exp > 2.0 ** -20).all())
    assert bool(((got - exp).abs() <= exp * (2 * 2.0 ** -11 + 2.0 ** -15) + 2.0 ** -25).all())


@pytest.mark.parametrize("news", [[1], [4], [9], [100]])
def test_attend_nan_and_inf(ops, news):
    """NaN codes of K and V reach the rows that see their token and no others; a query with an infinity gives what
    softmax gives (NaN for scores of +inf, and for a row whose scores are all -inf)."""
    announce(f"gqa_kv8 NaN and inf {news}")
    n, lens = news[0], [130]
    table = tables(lens, 16, 9, 1)
    for dtype, causal in ((BF16, True), (F16, True), (BF16, False)):
        cache = filled(ops, 9, 1, 64, 16, 2)
        put = [(cache.v, 129, 5), (cache.v, 127, 6), (cache.k, 128, 7)] + ([(cache.v, 70, 8)] if n == 100 else [])
        for code, t, c in put:
            p = table[0][t // 16]
            if code is cache.v:
                code.view(torch.uint8)[p, 0, c, t % 16] = 0x7F
            else:
                code.view(torch.uint8)[p, 0, t % 16, c] = 0xFF
        q = randn((n, 2, 64), 3, dtype, 0.05)
        check_attend(ops, cache, q, table, lens, news, causal)
    cache = filled(ops, 9, 1, 64, 16, 2)
    cache.k.view(torch.uint8)[..., 0] = 0x38  # one
    q = randn((n, 2, 64), 4, BF16, 0.05)
    q[0, 0, 0], q[n - 1, 1, 0] = float("-inf"), float("inf")
    check_attend(ops, cache, q, table, lens, news)


@pytest.mark.parametrize("scores", ["falling", "rising", "far"])
def test_attend_running_maximum(ops, scores):
    """Scores that fall, rise or lie hundreds apart from tile to tile: the sums follow the running maximum."""
    announce(f"gqa_kv8 running maximum {scores}")
    for news in ([1], [200]):
        lens = [400]
        cache = filled(ops, 7, 1, 64, 64, 8)
        table = tables(lens, 64, 7, 9)
        k = cache.k.view(torch.uint8)
        k.zero_()
        for t in range(400):
            step = {"falling": 400 - t, "rising": t, "far": 440 if t == 301 else t % 3}[scores]
            row = torch.tensor([float(step)]).to(torch.float8_e4m3fn).view(torch.uint8)
            k[table[0][t // 64], 0, t % 64, 0] = row.item()
        cache.k_scale.fill_(1.0)
        q = torch.zeros((news[0], 1, 64), dtype=BF16)
        q[:, :, 0] = 8
        check_attend(ops, cache, q, table, lens, news)


def test_attend_empty_rows_bad_numbers_and_rows_of_none(ops):
    """A sequence of no tokens, more rows than tokens, pages that are none, a sequence of no rows; rows before the
    first and behind the last sequence stay as they were."""
    announce("gqa_kv8 empty rows")
    cache = filled(ops, 8, 2, 64, 16, 1)
    table = [[-1, -1, -1], [0, 1, -1], [2, 8, 3], [-5, -1, 1 << 30], [4, 5, 6]]
    lens, news = [0, 20, 45, 40, 48], [3, 25, 7, 2, 0]
    cu = [2 + c for c in prefix(news)]
    oc = oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)
    for dtype, causal, more in itertools.product((BF16, F16), (True, False), ([], [90])):
        ns, ls = news + more, lens + [48] * len(more)
        tb = table + [[7, 6, 5]] * len(more)
        cu = [2 + c for c in prefix(ns)]
        q = randn((cu[-1] + 3, 4, 64), 2, dtype, 0.05)
        exp, weight, score = oc.attend(q, tb, ls, cu, causal)
        out = torch.full(q.shape, float("nan"), dtype=dtype, device="cuda")
        ops.gqa_kv8(q.cuda(), cache, i32(tb), i32(ls), i32(cu), max_q=max(ns), causal=causal, out=out)
        got = out.cpu().double()
        assert torch.equal(got.isnan(), exp.isnan())
        ok = ((got - exp).abs() <= bound(exp, weight, score, ls, 64, dtype, cache.v_scale)) | exp.isnan()
        assert bool(ok.all())
        assert bool((got[cu[0]:cu[1]] == 0).all())
    one = randn((5, 4, 64), 3, BF16)
    got = ops.gqa_kv8(one.cuda(), cache, i32(table), i32([0, -1, -2 ** 31, 40, 0]))
    assert bool((got == 0).all())


@pytest.mark.parametrize("news", [[1, 1, 1], [3, 9, 1], [30, 70, 65]])
def test_attend_hints_only_choose(ops, news):
    """max_q and max_kv too small, right and too large; lengths past the table's width count as its width."""
    announce(f"gqa_kv8 hints {news}")
    lens = [1500, 700, 65]
    cache = filled(ops, 40, 2, 64, 64, 1)
    table = tables(lens, 64, 40, 2)
    q = randn((sum(news), 8, 64), 3, BF16, 0.05)
    want = None
    for max_kv, max_q in itertools.product((1, 256, 1500, None), ((None,) if max(news) == 1 else (1, max(news), None))):
        more = {"max_kv": max_kv} if max(news) == 1 else {"max_kv": max_kv, "max_q": max_q}
        want = check_attend(ops, cache, q, table, lens, news, want=want, **more)
    full = [24 * 64, 700, 65]
    table[0] = table[0][:24]
    check_attend(ops, cache, q, table, full, news)
    out = ops.gqa_kv8(q.cuda(), cache, i32(table), i32([2 ** 31 - 1, 700, 65]), *(
        () if max(news) == 1 else (i32(prefix(news)), max(news))))
    same = ops.gqa_kv8(q.cuda(), cache, i32(table), i32(full), *(
        () if max(news) == 1 else (i32(prefix(news)), max(news))))
    assert torch.equal(out, same)


@pytest.mark.parametrize("causal", [True, False])
def test_attend_more_rows_than_hinted(ops, causal):
    """2300 rows of one sequence where max_q says 1: blocks of rows far from the last token, NaN codes here and there,
    which only the rows that see them may show."""
    announce(f"gqa_kv8 2300 rows, hint 1, causal={causal}")
    n, page = 2300, 64
    cache = filled(ops, 40, 1, 64, page, 5)
    table = tables([n + 7], page, 40, 6)
    for t in (60, 700, 2111, 2290) if causal else (700,):
        cache.v.view(torch.uint8)[table[0][t // page], 0, t % 64, t % page] = 0x7F
    q = randn((n, 1, 64), 7, BF16, 0.05)
    check_attend(ops, cache, q, table, [n + 7], [n], causal, max_q=1)


def test_far_pages(ops):
    """Codes past 2^32 bytes of each of the cache's tensors, written, copied and read."""
    announce("kv8 pages past 2^32 bytes")
    n_kv, d, page = 8, 128, 64
    pages = 2 ** 32 // (n_kv * d * page) + 40
    cache = ops.KV8Cache.empty(pages, n_kv, d, page)
    lens, news = [600, 100], [600, 100]
    table = tables(lens, page, 30, 1)
    far = [[p + pages - 30 if p >= 0 else p for p in row] for row in table]
    k, v = randn((700, n_kv, d), 1, BF16), randn((700, n_kv, d), 2, BF16)
    near = ops.KV8Cache.empty(30, n_kv, d, page)
    for c, t in ((cache, far), (near, table)):
        ops.kv8_append(k.cuda(), v.cuda(), c, i32(t), i32(lens), i32([0, 600, 700]), 600)
    for a, b in ((cache.k, near.k), (cache.v, near.v)):
        assert torch.equal(a[pages - 30:].view(torch.uint8), b.view(torch.uint8))
        assert not a[:30].view(torch.uint8).any()
    for m in (1, 200):
        q = randn((2 * m, 8, d), 3, BF16)
        more = () if m == 1 else (i32([0, m, 2 * m]), m)
        assert torch.equal(ops.gqa_kv8(q.cuda(), cache, i32(far), i32([600, 200]), *more),
                           ops.gqa_kv8(q.cuda(), near, i32(table), i32([600, 200]), *more))
    ops.kv8_copy_pages(cache, i32([pages - 1, pages - 30]), i32([5, 3]))
    assert torch.equal(cache.k[5].view(torch.uint8), near.k[29].view(torch.uint8))
    assert torch.equal(cache.v[3].view(torch.uint8), near.v[0].view(torch.uint8))


@pytest.mark.parametrize("news", [[1, 1], [3, 2], [70, 30]])
def test_graphs_and_streams(ops, news):
    """Append and attention captured, replayed on two streams, each with its own cache and workspace, between eager
    calls of the same kernels."""
    announce(f"kv8 graphs on two streams {news}")
    lens, cu = i32([900, 300]), i32(prefix(news))  # the graphs read them: they live as long
    table = i32(tables([900, 300], 64, 24, 1))
    more = {} if news == [1, 1] else {"cu_q": cu, "max_q": max(news)}
    sides = []
    for i in range(2):
        cache = filled(ops, 24, 2, 128, 64, i)
        kv = [randn((sum(news), 2, 128), 10 + 2 * i + j, BF16).cuda() for j in range(2)]
        q = randn((sum(news), 8, 128), 20 + i, BF16, 0.05).cuda()
        ws = torch.empty(max(16, ops.gqa_kv8_workspace_bytes(2, sum(news), max(news), 900, 8, 2, 128)), dtype=torch.uint8,
                         device="cuda")
        out = torch.empty_like(q)

        def step(cache=cache, kv=kv, q=q, ws=ws, out=out):
            ops.kv8_append(*kv, cache, table, lens, **more)
            ops.gqa_kv8(q, cache, table, lens, max_kv=900, out=out, workspace=ws, **more)

        step()
        torch.cuda.synchronize()
        want = out.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        sides.append((g, out, want, torch.cuda.Stream(), step))
    for _ in range(3):
        for g, out, want, stream, step in sides:
            out.fill_(float("nan"))
        torch.cuda.synchronize()
        for g, out, want, stream, step in sides:
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for g, out, want, stream, step in sides:
            assert torch.equal(out, want)
            step()
        torch.cuda.synchronize()
        for g, out, want, stream, step in sides:
            assert torch.equal(out, want)


def test_a_captured_step_follows_the_device(ops):
    """One captured step of decoding, replayed while lengths, table, tokens and queries change in place: as eager calls
    on a cache of their own, from a first token to lengths past the hint."""
    announce("kv8 captured step, other lengths at each replay")
    n_kv, d, page, most = 2, 128, 16, 60
    caches = [filled(ops, 2 * most, n_kv, d, page, 3) for _ in range(2)]
    table = i32(tables([most * page, most * page], page, 2 * most, 4))
    lens = i32([0, 1])
    k, v, q = (torch.empty((2, n, d), dtype=BF16, device="cuda") for n in (n_kv, n_kv, 8))
    out, x = torch.empty_like(q), [randn((2, 12, d), s, BF16, 0.3) for s in range(6)]
    ws = torch.empty(ops.gqa_kv8_workspace_bytes(2, 2, 1, 700, 8, n_kv, d), dtype=torch.uint8, device="cuda")
    assert ws.numel()

    def step():
        ops.kv8_append(k, v, caches[0], table, lens)
        ops.gqa_kv8(q, caches[0], table, lens, max_kv=700, out=out, workspace=ws)

    k.zero_(), v.zero_(), q.zero_()
    step()  # sequence 0 has no token yet, sequence 1 its first
    ops.kv8_append(k, v, caches[1], table, lens)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for i, n in enumerate(([1, 2], [2, 300], [17, 301], [700, 959], [701, 960], [5, 16])):
        lens.copy_(i32(n))
        if i == 3:
            table.copy_(table.flip(0))
        k.copy_(x[i][:, :2]), v.copy_(x[i][:, 2:4]), q.copy_(x[i][:, 4:])
        out.fill_(float("nan"))
        g.replay()
        ops.kv8_append(k, v, caches[1], table, lens)
        want = ops.gqa_kv8(q, caches[1], table, lens, max_kv=700)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for a, b in ((caches[0].k, caches[1].k), (caches[0].v, caches[1].v)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        assert torch.equal(caches[0].k_scale, caches[1].k_scale)


# ---- pages ----------------------------------------------------------------
@pytest.mark.parametrize("d,page,n_kv", [(64, 16, 1), (128, 64, 8), (64, 128, 3)])
def test_copy_pages(ops, d, page, n_kv):
    announce(f"kv8_copy_pages d{d} page{page} n_kv{n_kv}")
    cache = filled(ops, 20, n_kv, d, page, 1)
    was = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)]
    src, dst = [3, 3, 19, 7, 5, -1, 20, 8], [0, 1, 2, 18, 5, 9, 10, 77]
    ops.kv8_copy_pages(cache, i32(src), i32(dst))
    for a, b in zip(src, dst):
        if 0 <= a < 20 and 0 <= b < 20:
            for t in was:
                t[b] = t[a]
    for t, e in zip((cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale), was):
        assert torch.equal(t, e)
    ops.kv8_copy_pages(cache, i32([]), i32([]))


# ---- together -------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_layer_served_in_8_bits(ops, dtype):
    """Prompts through an int8 projection into the cache, attention and an int8 projection out; one sequence
    forked with its last page shared, both decoded on, one ended, the pool compacted: every step against the oracle."""
    announce(f"8-bit layer, prompts, fork, decode, compaction {dtype}")
    pool_of = import_submodule("kv_pages")
    n_q, n_kv, d, page, hidden = 8, 2, 64, 16, 256
    width = (n_q + 2 * n_kv) * d
    w_in, s_in = oint8.quantize_rows(randn((width, hidden), 1, BF16, hidden ** -0.5))
    w_out, s_out = oint8.quantize_rows(randn((hidden, n_q * d), 2, BF16, 0.05))
    gpu = [t.cuda() for t in (w_in, s_in, w_out, s_out)]
    pool = pool_of.KVPages(30, page)
    cache = ops.KV8Cache.empty(30, n_kv, d, page)
    mirror = oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)

    def copy(copies):
        if copies:
            ops.kv8_copy_pages(cache, *pool_of.copy_lists(copies))
            for a, b in copies:
                for t in (mirror.k, mirror.v, mirror.ks, mirror.vs):
                    t[b] = t[a]

    def step(seqs, news, seed):
        copy([c for s, n in zip(seqs, news) for c in pool.extend(s, n)])
        table, lens = pool.table(seqs)
        cu = prefix(news)
        x = randn((cu[-1], hidden), seed, dtype)
        qkv = ops.linear_int8(x.cuda(), gpu[0], gpu[1])
        q = qkv[:, :n_q * d].unflatten(1, (n_q, d))
        k, v = (qkv[:, (n_q + i * n_kv) * d:(n_q + (i + 1) * n_kv) * d].unflatten(1, (n_kv, d)) for i in range(2))
        args = (table.cuda(), lens.cuda(), i32(cu), max(news))
        ops.kv8_append(k, v, cache, *args)
        o = ops.gqa_kv8(q, cache, *args)
        y = ops.linear_int8(o.flatten(1), gpu[2], gpu[3])
        # each operator on what the one before it gave
        qe, se = oint8.quantize_rows(x)
        exact = oint8.product(qe, se, w_in, s_in)
        half = torch.finfo(dtype).eps / 2
        assert bool(((qkv.cpu().double() - exact).abs() <= exact.abs() * (half * 1.001 + 2.0 ** -22) + 2.0 ** -25).all())
        mirror.append(k, v, table.tolist(), lens.tolist(), cu)
        assert_cache(cache, mirror)
        exp, weight, score = mirror.attend(q, table.tolist(), lens.tolist(), cu)
        assert bool(((o.cpu().double() - exp).abs() <= bound(exp, weight, score, lens.tolist(), d, dtype, mirror.vs)).all())
        qe, se = oint8.quantize_rows(o.flatten(1))
        exact = oint8.product(qe, se, w_out, s_out)
        assert bool(((y.cpu().double() - exact).abs() <= exact.abs() * (half * 1.001 + 2.0 ** -22) + 2.0 ** -25).all())

    a, b = pool.new(), pool.new()
    step([a, b], [37, 90], 3)
    c = pool.fork(a)
    step([a, b, c], [1, 1, 1], 4)
    step([a, b, c], [1, 3, 2], 5)
    pool.free(b)
    copy(pool.compact())
    step([c, a], [20, 1], 6)
