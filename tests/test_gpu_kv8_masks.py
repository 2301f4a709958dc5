"""Attention over the paged 8-bit cache with a sliding window and sinks, and for drafted trees, against the 64-bit oracle."""
from __future__ import annotations

import random

import pytest
import torch

from conftest import announce, import_submodule
from oracle import kv8 as oracle
from test_gpu_kv8 import BF16, F16, bound, filled, i32, prefix, randn, tables

pytestmark = pytest.mark.gpu

drafts = import_submodule("drafts")


def in_window(lens, news, window, sinks):
    def seen(b, i):
        t, p = torch.arange(max(lens[b], 0)), lens[b] - news[b] + i
        return (t <= p) & ((p - t < window) | (t < sinks))
    return seen


def in_tree(lens, news, masks):
    """masks: of each sequence, the rows' masks as whole numbers."""
    def seen(b, i):
        first = lens[b] - news[b]
        bits = masks[b][i]
        return torch.tensor([t < first or bits >> (t - first) & 1 for t in range(max(lens[b], 0))], dtype=torch.bool)
    return seen


def words_of(masks, words):
    rows = [[(r >> 64 * w) & (1 << 64) - 1 for w in range(words)] for seq in masks for r in seq]
    return torch.tensor([[x - (1 << 64) if x >> 63 else x for x in r] for r in rows], dtype=torch.int64).cuda()


def compare(cache, oc, q, table, lens, news, seen, outs, scale=None):
    cu = prefix(news)
    exp, weight, score = oc.attend(q, table, lens, cu, scale=scale, seen=seen)
    vs = cache.v_scale[cache.v_scale.isfinite()]
    may = bound(exp, weight, score, lens, cache.d, q.dtype, vs.clamp_max(2.0 ** 30))
    for out in outs:
        got = out.cpu().double()
        assert torch.equal(got.isnan(), exp.isnan()), f"NaN: {int(got.isnan().sum())}, {int(exp.isnan().sum())}"
        off = (got - exp).abs()
        ok = (off <= may) | exp.isnan()
        assert bool(ok.all()), f"{int((~ok).sum())} of {ok.numel()} outputs are off, by up to {float(off.nan_to_num().max())}"


def crowd(table, lens, news, empty, page):
    """With that many empty sequences behind them, which choose the kernel: so many more workgroups, and a table of 1000 tokens."""
    wide = [row + [-1] * (-(-1000 // page) - len(row)) for row in table]
    return wide + [[-1] * len(wide[0])] * empty, lens + [0] * empty, news + [0] * empty


def forms(cache, table, lens, news, q):
    """(table, lens, news, max_kv) for more than 16 rows a KV head: blocks of 16 and of 32 side by side and whole tiles of rows,
    as far as their number allows."""
    yield table, lens, news, None
    if max(news) * q.shape[1] > 16 * cache.k.shape[1]:
        for empty, max_kv in ((120, 1000), (600, 300)):
            yield *crowd(table, lens, news, empty, cache.k.shape[2]), max_kv


def run_window(ops, cache, q, table, lens, news, window, sinks, oc=None, scale=None, **hints):
    oc = oc or oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)
    outs = []
    for t, l, n, max_kv in forms(cache, table, lens, news, q):
        outs.append(torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda"))
        more = {} if n == [1] * len(n) else {"cu_q": i32(prefix(n)), "max_q": max(max(n), 1)}
        ops.gqa_kv8_window(q.cuda(), cache, i32(t), i32(l), window, sinks, scale=scale, out=outs[-1],
                           **{"max_kv": max_kv, **more, **hints})
    compare(cache, oc, q, table, lens, news, in_window(lens, news, window, sinks), outs, scale)


def run_tree(ops, cache, q, table, lens, news, masks, words=None, oc=None, scale=None, **hints):
    oc = oc or oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)
    words = words or max(1, -(-max(news) // 64))
    outs = []
    for t, l, n, max_kv in forms(cache, table, lens, news, q):
        outs.append(torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda"))
        ops.gqa_kv8_tree(q.cuda(), cache, i32(t), i32(l), words_of(masks, words), i32(prefix(n)),
                         **{"max_q": max(n), "max_kv": max_kv, **hints}, scale=scale, out=outs[-1])
    cut = [[r & (1 << 64 * words) - 1 for r in seq] for seq in masks]
    compare(cache, oc, q, table, lens, news, in_tree(lens, news, cut), outs, scale)


def random_masks(rng, news):
    """Branches, as drafts have them; every seventh row any bits at all."""
    out = []
    for n in news:
        parents = [rng.randint(max(-1, i - 6), i - 1) for i in range(n)]
        rows = [sum((x % (1 << 64)) << 64 * w for w, x in enumerate(r)) for r in drafts.masks(parents).tolist()] if n else []
        out.append([rng.getrandbits(n) if i % 7 == 6 else r for i, r in enumerate(rows)])
    return out


SHAPES = [  # d, page, n_kv, group
    (64, 16, 2, 1), (128, 16, 1, 4), (64, 32, 1, 7), (128, 64, 2, 4), (64, 128, 2, 4), (128, 128, 1, 16), (128, 32, 2, 2)]


# ---- window ---------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,page,n_kv,group", SHAPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (17, 4), (64, 64), (100, 0), (130, 70), (1000, 3), (5000, 5000)])
def test_window_single_tokens(ops, dtype, d, page, n_kv, group, window, sinks):
    """Sequences from nothing to several times the window, pages that the window begins and ends inside."""
    announce(f"window single d{d} page{page} n_kv{n_kv} group{group} w{window} s{sinks} {dtype}")
    lens = [0, 1, 2, 15, 64, 65, 130, 257, 700]
    cache = filled(ops, sum(-(-n // page) for n in lens) + 2, n_kv, d, page, 1)
    table = tables(lens, page, cache.pages, 2)
    q = randn((len(lens), n_kv * group, d), 3, dtype)
    run_window(ops, cache, q, table, lens, [1] * len(lens), window, sinks, scale=0.02)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,page,n_kv,group", SHAPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (20, 4), (64, 0), (150, 70), (400, 1)])
def test_window_prompts(ops, dtype, d, page, n_kv, group, window, sinks):
    """Chunks of a few rows and of several tiles of rows, whole prompts, a sequence without rows."""
    announce(f"window prompts d{d} page{page} n_kv{n_kv} group{group} w{window} s{sinks} {dtype}")
    lens = [333, 40, 500, 100, 7]
    news = [max(1, 300 // group), 40, 5, 0, 7]
    cache = filled(ops, sum(-(-n // page) for n in lens) + 2, n_kv, d, page, 4)
    table = tables(lens, page, cache.pages, 5)
    q = randn((sum(news), n_kv * group, d), 6, dtype)
    run_window(ops, cache, q, table, lens, news, window, sinks, scale=0.02)


@pytest.mark.parametrize("max_q", [1, 5, 8, 9])
@pytest.mark.parametrize("d,page", [(128, 64), (64, 16), (128, 32)])
def test_window_split_keys(ops, max_q, d, page):
    """Long windows over few sequences: the keys are split, in the rows kernel's two forms and the tile kernel's; hints that are too
    small and too large."""
    announce(f"window split max_q{max_q} d{d} page{page}")
    lens, news = [9000, 6000, 100], [max_q, max(1, max_q - 1), max_q]
    cache = filled(ops, sum(-(-n // page) for n in lens) + 2, 1, d, page, 7)
    table = tables(lens, page, cache.pages, 8)
    q = randn((sum(news), 4, d), 9, BF16)
    assert ops.gqa_kv8_window_workspace_bytes(3, sum(news), max_q, 9000, 4, 1, d, 4000, 130) > 0
    oc = oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)
    for window, sinks in ((4000, 130), (8990, 2), (1500, 3000)):
        run_window(ops, cache, q, table, lens, news, window, sinks, oc, 0.02)
    run_window(ops, cache, q, table, lens, news, 4000, 130, oc, 0.02, max_kv=300)
    run_window(ops, cache, q, table, lens, news, 4000, 130, oc, 0.02, max_kv=10 ** 6)
    if max_q > 1:
        run_window(ops, cache, q, table, lens, news, 4000, 130, oc, 0.02, max_q=1)
        run_window(ops, cache, q, table, lens, news, 4000, 130, oc, 0.02, max_q=300)


@pytest.mark.parametrize("d,page", [(128, 64), (64, 16), (128, 32)])
def test_split_keys_of_tiles(ops, d, page):
    """Long contexts of 256 rows a KV head among sequences that are empty: the keys are split in the tile kernel."""
    announce(f"window and tree split tiles d{d} page{page}")
    lens, news, empty = [5000, 3001, 90], [64, 33, 1], 137
    cache = filled(ops, sum(-(-n // page) for n in lens) + 2, 1, d, page, 60)
    table = tables(lens, page, cache.pages, 61)
    q = randn((sum(news), 4, d), 62, BF16)
    oc = oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)
    t, l, n = crowd(table, lens, news, empty, page)
    t, l, cu = i32(t), i32(l), i32(prefix(n))
    assert ops.gqa_kv8_window_workspace_bytes(140, 98, 64, 5000, 4, 1, d, 2500, 100) > 0
    assert ops.gqa_kv8_tree_workspace_bytes(140, 98, 64, 5000, 4, 1, d) > 0
    for window, sinks in ((2500, 100), (4000, 0)):
        out = torch.full(q.shape, float("nan"), dtype=BF16, device="cuda")
        ops.gqa_kv8_window(q.cuda(), cache, t, l, window, sinks, cu, 64, 5000, 0.02, out)
        compare(cache, oc, q, table, lens, news, in_window(lens, news, window, sinks), [out], 0.02)
    masks = random_masks(random.Random(9), news)
    out = torch.full(q.shape, float("nan"), dtype=BF16, device="cuda")
    ops.gqa_kv8_tree(q.cuda(), cache, t, l, words_of(masks, 1), cu, 64, 5000, 0.02, out)
    compare(cache, oc, q, table, lens, news, in_tree(lens, news, masks), [out], 0.02)


@pytest.mark.parametrize("group,n", [(1, 1), (4, 3), (4, 70), (1, 200)])
@pytest.mark.parametrize("page", [16, 64])
def test_window_pages_out_of_view(ops, group, n, page):
    """Pages that no row sees given back: no page at all, or another's, whose scales and codes are anything; NaN codes on
    the tokens beside the window and between a window's rows, which only the rows that see them get."""
    announce(f"window pages out of view group{group} n{n} page{page}")
    d, window, sinks = 64, 150, 20
    lens, news = [700, 640], [n, n]
    for junk in (-1, 2 ** 30, "page"):
        cache = filled(ops, 100, 1, d, page, 10)
        table = tables(lens, page, 98, 11)
        bad = 99
        cache.k_scale[bad], cache.v_scale[bad] = float("nan"), 0.0
        cache.k.view(torch.uint8)[bad] = 0x7F
        cache.v.view(torch.uint8)[bad] = 0xFF
        for b in range(2):
            from_a = lens[b] - n - window + 1
            for j in range(-(-lens[b] // page)):
                if j * page >= sinks and (j + 1) * page <= from_a:
                    table[b][j] = bad if junk == "page" else junk
        places = [lens[0] - window - 3, lens[0] - window - n // 2, lens[0] - 1 - n // 3, sinks, sinks - 1]
        for t in places:
            p = table[0][t // page]
            if 0 <= p < 98:
                cache.v.view(torch.uint8)[p, 0, t % d, t % page] = 0x7F
                cache.k.view(torch.uint8)[p, 0, t % page, 5] = 0xFF if t == lens[0] - 1 - n // 3 else 0x30
        q = randn((2 * n, group, d), 12, BF16)
        run_window(ops, cache, q, table, lens, news, window, sinks, scale=0.02)


def test_window_as_plain_attention(ops):
    """A window past every sequence: bit for bit what gqa_kv8 gives where both take one kernel and the keys are not split."""
    announce("window as plain")
    for news, group in (([1, 1, 1], 4), ([3, 8, 1], 2), ([60, 100, 5], 4)):
        lens, page = [120, 300, 77], 16
        cache = filled(ops, 40, 2, 64, page, 13)
        table = tables(lens, page, 40, 14)
        q = randn((sum(news), 2 * group, 64), 15, BF16).cuda()
        if max(news) * group > 16:
            table, lens, news = crowd(table, lens, news, 600, page)
        args = (i32(prefix(news)), max(news), 300)
        want = ops.gqa_kv8(q, cache, i32(table), i32(lens), *args)
        got = ops.gqa_kv8_window(q, cache, i32(table), i32(lens), 2 ** 31 - 1, 0, *args)
        assert torch.equal(got, want)


def test_window_bad_numbers(ops):
    """Lengths past the table and below zero, fewer tokens than rows, a negative scale, rows of no sequence, views of a
    fused projection."""
    announce("window bad numbers")
    page, d = 16, 64
    cache = filled(ops, 9, 1, d, page, 16)
    table = [[0, 1, 2], [3, -9, 4], [5, 6, 7]]
    lens, news = [48, 45, 3], [2, 40, 6]
    cu = [1 + c for c in prefix(news)]
    qkv = randn((cu[-1] + 2, 6 * d), 17, BF16)
    q = qkv[:, :4 * d].unflatten(1, (4, d))
    oc = oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)
    exp, weight, score = oc.attend(q, table, lens, cu, scale=-0.05, seen=in_window(lens, news, 9, 2))
    out = torch.full(q.shape, 7.0, dtype=BF16, device="cuda")
    ops.gqa_kv8_window(qkv.cuda()[:, :4 * d].unflatten(1, (4, d)), cache, i32(table), i32([2 ** 31 - 1, 45, 3]), 9, 2, i32(cu),
                       40, scale=-0.05, out=out)
    got = out.cpu().double()
    assert bool((got[0] == 7).all()) and bool((got[-2:] == 7).all())
    rows = slice(1, cu[-1])
    assert bool(((got - exp).abs()[rows] <= bound(exp, weight, score, lens, d, BF16, cache.v_scale)[rows]).all())
    out.fill_(7.0)
    ops.gqa_kv8_window(q[:3].contiguous().cuda(), cache, i32(table), i32([-5, -2 ** 31, 0]), 9, 2, out=out[:3])
    assert bool((out[:3] == 0).all())


# ---- tree -----------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,page,n_kv,group", SHAPES)
@pytest.mark.parametrize("most", [1, 4, 13, 64, 100])
def test_tree(ops, dtype, d, page, n_kv, group, most):
    """Trees of one token to more than a word of their masks, behind nothing, a few and many tokens."""
    announce(f"tree d{d} page{page} n_kv{n_kv} group{group} most{most} {dtype}")
    if group * n_kv * most > 900:
        most = 900 // (group * n_kv)
    rng = random.Random(most)
    news = [most, max(1, most // 2), max(1, most - 1), 0, min(most, 3)]
    lens = [most, most // 2 + 301, most + 62, 30, 128 + min(most, 3)]
    cache = filled(ops, sum(-(-n // page) for n in lens) + 2, n_kv, d, page, 20)
    table = tables(lens, page, cache.pages, 21)
    q = randn((sum(news), n_kv * group, d), 22, dtype)
    run_tree(ops, cache, q, table, lens, news, random_masks(rng, news), scale=0.02)


@pytest.mark.parametrize("group,most", [(4, 4), (4, 8), (4, 20), (1, 33)])
@pytest.mark.parametrize("d,page", [(128, 64), (64, 16)])
def test_tree_split_keys(ops, group, most, d, page):
    """Long contexts: the keys are split in every kernel form; hints that are too small and too large."""
    announce(f"tree split group{group} most{most} d{d} page{page}")
    rng = random.Random(3)
    news, lens = [most, most - 1, 1], [5000, 3001, 90]
    cache = filled(ops, sum(-(-n // page) for n in lens) + 2, 1, d, page, 23)
    table = tables(lens, page, cache.pages, 24)
    q = randn((sum(news), group, d), 25, BF16)
    masks = random_masks(rng, news)
    oc = oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)
    assert ops.gqa_kv8_tree_workspace_bytes(3, sum(news), most, 5000, group, 1, d) > 0
    for hints in ({}, {"max_kv": 100}, {"max_q": 1}, {"max_q": 200, "max_kv": 10 ** 6}):
        run_tree(ops, cache, q, table, lens, news, masks, 2, oc, 0.02, **hints)


@pytest.mark.parametrize("group,n", [(2, 5), (4, 60), (1, 300)])
def test_tree_masks(ops, group, n):
    """Masks of nothing (with and without tokens before them), of everything, of a row's later tokens, of bits past the drafted
    tokens; fewer words than drafted tokens; more words than they need; NaN codes among the drafted tokens."""
    announce(f"tree masks group{group} n{n}")
    d, page = 64, 16
    lens, news = [n, n + 77, n + 130], [n, n, n]
    rng = random.Random(4)
    masks = [[rng.choice([0, (1 << n) - 1, 1 << n - 1, 1 << i, -1 % (1 << 1024), rng.getrandbits(n)]) for i in range(n)]
             for _ in news]
    cache = filled(ops, sum(-(-m // page) for m in lens) + 2, 1, d, page, 26)
    table = tables(lens, page, cache.pages, 27)
    q = randn((sum(news), group, d), 28, BF16)
    for words in sorted({1, -(-n // 64), 16}):
        run_tree(ops, cache, q, table, lens, news, masks, words, scale=0.02)
    for b in range(3):
        for j in (0, n // 2, n - 1):
            t = lens[b] - n + j
            cache.v.view(torch.uint8)[table[b][t // page], 0, (7 * j) % d, t % page] = 0x7F
            if j == n // 2:
                cache.k.view(torch.uint8)[table[b][t // page], 0, t % page, 3] = 0xFF
    run_tree(ops, cache, q, table, lens, news, masks, 16, scale=0.02)


def test_tree_of_one_branch(ops):
    """A chain is a causal mask: bit for bit what gqa_kv8 gives where both take one kernel."""
    announce("tree of one branch")
    for n, group in ((3, 4), (8, 4), (50, 8)):
        lens, news, page = [120, 300, n], [n, n, n], 64
        cache = filled(ops, 20, 2, 128, page, 29)
        table = tables(lens, page, 20, 30)
        q = randn((3 * n, 2 * group, 128), 31, BF16).cuda()
        tree = drafts.masks(list(range(-1, n - 1))).repeat(3, 1).cuda()
        if n * group > 16:
            table, lens, news = crowd(table, lens, news, 600, page)
        args = (i32(prefix(news)), n, 300)
        want = ops.gqa_kv8(q, cache, i32(table), i32(lens), *args)
        assert torch.equal(ops.gqa_kv8_tree(q, cache, i32(table), i32(lens), tree, *args), want)
        assert torch.equal(ops.gqa_kv8_tree(q, cache, i32(table), i32(lens), tree[:, 0].contiguous(), *args), want)


def test_tree_bad_numbers(ops):
    """Fewer tokens than drafted rows, pages that are none, a negative scale, rows of no sequence; one row a sequence
    without cu_q."""
    announce("tree bad numbers")
    page, d, n = 16, 64, 20
    cache = filled(ops, 9, 1, d, page, 32)
    table, lens, news = [[0, 1, 2], [3, -9, 4], [5, 6, 7]], [40, 45, 6], [n, n, n]
    masks = random_masks(random.Random(5), news)
    q = randn((3 * n, 4, d), 33, F16)
    run_tree(ops, cache, q, table, lens, news, masks, scale=-0.05)
    q1 = randn((3, 4, d), 34, F16)
    oc = oracle.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)
    exp, weight, score = oc.attend(q1, table, lens, [0, 1, 2, 3], seen=in_tree(lens, [1] * 3, [[1], [0], [1]]))
    got = ops.gqa_kv8_tree(q1.cuda(), cache, i32(table), i32(lens), torch.tensor([1, 0, 1]).cuda()).cpu().double()
    assert bool(((got - exp).abs() <= bound(exp, weight, score, lens, d, F16, cache.v_scale)).all())


# ---- both -----------------------------------------------------------------
def test_masks_graph_and_workspace(ops):
    """Captured calls replayed with other lengths and masks, each graph with its own workspace; two streams; a workspace that
    is too small."""
    announce("window and tree graphs")
    page, d, n = 64, 128, 6
    lens, news = [3000, 2500], [n, n]
    cache = filled(ops, 100, 1, d, page, 40)
    table = i32(tables(lens, page, 100, 41))
    q = randn((2 * n, 4, d), 42, BF16).cuda()
    kv_lens, cu = i32(lens), i32(prefix(news))
    tree = words_of(random_masks(random.Random(6), news), 1)
    need_w = ops.gqa_kv8_window_workspace_bytes(2, 2 * n, n, 3000, 4, 1, d, 2000, 5)
    need_t = ops.gqa_kv8_tree_workspace_bytes(2, 2 * n, n, 3000, 4, 1, d)
    assert need_w > 0 and need_t > 0
    ws_w, ws_t = (torch.empty(m, dtype=torch.uint8, device="cuda") for m in (need_w, need_t))
    out_w, out_t = torch.empty_like(q), torch.empty_like(q)

    def window(**more):
        return ops.gqa_kv8_window(q, cache, table, kv_lens, 2000, 5, cu, n, 3000, **more)

    def drafted(**more):
        return ops.gqa_kv8_tree(q, cache, table, kv_lens, tree, cu, n, 3000, **more)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        window(out=out_w, workspace=ws_w)
    drafted(out=out_t, workspace=ws_t)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out_w, window()) and torch.equal(out_t, drafted())
    graphs = []
    for f, out, ws in ((window, out_w, ws_w), (drafted, out_t, ws_t)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            f(out=out, workspace=ws)
        graphs.append(g)
    for r in range(3):
        kv_lens.copy_(torch.tensor([3000 - 700 * r, 100 + r]))
        tree.copy_(words_of(random_masks(random.Random(7 + r), news), 1))
        want = window(), drafted()
        for t in (out_w, out_t):
            t.fill_(float("nan"))
        for t in (ws_w, ws_t):
            t.fill_(0xFF)
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out_w, want[0]) and torch.equal(out_t, want[1])
    with pytest.raises(RuntimeError, match="workspace"):
        window(workspace=ws_w[:-1].clone())
    with pytest.raises(RuntimeError, match="workspace"):
        drafted(workspace=ws_t[:-1].clone())


def test_masks_refusals(ops):
    cache = filled(ops, 4, 2, 64, 16, 50)
    q, table, lens = torch.zeros((2, 4, 64), dtype=BF16, device="cuda"), i32([[0], [1]]), i32([3, 4])
    tree = torch.ones((2, 1), dtype=torch.int64, device="cuda")
    ops.gqa_kv8_window(q, cache, table, lens, 1)
    ops.gqa_kv8_tree(q, cache, table, lens, tree)
    for window, sinks in ((0, 0), (-1, 0), (1, -1), (2 ** 31, 0), (1, 2 ** 31)):
        with pytest.raises(ValueError):
            ops.gqa_kv8_window(q, cache, table, lens, window, sinks)
    for bad, error in ((tree.int(), TypeError), (tree[:1], ValueError), (torch.ones((2, 17), dtype=torch.int64, device="cuda"), ValueError),
                       (tree.cpu(), ValueError), (tree[None], ValueError),
                       (torch.ones((2, 4), dtype=torch.int64, device="cuda")[:, ::2], ValueError)):
        with pytest.raises(error):
            ops.gqa_kv8_tree(q, cache, table, lens, bad)
    for args, more, error in (((q[:, :3], cache, table, lens), {}, ValueError), ((q[..., :32], cache, table, lens), {}, ValueError),
                              ((q.float(), cache, table, lens), {}, TypeError), ((q[:1], cache, table, lens), {}, ValueError),
                              ((q, cache, table.long(), lens), {}, TypeError), ((q, cache, table, lens[:1]), {}, ValueError),
                              ((q, None, table, lens), {}, TypeError), ((q, cache, table, lens), {"max_kv": 0}, ValueError),
                              ((q, cache, table, lens), {"max_q": 2}, ValueError),
                              ((q, cache, table, lens), {"out": torch.empty_like(q).half()}, TypeError)):
        with pytest.raises(error):
            ops.gqa_kv8_window(*args, 5, **more)
        with pytest.raises(error):
            ops.gqa_kv8_tree(*args, torch.ones(args[0].shape[0], dtype=torch.int64, device="cuda"), **more)
