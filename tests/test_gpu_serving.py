"""A decoder's step as it is served: heads normed and turned, the 8-bit cache, windowed layers, a drafted tree verified by
the log probabilities of its tokens; every operator against the 64-bit oracle on what the one before it gave."""
from __future__ import annotations

import pytest
import torch

from conftest import announce, import_submodule
from oracle import int8 as oint8
from oracle import kv8 as okv8
from test_gpu_kv8 import BF16, F16, assert_cache, check_attend, i32, prefix, randn
from test_gpu_kv8_masks import compare, in_tree, in_window
from test_gpu_logprobs import check as check_logprobs
from test_gpu_rope import check as check_rope
from test_gpu_rope import table_of

pytestmark = pytest.mark.gpu

drafts = import_submodule("drafts")
kv_pages = import_submodule("kv_pages")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n_q,n_kv,d,page", [(8, 2, 64, 16), (8, 2, 128, 64)])
def test_a_drafted_tree_is_verified(ops, dtype, n_q, n_kv, d, page):
    """Two prompts through a windowed layer; drafted trees of both appended, attended over and scored; the accepted branches
    appended again over the drafted tokens, which the next token then follows as if they had been decoded."""
    announce(f"a drafted tree is verified n_q{n_q} d{d} page{page} {dtype}")
    hidden, vocab, window, sinks = 256, 1000, 24, 3
    width = (n_q + 2 * n_kv) * d
    w_in, s_in = oint8.quantize_rows(randn((width, hidden), 1, BF16, hidden ** -0.5))
    w_out, s_out = oint8.quantize_rows(randn((vocab, n_q * d), 2, BF16, 0.2))
    gpu = [t.cuda() for t in (w_in, s_in, w_out, s_out)]
    wq, wk, angles = randn((d,), 3, dtype), randn((d,), 4, dtype), table_of(300, d // 2)
    pool = kv_pages.KVPages(30, page)
    cache = ops.KV8Cache.empty(30, n_kv, d, page)
    mirror = okv8.Cache(cache.k, cache.v, cache.k_scale, cache.v_scale)

    def project(rows, positions, seed):
        """Views of one projection, queries and keys normed and turned in place."""
        x = randn((rows, hidden), seed, dtype)
        qkv = ops.linear_int8(x.cuda(), gpu[0], gpu[1])
        raw = qkv.cpu()
        q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split([n_q * d, n_kv * d, n_kv * d], dim=1))
        ops.qk_norm_rope(q, k, wq.cuda(), wk.cuda(), angles.cuda(), i32(positions), q_out=q, k_out=k)
        check_rope(q, raw[:, :n_q * d].unflatten(1, (n_q, d)), wq, angles, positions, 1e-6, False)
        check_rope(k, raw[:, n_q * d:(n_q + n_kv) * d].unflatten(1, (n_kv, d)), wk, angles, positions, 1e-6, False)
        assert torch.equal(qkv.cpu()[:, (n_q + n_kv) * d:], raw[:, (n_q + n_kv) * d:])
        return q, k, v

    def append(seqs, news, k, v):
        table, lens = pool.table(seqs)
        ops.kv8_append(k, v, cache, table.cuda(), lens.cuda(), i32(prefix(news)), max(news))
        mirror.append(k, v, table.tolist(), lens.tolist(), prefix(news))
        assert_cache(cache, mirror)
        return table, lens

    seqs, news = [pool.new(), pool.new()], [37, 90]
    pool.extend_all(zip(seqs, news))
    q, k, v = project(sum(news), [*range(37), *range(90)], 5)
    table, lens = append(seqs, news, k, v)
    out = ops.gqa_kv8_window(q, cache, table.cuda(), lens.cuda(), window, sinks, i32(prefix(news)), max(news))
    compare(cache, mirror, q, table.tolist(), lens.tolist(), news, in_window(lens.tolist(), news, window, sinks), [out])

    parents = [[-1, 0, 0, 1, 2, 2, 4], [-1, 0, 1, 1, 0, 4, 5, 5, 6, 6, 6, 2, 11]]
    base, news = news, [len(p) for p in parents]
    pool.extend_all(zip(seqs, news))
    positions = [b + t for b, p in zip(base, parents) for t in drafts.depths(p).tolist()]
    q, k, v = project(sum(news), positions, 6)
    table, lens = append(seqs, news, k, v)
    tree = torch.cat([drafts.masks(p) for p in parents]).cuda()
    out = ops.gqa_kv8_tree(q, cache, table.cuda(), lens.cuda(), tree, i32(prefix(news)), max(news))
    rows = [drafts.masks(p)[:, 0].tolist() for p in parents]
    compare(cache, mirror, q, table.tolist(), lens.tolist(), news, in_tree(lens.tolist(), news, rows), [out])
    logits = ops.linear_int8(out.flatten(1), gpu[2], gpu[3])
    children = [[i for i, p in enumerate(ps) if p == t] for ps in parents for t in range(len(ps))]
    drafted = torch.randint(0, vocab, (sum(news),), generator=torch.Generator().manual_seed(7))
    given = torch.full((sum(news), max(map(len, children))), -1, dtype=torch.int32)
    for r, c in enumerate(children):
        first = 0 if r < news[0] else news[0]
        given[r, :len(c)] = drafted[[first + j for j in c]].int()
    check_logprobs(ops, logits.cpu(), given, 5, dev=logits)

    kept = [[0, 2, 4, 6], [0, 4]]
    for s, b in zip(seqs, base):
        pool.truncate(s, b)
    news = [len(t) for t in kept]
    pool.extend_all(zip(seqs, news))
    at = torch.tensor(kept[0] + [7 + t for t in kept[1]]).cuda()
    assert [positions[t] for t in at.tolist()] == [37, 38, 39, 40, 90, 91]
    append(seqs, news, k[at], v[at])
    pool.extend_all((s, 1) for s in seqs)
    q, k, v = project(2, [41, 92], 8)
    table, lens = append(seqs, [1, 1], k, v)
    check_attend(ops, cache, q.cpu(), table.tolist(), lens.tolist(), [1, 1])
    out = ops.gqa_kv8_window(q, cache, table.cuda(), lens.cuda(), window, sinks)
    compare(cache, mirror, q, table.tolist(), lens.tolist(), [1, 1], in_window(lens.tolist(), [1, 1], window, sinks), [out])


def test_a_captured_step(ops):
    """Rotation, append, tree attention and log probabilities in one graph, every buffer the caller's: replays on other
    inputs, lengths and trees give what eager calls on another cache give."""
    announce("a captured step")
    n_q, n_kv, d, page, B, n, vocab = 8, 2, 128, 64, 3, 12, 5003
    T = B * n
    w, angles = randn((d,), 1, BF16).cuda(), table_of(3000, d).cuda()
    caches = [ops.KV8Cache.empty(160, n_kv, d, page) for _ in range(2)]
    first = [t.clone() for t in (caches[0].k, caches[0].v, caches[0].k_scale, caches[0].v_scale)]
    table = torch.arange(150, dtype=torch.int32).view(B, 50).cuda()
    lens, cu, positions = i32([2000, 1500, 40]), i32(prefix([n] * B)), i32([0] * T)
    tree, given = torch.ones(T, dtype=torch.int64).cuda(), i32([[1]] * T)
    qkv, logits = torch.empty((T, (n_q + 2 * n_kv) * d), dtype=BF16).cuda(), torch.empty((T, vocab), dtype=BF16).cuda()
    q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split([n_q * d, n_kv * d, n_kv * d], dim=1))
    qo, ko, o = torch.empty((T, n_q, d), dtype=BF16).cuda(), torch.empty((T, n_kv, d), dtype=BF16).cuda(), torch.empty(
        (T, n_q, d), dtype=BF16).cuda()
    lp = (torch.empty((T, 1)).cuda(), torch.empty(T).cuda(), i32([[0] * 4] * T), torch.empty((T, 4)).cuda())
    ws = torch.empty(ops.gqa_kv8_tree_workspace_bytes(B, T, n, 2000, n_q, n_kv, d), dtype=torch.uint8).cuda()
    ws2 = torch.empty(max(1, ops.token_logprobs_workspace_bytes(T, vocab, 4, BF16)), dtype=torch.uint8).cuda()
    assert ws.numel() > 0

    def step(cache, qo, ko, o, lp, ws, ws2):
        ops.qk_norm_rope(q, k, w, w, angles, positions, q_out=qo, k_out=ko)
        ops.kv8_append(ko, v, cache, table, lens, cu, n)
        o = ops.gqa_kv8_tree(qo, cache, table, lens, tree, cu, n, 2000, out=o, workspace=ws)
        return o, *ops.token_logprobs(logits, given, 4, out=lp, workspace=ws2)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[0], qo, ko, o, lp, ws, ws2)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(caches[0], qo, ko, o, lp, ws, ws2)
    for r in range(3):
        qkv.copy_(randn(qkv.shape, 10 + r, BF16))
        logits.copy_(randn(logits.shape, 20 + r, BF16, 3.0))
        lens.copy_(torch.tensor([2000 - 300 * r, 1500 + r, 40 - 10 * r]))
        base = [m - n for m in lens.tolist()]
        parents = [max(-1, (7 * i + r) % (i + 1) - 1) for i in range(n)]
        tree.copy_(drafts.masks(parents)[:, 0].repeat(B))
        positions.copy_(torch.cat([b + drafts.depths(parents) for b in base]))
        given.copy_(torch.randint(0, vocab, (T, 1), generator=torch.Generator().manual_seed(r)))
        for cache in caches:
            for t, was in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), first):
                t.view(torch.uint8).copy_(was.view(torch.uint8))
        want = step(caches[1], torch.empty_like(qo), torch.empty_like(ko), None, None, None, None)
        for t in (qo, ko, o, *lp):
            t.fill_(-3)
        ws.fill_(0xFF)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, (o, *lp)):
            assert torch.equal(a, b)
        assert torch.equal(caches[0].k.view(torch.uint8), caches[1].k.view(torch.uint8))
        assert torch.equal(caches[0].v_scale, caches[1].v_scale)
