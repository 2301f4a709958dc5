"""Log probabilities, entropy and top alternatives on the GPU, against the 64-bit oracle."""
from __future__ import annotations

import math

import pytest
import torch

from conftest import announce
from oracle import logprobs as oracle

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def logits_of(T, V, dtype, seed, scale=3.0):
    return (torch.randn((T, V), generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def tokens_of(T, V, m, seed):
    return torch.randint(0, V, (T, m), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)


def check(ops, x, tokens, top, dev=None, **more):
    """A logit's exponential is off by 2 steps of 2^-23, its exponent's rounding and log2(e)'s (2^-24 of the distance to
    the maximum); a sum of V logits in fp32 takes 8 additions in a chunk, one for each chunk of 4096 and some
    20 to join: together below 2^-24 (64 + V / 4096) of S.  The logarithm: 2 steps of its value, at most 30.  A
    log probability adds its own exponent's roundings; the entropy those of E, a sum of p |y| whose terms' exponents are off by
    2^-24 |y| each (the sum of p y^2)."""
    T, V = x.shape
    got = ops.token_logprobs(x.cuda() if dev is None else dev, None if tokens is None else tokens.cuda(), top, **more)
    given = [[]] * T if tokens is None else tokens.reshape(T, -1).tolist()
    lp, h, ids, best, spread = oracle.token_logprobs(x, given, top)
    unit = 2.0 ** -24
    most = 64 + V / 4096 + 60

    def near(a, b, tol):
        a = a.cpu().double().reshape(b.shape)
        assert torch.equal(a.isnan(), b.isnan())
        fine = b.isfinite()
        assert torch.equal(a[~fine & ~b.isnan()], b[~fine & ~b.isnan()])
        assert bool(((a - b).abs() <= tol)[fine].all()), float(((a - b).abs() / tol)[fine].max())

    if tokens is None:
        assert got[0] is None
    else:
        near(got[0], lp, unit * (most + 8 * lp.abs()))
    near(got[1], h, unit * (most * (1 + h + math.log(V)) + 4 * spread))
    assert got[2].dtype == torch.int32 and torch.equal(got[2].cpu(), ids)
    near(got[3], best, unit * (most + 8 * best.abs()))
    return got


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,V,top", [(1, 1, 1), (1, 5, 5), (3, 7, 2), (2, 64, 32), (5, 257, 20), (2, 2047, 1), (1, 4100, 0),
                                     (3, 32000, 5), (64, 9001, 7), (700, 1003, 3), (1, 200003, 20), (513, 16389, 32)])
def test_sizes(ops, dtype, T, V, top):
    """One logit to a large vocabulary, rows of one slice and of many, blocks' edges inside."""
    announce(f"token_logprobs T{T} V{V} top{top} {dtype}")
    x = logits_of(T, V, dtype, T + V)
    if T > 100:  # the oracle sorts few of them: the others repeat
        x = x[:24].repeat(-(-T // 24), 1)[:T].contiguous()
    check(ops, x, tokens_of(T, V, 3, 1), top)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_alignment(ops, dtype):
    """Rows apart by odd numbers, from every alignment, the outputs' neighbours untouched."""
    announce(f"token_logprobs alignment {dtype}")
    for off in range(9):
        big = logits_of(4, 4111, dtype, off, 2.0)
        big[:, :off] = 1000.0  # what lies beside the rows would win
        big[:, off + 4090:] = 1000.0
        x = big[:, off:off + 4090]
        check(ops, x.contiguous(), tokens_of(4, 4090, 1, off), 6, dev=big.cuda()[:, off:off + 4090])


@pytest.mark.parametrize("T,V", [(2, 33000), (2, 32999), (2, 30001), (600, 33000)])
def test_ties(ops, T, V):
    """Rows of one value, of few values, zeros of both signs: the lowest ids first, whichever wave or slice holds them."""
    announce(f"token_logprobs ties T{T} V{V}")
    x = torch.zeros((T, V), dtype=BF16)
    x[0] = -0.0
    x[0, 100::7] = 0.0
    x[1] = torch.randint(0, 3, (V,), generator=torch.Generator().manual_seed(1)).to(BF16)
    check(ops, x, tokens_of(T, V, 2, 2), 32)
    y = logits_of(2, V, BF16, 3, 0.5)
    y[:, [0, 8191, 8192, 16384, V - 5, V - 1]] = 9.0
    check(ops, y, tokens_of(2, V, 2, 2), 9)


@pytest.mark.parametrize("T", [8, 520])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_masked_and_odd_rows(ops, T, dtype):
    """-inf nearly everywhere, with fewer tokens left than alternatives; one left; none left; the type's lowest value in the masked
    places; a NaN; an infinity; the largest logits; whole lanes and slices of -inf."""
    announce(f"token_logprobs masks T{T} {dtype}")
    V = 20011
    x = logits_of(8, V, dtype, 5)
    keep = x[0, [17, 9000, 20010]].clone()
    x[0] = -math.inf
    x[0, [17, 9000, 20010]] = keep
    x[1] = -math.inf
    x[1, 20010] = 3.0
    x[2] = -math.inf
    x[3, 5000:] = torch.finfo(dtype).min if dtype == F16 else -1e30
    x[4, 19999] = math.nan
    x[5, 3] = math.inf
    x[6] *= 20000 / 13 if dtype == F16 else 1e6
    x[7, :16384] = -math.inf
    x = x.repeat(-(-T // 8), 1)[:T].contiguous()
    got = check(ops, x, torch.tensor([[17, 20010]] * T, dtype=torch.int32), 5)
    assert got[2][0, :3].tolist() != [-1] * 3 and got[2][2].tolist() == [-1] * 5


def test_tokens(ops):
    """One token a row, several, the same twice, none; numbers that are no token."""
    announce("token_logprobs tokens")
    x = logits_of(3, 1000, F32, 7)
    got = check(ops, x, torch.tensor([5, -1, 999], dtype=torch.int32), 0)
    assert got[0].shape == (3,)
    check(ops, x, torch.tensor([[1, 1, -1], [1000, 2 ** 31 - 1, -2 ** 31], [0, 999, 500]], dtype=torch.int32), 2)
    check(ops, x, None, 2)
    check(ops, x, torch.zeros((3, 0), dtype=torch.int32), 2)
    check(ops, x, tokens_of(3, 1000, 100, 1), 2)


def test_rows_far_apart(ops):
    """Offsets past 2^31 logits."""
    announce("token_logprobs rows far apart")
    stride = 1_200_000_007
    big = torch.empty(2 * stride + 5000, dtype=BF16, device="cuda").as_strided((3, 5000), (stride, 1))
    x = logits_of(3, 5000, BF16, 11)
    big.copy_(x)
    check(ops, x, tokens_of(3, 5000, 2, 1), 4, dev=big)


def test_sharp_rows(ops):
    """One token far ahead of the rest: an entropy near zero."""
    announce("token_logprobs sharp rows")
    for lead in (10.0, 25.0, 60.0, 500.0):
        x = logits_of(3, 30000, F32, 8, 1.0)
        x[:, 12345] = lead
        check(ops, x, torch.tensor([12345, 0, 1], dtype=torch.int32), 3)


def test_out_workspace_graph_and_streams(ops):
    """No allocation with out and workspace; a captured call replays with other logits; two calls on two streams, each with
    its own workspace; a larger workspace serves."""
    announce("token_logprobs graph")
    T, V, top = 6, 50001, 8
    need = ops.token_logprobs_workspace_bytes(T, V, top, BF16)
    assert need > 0
    x, tokens = logits_of(T, V, BF16, 9).cuda(), tokens_of(T, V, 2, 10).cuda()

    def buffers():
        return ((torch.empty((T, 2), device="cuda"), torch.empty(T, device="cuda"),
                 torch.empty((T, top), dtype=torch.int32, device="cuda"), torch.empty((T, top), device="cuda")),
                torch.empty(need + 64, dtype=torch.uint8, device="cuda"))

    (out, ws), (out2, ws2) = buffers(), buffers()
    want = ops.token_logprobs(x, tokens, top)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.token_logprobs(x, tokens, top, out=out2, workspace=ws2)
    assert ops.token_logprobs(x, tokens, top, out=out, workspace=ws) is not None
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b, c in zip(want, out, out2):
        assert torch.equal(a, b) and torch.equal(a, c)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.token_logprobs(x, tokens, top, out=out, workspace=ws)
    for r in range(3):
        x.copy_(logits_of(T, V, BF16, 20 + r))
        want = ops.token_logprobs(x, tokens, top)
        for t in out:
            t.fill_(-7)
        ws.fill_(0xFF)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, out):
            assert torch.equal(a, b)


def test_refusals(ops):
    x, t = torch.zeros((2, 100), dtype=BF16, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for args, more, error in [
            ((x.double(), t), {}, TypeError), ((x, t.long()), {}, TypeError), ((x, t[:1]), {}, ValueError),
            ((x, t, 33), {}, ValueError), ((x, t, -1), {}, ValueError), ((x[:, :4], t, 5), {}, ValueError),
            ((x.cpu(), t), {}, ValueError), ((x[0], t), {}, ValueError), ((x[:0], t[:0]), {}, ValueError),
            ((x[:, :0], t), {}, ValueError), ((x.t(), torch.zeros(100, dtype=torch.int32, device="cuda")), {}, ValueError),
            ((x, t, 1), {"out": ops.token_logprobs(x, t, 2)}, ValueError),
            ((x, None, 2), {"out": ops.token_logprobs(x, t, 2)}, ValueError)]:
        with pytest.raises(error):
            ops.token_logprobs(*args, **more)
    big = torch.zeros((2, 100000), dtype=BF16, device="cuda")
    with pytest.raises(RuntimeError, match="workspace"):
        ops.token_logprobs(big, t, 2, workspace=torch.empty(64, dtype=torch.uint8, device="cuda"))
