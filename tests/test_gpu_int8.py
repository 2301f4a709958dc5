"""int8 quantiser, product and linear layer on the GPU against the 64-bit oracle."""
from __future__ import annotations

import pytest
import torch

from conftest import announce
from oracle import int8 as oracle

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def bound(exact: torch.Tensor, dtype) -> torch.Tensor:
    """How far the product may be off: its rounding to `dtype` (half a step relative to the value), after three
    fp32 roundings (the int32 sum's conversion, two scales); among the subnormals half of the type's step (f16 2^-24,
    bf16 2^-133) after two roundings of half fp32's (2^-149), the first of them times a scale below 1."""
    fp32 = 3 * 2.0 ** -24
    least = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134
    return exact.abs() * ((1 + fp32) * torch.finfo(dtype).eps / 2 + fp32 * 1.0001) + least + 2.0 ** -149


def rows(m, k, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((m, k), generator=g) * torch.exp(torch.randn(k, generator=g))).to(dtype)


def codes(m, k, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(-128, 128, (m, k), generator=g, dtype=torch.int32).to(torch.int8),
            torch.rand(m, generator=g) * 0.02 + 1e-4)


def same(q, s, x):
    qe, se = oracle.quantize_rows(x)
    assert torch.equal(q.cpu(), qe)
    assert torch.equal(s.cpu().view(torch.int32)[~se.isnan()], se.view(torch.int32)[~se.isnan()])
    assert torch.equal(s.cpu().isnan(), se.isnan())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 16), (3, 48), (5, 4096), (2, 4112), (7, 8208), (2, 16400), (300, 1040),
                                 (2047, 1024), (2048, 16), (2051, 496), (2050, 1024), (2049, 1040)])
def test_quantiser(ops, dtype, m, k):
    announce(f"quant_int8 {m}x{k} {dtype}")
    x = rows(m, k, dtype, m + k)
    same(*ops.quant_int8(x.cuda()), x)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantiser_ties_and_special_rows(ops, dtype):
    announce(f"quant_int8 special rows {dtype}")
    x = torch.zeros((10, 64), dtype=dtype)
    x[0] = torch.arange(64) - 31.5                       # scale 1 below: exact ties
    x[0, 0] = 127
    x[1] = (torch.arange(64) - 31.5) * 2.0 ** -8
    x[1, 5] = -127 * 2.0 ** -8
    x[3, 7] = float("inf")
    x[4, 63] = float("nan")
    x[5] = torch.finfo(dtype).max
    x[6] = torch.finfo(dtype).smallest_normal
    x[7, ::3] = torch.finfo(dtype).smallest_normal / 16  # subnormal
    x[8] = -0.0
    x[9] = torch.linspace(-1, 1, 64).to(dtype)
    same(*ops.quant_int8(x.cuda()), x)


def test_quantiser_strided_rows(ops):
    announce("quant_int8 strided rows")
    x = rows(9, 512, torch.bfloat16, 3).cuda()
    q, s = ops.quant_int8(x[:, 128:384])
    same(q, s, x[:, 128:384].contiguous().cpu())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [
    (1, 1, 16), (1, 17, 48), (1, 1024, 4096), (2, 24, 144), (15, 33, 112), (16, 100, 1040), (17, 256, 256), (31, 130, 400),
    (33, 64, 128), (48, 72, 2064), (64, 500, 640), (65, 65, 65 * 16), (100, 129, 272), (128, 128, 128), (200, 264, 528),
    (255, 257, 144), (700, 1000, 96), (513, 771, 1552), (1024, 1024, 1024)])
def test_product(ops, dtype, m, n, k):
    announce(f"gemm_int8 {m}x{n}x{k} {dtype}")
    a, sa = codes(m, k, m * 7 + k)
    w, sw = codes(n, k, n * 5 + k)
    exact = oracle.product(a, sa, w, sw)
    out = torch.full((m + 2, n), float("nan"), dtype=dtype, device="cuda")
    ops.gemm_int8(a.cuda(), sa.cuda(), w.cuda(), sw.cuda(), out=out[:m])
    assert bool(((out[:m].cpu().double() - exact).abs() <= bound(exact, dtype)).all())
    assert bool(out[m:].isnan().all())  # nothing behind the last row is touched


# Each launch variant once (mx_gemm_int8 chooses by the sizes), with ragged rows, columns and inner dimensions; the
# tiles with columns that store wide, in pairs and one by one.
VARIANTS = [
    (0, 129, 100, 16), (1, 34, 5242, 144), (2, 1025, 98, 144), (2, 129, 776, 400), (3, 292, 418, 144), (3, 324, 1381, 16),
    (4, 255, 2050, 144), (4, 1024, 1023, 2064), (4, 1024, 1016, 2064), (4, 2001, 258, 4112), (5, 1925, 811, 400),
    (5, 1925, 816, 400), (5, 1925, 810, 400), (6, 300, 6001, 400), (6, 300, 6008, 400), (7, 513, 6001, 144),
    (7, 513, 6008, 144), (7, 513, 6002, 144), (8, 4017, 4015, 144), (8, 4017, 4016, 144), (8, 4017, 4018, 144)]


@pytest.mark.parametrize("variant,m,n,k", VARIANTS)
def test_product_of_every_variant(ops, variant, m, n, k):
    announce(f"gemm_int8 variant {variant} {m}x{n}x{k}")
    dtype = DTYPES[(variant + n) % 2]
    a, sa = codes(m, k, m + k)
    w, sw = codes(n, k, n + k)
    exact = oracle.product(a, sa, w, sw)
    out = torch.full((m + 2, n), float("nan"), dtype=dtype, device="cuda")
    ops.gemm_int8(a.cuda(), sa.cuda(), w.cuda(), sw.cuda(), out=out[:m])
    assert bool(((out[:m].cpu().double() - exact).abs() <= bound(exact, dtype)).all())
    assert bool(out[m:].isnan().all())


def test_product_of_extremes(ops):
    """The longest sum of the largest products: 131056 * 128 * 128 lies 2^18 below 2^31."""
    announce("gemm_int8 largest sum")
    k = 131056
    a = torch.full((2, k), -128, dtype=torch.int8)
    a[1] = 127
    w = torch.full((20, k), -128, dtype=torch.int8)
    w[3:] = 127
    one = torch.ones
    exact = oracle.product(a, one(2), w, one(20))
    for rows_ in (2, 70):  # the kernel for few rows, and tiles
        out = ops.gemm_int8(a.repeat(rows_ // 2, 1).cuda(), one(rows_).cuda(), w.cuda(), one(20).cuda())
        assert bool(((out.cpu().double() - exact.repeat(rows_ // 2, 1)).abs() <= bound(exact, torch.bfloat16).repeat(
            rows_ // 2, 1)).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 40, 256), (37, 300, 1040), (130, 260, 512), (1, 17, 16), (1, 8200, 16384), (2, 33, 8192),
                                   (3, 1, 5456), (4, 70, 4096), (4, 8211, 2064), (3, 100, 144), (4, 64, 4112), (5, 64, 256),
                                   (1, 8200, 8192), (2, 8195, 4096), (2, 50, 4080), (3, 70, 1360), (8, 33, 512),
                                   (8, 8204, 496), (7, 90, 576), (9, 64, 256), (1, 64, 8208)])
def test_linear(ops, dtype, m, n, k):
    """Against the oracle's quantiser and product, with the caller's workspace, on rows that lie apart."""
    announce(f"linear_int8 {m}x{n}x{k} {dtype}")
    x = rows(m, 2 * k, dtype, 11)
    w, sw = oracle.quantize_rows(rows(n, k, dtype, 12))
    q, sx = oracle.quantize_rows(x[:, k:].contiguous())
    exact = oracle.product(q, sx, w, sw)
    ws = torch.empty(max(1, ops.linear_int8_workspace_bytes(m, k)), dtype=torch.uint8, device="cuda")
    y = ops.linear_int8(x.cuda()[:, k:], w.cuda(), sw.cuda(), workspace=ws)
    assert y.dtype == dtype
    assert bool(((y.cpu().double() - exact).abs() <= bound(exact, dtype)).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_special_rows(ops, dtype):
    """In either kernel (one for few rows, quantiser and product for more): rows of NaN or infinity poison themselves
    alone, zero rows give zeros, tiny and exactly tied values what the oracle gives."""
    announce(f"linear_int8 special rows {dtype}")
    x = rows(8, 256, dtype, 1)
    x[1, 9], x[3, 0] = float("nan"), float("-inf")
    x[2] = 0
    x[4] = torch.finfo(dtype).smallest_normal / 8
    x[5] = (torch.arange(256) - 127.5) * 0.5
    x[5, 0] = 127
    x[6] = torch.finfo(dtype).max
    w, sw = oracle.quantize_rows(rows(48, 256, torch.bfloat16, 2))
    q, sx = oracle.quantize_rows(x)
    exact = oracle.product(q, sx, w, sw)
    for a, b, more in ((0, 8, 0), (0, 4, 0), (4, 8, 0), (1, 2, 0), (2, 4, 0), (5, 7, 0), (0, 8, 1), (0, 8, 40)):
        xs = torch.cat([x[a:b], x[:1].expand(more, -1)])
        y = ops.linear_int8(xs.cuda(), w.cuda(), sw.cuda()).cpu().double()[:b - a]
        assert torch.equal(y.isnan(), exact[a:b].isnan())
        over = exact[a:b].abs() > torch.finfo(dtype).max
        ok = ((y - exact[a:b]).abs() <= bound(exact[a:b], dtype)) | y.isnan() | over
        assert bool(ok.all()) and bool((y[over].abs() >= torch.finfo(dtype).max).all())


def test_rows_of_any_stride(ops):
    """One row has no stride that could matter; strides past 2^31 elements are refused, not cut."""
    announce("int8 strides of one row and of far rows")
    x = rows(1, 512, torch.bfloat16, 9)
    w, sw = oracle.quantize_rows(rows(40, 512, torch.bfloat16, 8))
    w, sw = w.cuda(), sw.cuda()
    want = ops.linear_int8(x.cuda(), w, sw)
    for stride in (0, 3, 511, 513, 10 ** 10):
        y = x.cuda().as_strided((1, 512), (stride, 1))
        q, s = ops.quant_int8(y)
        same(q, s, x)
        assert torch.equal(ops.linear_int8(y, w, sw), want)
    big = torch.empty(2 ** 31 + 512, dtype=torch.bfloat16, device="cuda")
    for stride in (2 ** 31, 2 ** 30):
        far = big.as_strided((2, 512), (stride, 1))
        far.copy_(x.expand(2, -1))
        with pytest.raises((ValueError, RuntimeError)):
            ops.linear_int8(far, w, sw)
    q, s = ops.quant_int8(far)
    same(q, s, x.expand(2, -1))
    far = big.as_strided((2, 512), (2 ** 31, 1))
    with pytest.raises(ValueError):
        ops.quant_int8(far)
    del big, far


def test_quantiser_of_many_rows(ops):
    """More rows than one launch takes."""
    announce("quant_int8 of 2^23 + 3 rows")
    m = 2 ** 23 + 3
    x = torch.zeros((m, 16), dtype=torch.bfloat16, device="cuda")
    x[:, 5] = 2
    x[-2:, 3] = 4
    q, s = ops.quant_int8(x)
    assert bool((s[:-2] == torch.tensor(2.0) / 127).all()) and bool((s[-2:] == torch.tensor(4.0) / 127).all())
    assert bool((q[:, 5] == torch.tensor([127] * (m - 2) + [64, 64], dtype=torch.int8, device="cuda")).all())
    assert int(q.count_nonzero()) == m + 2


def test_streams_and_capture(ops):
    """Two graphs of two layers with workspaces of their own, replayed on two streams between eager calls."""
    announce("linear_int8 graphs on two streams")
    w, sw = oracle.quantize_rows(rows(320, 512, torch.bfloat16, 5))
    w, sw = w.cuda(), sw.cuda()
    xs = [rows(m, 512, torch.bfloat16, m).cuda() for m in (12, 90)]
    want = [ops.linear_int8(x, w, sw) for x in xs]
    outs = [torch.empty_like(y) for y in want]
    spaces = [torch.empty(max(1, ops.linear_int8_workspace_bytes(*x.shape)), dtype=torch.uint8, device="cuda") for x in xs]
    torch.cuda.synchronize()
    graphs = []
    for x, y, ws in zip(xs, outs, spaces):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.linear_int8(x, w, sw, out=y, workspace=ws)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for y in outs:
            y.fill_(float("nan"))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = ops.linear_int8(xs[0], w, sw)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0])
        for y, e in zip(outs, want):
            assert torch.equal(y, e)


@pytest.mark.parametrize("m", [1, 3, 20, 300])
def test_scales_far_from_one(ops, m):
    """Products whose sum times the token's scale leaves fp32's normal range, though the result does not: rows near
    bf16's largest value through every kernel, and scales from 2^-140 to 2^120 with the other one at the far end."""
    announce(f"int8 scales far from one, {m} rows")
    n, k = 40, 256
    x = torch.zeros((m, k))
    x[:, 3], x[:, 7] = 3e38, 1e38
    x[m // 2] = -x[m // 2]
    x = x.to(torch.bfloat16)
    w = torch.zeros((n, k))
    w[:, 3], w[:, 7] = torch.linspace(-0.7, 0.7, n), 0.3
    w, sw = oracle.quantize_rows(w.to(torch.bfloat16))
    q, sx = oracle.quantize_rows(x)
    exact = oracle.product(q, sx, w, sw)
    assert bool((exact.abs() < torch.finfo(torch.bfloat16).max).all())
    y = ops.linear_int8(x.cuda(), w.cuda(), sw.cuda())
    assert bool(((y.cpu().double() - exact).abs() <= bound(exact, torch.bfloat16)).all())
    a, _ = codes(m, k, 5)
    b, _ = codes(n, k, 6)
    for e, f in ((120, -120), (100, -30), (-140, 120), (-100, 110), (96, 10), (-97, -20), (0, -120)):
        g = torch.Generator().manual_seed(e + 200)
        sa, sb = ((1 + torch.rand(r, generator=g)) * 2.0 ** x for r, x in ((m, e), (n, f)))
        sa[::3] = 1.5 * 2.0 ** -f  # rows of ordinary size beside them
        exact = oracle.product(a, sa, b, sb)
        for dtype in DTYPES:
            out = ops.gemm_int8(a.cuda(), sa.cuda(), b.cuda(), sb.cuda(), dtype=dtype)
            over = exact.abs() > torch.finfo(dtype).max * (1 - 2.0 ** -10)
            ok = ((out.cpu().double() - exact).abs() <= bound(exact, dtype)) | over
            assert bool(ok.all()), f"scales 2^{e}, 2^{f}, {dtype}: {int((~ok).sum())} outputs"
