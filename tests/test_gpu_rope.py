"""Norm and rotation of query and key heads on the GPU, against the 64-bit oracle."""
from __future__ import annotations

import pytest
import torch

from conftest import announce
from oracle import rope as oracle

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def randn(shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def table_of(rows, rot, seed=0):
    angle = torch.rand((rows, rot // 2), generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * 6.3
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def bound(out, weight, d, dtype):
    """How far an output may be off: the fp32 sum of d squares (8 in a lane, up to 5 joins of lanes: 13 roundings,
    halved by the root), its quotient, eps, the root (2 steps of 2^-23), three products, the rotation's product and
    FMA: below 20 steps of 2^-24 of |a cos| + |b sin|; then the output's own rounding (half a step), in f16 up to
    2^-25 below its normal numbers, 2^-126 in bf16."""
    half = torch.finfo(dtype).eps / 2
    off = 20 * 2.0 ** -24 * weight
    return off + (out.abs() + off) * half + (2.0 ** -25 if dtype == F16 else 2.0 ** -126)


def check(got, x, w, table, positions, eps, neighbours):
    exp, weight = oracle.norm_rope(x, w, table, positions, eps, neighbours)
    got = got.cpu().double()
    there = torch.tensor([0 <= p < table.shape[0] for p in positions])
    off = (got - exp).abs()[there]
    ok = off <= bound(exp, weight, x.shape[2], x.dtype)[there]
    assert bool(ok.all()), f"{int((~ok).sum())} of {ok.numel()} are off, by up to {float(off.max())}"
    return there


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("T,n_q,n_kv,d,rot", [
    (1, 1, 1, 16, 16), (1, 32, 8, 128, 128), (3, 7, 3, 64, 32), (5, 5, 1, 80, 48), (2, 3, 2, 256, 256), (9, 16, 16, 48, 16),
    (1000, 4, 1, 128, 64), (17, 33, 9, 96, 96), (4, 9, 5, 208, 144), (6000, 2, 1, 64, 64)])
def test_norm_rope(ops, dtype, neighbours, T, n_q, n_kv, d, rot):
    """One token to more than the launch has waves for, heads that fill no wave, head dims between the lanes' powers of two,
    rotations of a part; q and k as views of a fused projection."""
    announce(f"qk_norm_rope T{T} n_q{n_q} n_kv{n_kv} d{d} rot{rot} {neighbours} {dtype}")
    qkv = randn((T, (n_q + 2 * n_kv) * d), 1, dtype, 3.0)
    q, k = qkv[:, :n_q * d].unflatten(1, (n_q, d)), qkv[:, n_q * d:(n_q + n_kv) * d].unflatten(1, (n_kv, d))
    wq, wk = randn((d,), 2, dtype), randn((d,), 3, dtype)
    table = table_of(50, rot)
    positions = torch.randint(0, 50, (T,), generator=torch.Generator().manual_seed(4)).tolist()
    dev = qkv.cuda()
    qd, kd = dev[:, :n_q * d].unflatten(1, (n_q, d)), dev[:, n_q * d:(n_q + n_kv) * d].unflatten(1, (n_kv, d))
    qo, ko = ops.qk_norm_rope(qd, kd, wq.cuda(), wk.cuda(), table.cuda(), i32(positions), eps=1e-5, neighbours=neighbours)
    assert torch.equal(dev.cpu(), qkv)
    check(qo, q, wq, table, positions, 1e-5, neighbours)
    check(ko, k, wk, table, positions, 1e-5, neighbours)


def test_in_place_and_padding(ops):
    """In place in a fused projection, whose values' part stays as it is; tokens whose position is no row are left."""
    announce("qk_norm_rope in place")
    T, n_q, n_kv, d = 37, 6, 2, 64
    qkv = randn((T, (n_q + 2 * n_kv) * d), 5, BF16)
    w, table = randn((d,), 6, BF16), table_of(9, 64)
    positions = [(t * 5) % 14 - 3 for t in range(T)]
    positions[7], positions[8] = 2 ** 31 - 1, -2 ** 31
    dev = qkv.cuda()
    q, k = dev[:, :n_q * d].unflatten(1, (n_q, d)), dev[:, n_q * d:(n_q + n_kv) * d].unflatten(1, (n_kv, d))
    qo, ko = ops.qk_norm_rope(q, k, w.cuda(), w.cuda(), table.cuda(), i32(positions), q_out=q, k_out=k)
    assert qo is q and ko is k
    there = check(q, qkv[:, :n_q * d].unflatten(1, (n_q, d)), w, table, positions, 1e-6, False)
    check(k, qkv[:, n_q * d:(n_q + n_kv) * d].unflatten(1, (n_kv, d)), w, table, positions, 1e-6, False)
    got = dev.cpu()
    assert torch.equal(got[:, (n_q + n_kv) * d:], qkv[:, (n_q + n_kv) * d:]) and torch.equal(got[~there], qkv[~there])


def test_special_values(ops):
    """Zeros, the smallest and largest squares that fp32 holds, an infinity, a NaN: each head for itself."""
    announce("qk_norm_rope special values")
    d = 32
    x = torch.zeros((1, 6, d), dtype=BF16)
    x[0, 1] = 2.0 ** -70
    x[0, 2] = 2.0 ** 61
    x[0, 3, 5] = float("inf")
    x[0, 4, 6] = float("nan")
    x[0, 5] = 1.0
    w, table = torch.ones(d, dtype=BF16), table_of(1, 16)
    q, _ = ops.qk_norm_rope(x.cuda(), x.cuda(), w.cuda(), w.cuda(), table.cuda(), i32([0]), eps=0.0)
    q = q.cpu()
    assert bool(q[0, 0].isnan().all())  # 0 / 0
    q, _ = ops.qk_norm_rope(x.cuda(), x.cuda(), w.cuda(), w.cuda(), table.cuda(), i32([0]))
    q = q.cpu()
    assert bool((q[0, 0] == 0).all()) and bool(q[0, 4].isnan().all()) and bool(q[0, 3, 5].isnan())
    exp, weight = oracle.norm_rope(x[:, [1, 2, 5]], w, table, [0], 1e-6)
    assert bool(((q[:, [1, 2, 5]].double() - exp).abs() <= bound(exp, weight, d, BF16)).all())


def test_rows_far_apart(ops):
    """Offsets past 2^31 values, in and out."""
    announce("qk_norm_rope rows far apart")
    stride = 1_200_000_000
    big = torch.empty(2 * stride + 4096, dtype=BF16, device="cuda")
    q, k = big.as_strided((3, 4, 64), (stride, 64, 1)), big.as_strided((3, 2, 64), (stride, 64, 1), 1024)
    qc, kc = randn((3, 4, 64), 1, BF16), randn((3, 2, 64), 2, BF16)
    q.copy_(qc)
    k.copy_(kc)
    w, table = randn((64,), 3, BF16), table_of(9, 64)
    ops.qk_norm_rope(q, k, w.cuda(), w.cuda(), table.cuda(), i32([1, 8, 3]), q_out=q, k_out=k)
    check(q, qc, w, table, [1, 8, 3], 1e-6, False)
    check(k, kc, w, table, [1, 8, 3], 1e-6, False)


def test_table(ops):
    """rope_table: angles in 64 bits, at far positions too."""
    t = ops.rope_table(100000, 32, 5000.0).cpu()
    angle = 99999 * 5000.0 ** (-torch.arange(0, 32, 2, dtype=torch.float64) / 32)
    assert float((t[-1].double() - torch.cat([angle.cos(), angle.sin()])).abs().max()) < 1e-7


def test_refusals(ops):
    q, k = torch.zeros((2, 4, 64), dtype=BF16, device="cuda"), torch.zeros((2, 2, 64), dtype=BF16, device="cuda")
    w, table, pos = torch.ones(64, dtype=BF16, device="cuda"), torch.zeros((5, 64), device="cuda"), i32([0, 1])
    ops.qk_norm_rope(q, k, w, w, table, pos)
    big = torch.zeros((2, 8, 64), dtype=BF16, device="cuda")
    for args, more, error in [
            ((q.half(), k, w, w, table, pos), {}, TypeError), ((q, k, w.float(), w, table, pos), {}, TypeError),
            ((q, k[:1], w, w, table, pos), {}, ValueError), ((q, k[..., :32], w, w, table, pos), {}, ValueError),
            ((q, k, w[:32], w, table, pos), {}, ValueError), ((q, k, w, w, table[:, :40].contiguous(), pos), {}, ValueError),
            ((q, k, w, w, table.double(), pos), {}, TypeError), ((q, k, w, w, table, pos[:1]), {}, ValueError),
            ((q, k, w, w, table, pos.long()), {}, TypeError), ((q.cpu(), k, w, w, table, pos), {}, ValueError),
            ((q, k, w, w, table, pos), {"q_out": k}, ValueError),
            ((q[:0], k[:0], w, w, table, pos[:0]), {}, ValueError),
            ((big[:, :4], big[:, 4:6], w, w, table, pos), {"q_out": big[:, 2:6]}, RuntimeError),  # meets its input and k
            ((big[:, :4], big[:, 4:6], w, w, table, pos), {"k_out": big[:, 3:5]}, RuntimeError),
            ((q, k, w, w, table, pos), {"q_out": big[:, :4], "k_out": big[:, 3:5]}, RuntimeError)]:
        with pytest.raises(error):
            ops.qk_norm_rope(*args, **more)
    ops.qk_norm_rope(big[:, :4], big[:, 4:6], w, w, table, pos, k_out=big[:, 6:])  # one beside the other


def test_graph_and_streams(ops):
    """A captured call replays with other inputs; a call on another stream, ordered by the caller."""
    announce("qk_norm_rope graph")
    q, k = randn((5, 4, 128), 1, BF16).cuda(), randn((5, 2, 128), 2, BF16).cuda()
    w, table, pos = randn((128,), 3, BF16).cuda(), table_of(64, 128).cuda(), i32([3, 9, 0, 63, 5])
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.qk_norm_rope(q, k, w, w, table, pos, q_out=qo, k_out=ko)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.qk_norm_rope(q, k, w, w, table, pos, q_out=qo, k_out=ko)
    for r in range(3):
        q.copy_(randn((5, 4, 128), 10 + r, BF16))
        pos.copy_(torch.tensor([r, 9, 1, 62, 5]))
        want = ops.qk_norm_rope(q, k, w, w, table, pos)
        qo.fill_(float("nan"))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("d", [32, 80, 256])
@pytest.mark.parametrize("eps", [0.0, 2.0 ** -140, 2.0 ** -101, 2.0 ** -99])
def test_small_heads(ops, dtype, neighbours, d, eps):
    """Heads whose mean square lies below fp32's normal numbers, down to the type's smallest values, beside heads of one and
    of zeros, with and without an eps of that size."""
    announce(f"qk_norm_rope small heads d{d} {neighbours} eps{eps} {dtype}")
    least = 2.0 ** -133 if dtype == BF16 else 2.0 ** -24
    x = randn((1, 12, d), 20, dtype)
    for h, e in enumerate([-50, -55, -62, -64, -66, -70, -80, -110, -126]):
        x[0, h] = (x[0, h].double() * 2.0 ** e).to(dtype)
    x[0, 9] = 0.0
    x[0, 9, 3] = least
    x[0, 10] = least
    x[0, 11] = 0.0
    w, table = randn((d,), 21, dtype), table_of(1, 16)
    got, _ = ops.qk_norm_rope(x.cuda(), x.cuda(), w.cuda(), w.cuda(), table.cuda(), i32([0]), eps=eps, neighbours=neighbours)
    got = got.cpu().double()
    exp, weight = oracle.norm_rope(x, w, table, [0], eps, neighbours)  # (0 / 0 without an eps: NaN)
    assert torch.equal(got.isnan(), exp.isnan())
    off = (got - exp).abs()
    assert bool((off <= bound(exp, weight, d, dtype))[~exp.isnan()].all()), float(off.nan_to_num().max())
