"""Rotary positions against the formula in float64: layouts, parts of a head, types, strides,
odd sizes, positions outside the tables; gradients against the formula's and against differences."""
from __future__ import annotations

import pytest
import torch

from model.rotary import plain_rotary, rotary

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = {BF: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}  # half a step of each type


def tables(rows, rd, dtype=F32, seed=3):
    g = torch.Generator().manual_seed(seed)
    a = torch.rand(rows, rd // 2, generator=g, dtype=torch.float64) * 40
    return (1.1 * a.cos()).to(dtype), (1.1 * a.sin()).to(dtype)


def exact(x, cos, sin, positions, inter, back=False):
    """(result, the sums of its terms' absolute values), in float64 on the CPU."""
    x = x.detach().double().cpu()
    at = positions.cpu().long()
    c, s = (t.double().cpu()[at.clamp(0, len(t) - 1)].unsqueeze(-2) for t in (cos, sin))
    s = -s if back else s
    rd = 2 * cos.shape[1]
    lo, hi = (slice(0, rd, 2), slice(1, rd, 2)) if inter else (slice(0, rd // 2), slice(rd // 2, rd))
    y, size = x.clone(), torch.zeros_like(x)
    a, b = x[..., lo], x[..., hi]
    y[..., lo], y[..., hi] = a * c - b * s, b * c + a * s
    size[..., lo], size[..., hi] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    y[..., :rd][((at < 0) | (at >= len(cos)))] = float("nan")
    return y, size


def close(got, want, dtype):
    """One rounding of the result, and three of fp32 (two products, a sum) on the terms' sizes; fp16
    rounds to multiples of 2^-24 below 2^-14."""
    y, size = want
    got = got.detach().double().cpu()
    assert got.shape == y.shape
    assert torch.equal(got.isnan(), y.isnan())
    bar = EPS[dtype] * y.abs() + 1.5 * 2.0 ** -23 * size + (2.0 ** -25 if dtype == F16 else 0.0)
    worst = ((got - y).abs() - bar).nan_to_num(-1.0)
    assert worst.numel() == 0 or worst.max().item() <= 0.0, worst.max().item()


CASES = [
    # rows, heads, kv heads, head_dim, rotary_dim
    (1, 8, 4, 96, 96), (77, 8, 4, 96, 48), (33, 6, 2, 64, 16), (130, 16, 2, 128, 64), (19, 3, 1, 96, 24),
    (7, 2, 2, 96, 72), (5, 4, 4, 80, 80), (9, 1, 1, 256, 128), (4, 2, 1, 200, 40), (6, 3, 3, 5, 4), (3, 1, 2, 7, 0),
    (2, 100, 5, 64, 64), (11, 2, 1, 90, 30), (1500, 8, 4, 96, 96), (300, 40, 40, 64, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,heads,kv,hd,rd", CASES)
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("inter", [False, True])
def test_forward_and_gradients(dev, rows, heads, kv, hd, rd, dtype, inter):
    torch.manual_seed(rows + hd + rd)
    q, k, gq, gk = (torch.randn(rows, h, hd).to(dtype).to(dev) for h in (heads, kv, heads, kv))
    cos, sin = (t.to(dev) for t in tables(60, rd))
    positions = torch.randint(0, 60, (rows,), device=dev, dtype=torch.int32 if inter else torch.int64)
    leaves = [q.clone().requires_grad_(), k.clone().requires_grad_()]
    out = rotary(*leaves, cos, sin, positions, interleaved=inter)
    grads = torch.autograd.grad(out, leaves, (gq, gk))
    for got, x in zip(out, (q, k)):
        close(got, exact(x, cos, sin, positions, inter), dtype)
    for got, g in zip(grads, (gq, gk)):
        close(got, exact(g, cos, sin, positions, inter, back=True), dtype)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(out, rotary(q, k, cos, sin, positions, interleaved=inter)))
        assert torch.equal(rotary(q, None, cos, sin, positions, interleaved=inter)[0], out[0])
        for a, b in zip(out, plain_rotary(q, k, cos, sin, positions, inter)):
            assert float((a.double() - b.double()).abs().max()) <= 2 * EPS[dtype] * float(b.abs().max()) + 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("table", [BF, F16, F32])
def test_tables_types_and_strides(dev, table):
    """Tables of 16 bits, cut from wider rows, at odd addresses, in another order."""
    torch.manual_seed(0)
    q, k = (torch.randn(50, h, 96).to(BF).to(dev) for h in (8, 4))
    positions = torch.randint(0, 40, (50,), device=dev)
    for rd in (96, 24):
        cos, sin = (t.to(dev) for t in tables(40, rd, table))
        want = [exact(x, cos, sin, positions, False) for x in (q, k)]
        both = [torch.cat([t, t], 1) for t in (cos, sin)]
        odd = [torch.empty(t.numel() + 1, dtype=table, device=dev)[1:].view(t.shape).copy_(t) for t in (cos, sin)]
        for c, s in ((cos, sin), [b[:, :rd // 2] for b in both], odd, [t.t().contiguous().t() for t in (cos, sin)]):
            for got, w in zip(rotary(q, k, c, s, positions), want):
                close(got, w, BF)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides(dev, dtype):
    """Slices of one projection, transposed tensors, odd addresses, broadcast heads, more
    dimensions: the same bits."""
    torch.manual_seed(1)
    B, T, H, KV, hd = 3, 21, 4, 2, 64
    q, k = torch.randn(B, T, H, hd).to(dtype).to(dev), torch.randn(B, T, KV, hd).to(dtype).to(dev)
    cos, sin = (t.to(dev) for t in tables(30, 32))
    positions = torch.randint(0, 30, (B, T), device=dev)
    want = rotary(q, k, cos, sin, positions)
    close(want[0], exact(q, cos, sin, positions, False), dtype)
    fused = torch.cat([q, k], 2)
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k)]
    odd = [torch.empty(t.numel() + 1, dtype=dtype, device=dev)[1:].view(t.shape).copy_(t) for t in (q, k)]
    last = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k)]
    for a, b in ((fused[:, :, :H], fused[:, :, H:]), turned, odd, last):
        got = rotary(a, b, cos, sin, positions)
        assert all(torch.equal(x, y) and x.is_contiguous() for x, y in zip(got, want))
    one = k[:, :, :1].clone().requires_grad_()
    g = torch.randn(B, T, H, hd).to(dtype).to(dev)
    wide = rotary(one.expand(-1, -1, H, -1), None, cos, sin, positions.t().contiguous().t())[0]
    got, = torch.autograd.grad(wide, one, g)
    each = rotary(g, None, cos, -sin, positions)[0]
    assert torch.equal(got, each.sum(2, keepdim=True))


@pytest.mark.gpu
def test_positions_outside_the_tables(dev):
    q, k = torch.randn(6, 2, 64, device=dev), torch.randn(6, 1, 64, device=dev)
    cos, sin = (t.to(dev) for t in tables(10, 32))
    for dtype in (torch.int32, torch.int64):
        big = torch.iinfo(dtype)
        positions = torch.tensor([0, 9, 10, -1, big.max, big.min], dtype=dtype, device=dev)
        q1 = q.clone().requires_grad_()
        out = rotary(q1, k, cos, sin, positions)
        for x, y in zip(out, (q, k)):
            close(x, exact(y, cos, sin, positions, False), F32)
            assert torch.equal(x[..., 32:], y[..., 32:])
        g, = torch.autograd.grad(out[0], q1, torch.ones_like(q))
        assert bool(g[2:, :, :32].isnan().all()) and bool(torch.isfinite(g[:2]).all())
    assert bool(rotary(q, None, cos[:0], sin[:0], positions)[0][..., :32].isnan().all())
    assert [t.shape for t in rotary(q[:0], k[:0], cos, sin, positions[:0])] == [(0, 2, 64), (0, 1, 64)]


@pytest.mark.gpu
def test_values_that_are_not_finite_stay_in_their_pair(dev):
    q = torch.randn(4, 2, 64, device=dev).to(BF)
    cos, sin = (t.to(dev) for t in tables(10, 64))
    positions = torch.arange(4, device=dev)
    want = rotary(q, None, cos, sin, positions)[0]
    q[1, 0, 3], q[2, 1, 40] = float("inf"), float("nan")
    got = rotary(q, None, cos, sin, positions)[0]
    differ = (got != want) | got.isnan()
    assert sorted(map(tuple, differ.nonzero().tolist())) == [(1, 0, 3), (1, 0, 35), (2, 1, 8), (2, 1, 40)]


@pytest.mark.gpu
def test_gradients_against_differences_and_twice(dev):
    """The map is linear: differences of the outputs are the gradient's product, up to 2^-22 of the sums'
    sizes; and the gradient can be differentiated again."""
    torch.manual_seed(2)
    q, k = (torch.randn(9, h, 40, device=dev, requires_grad=True) for h in (3, 2))
    g, d = torch.randn(9, 3, 40, device=dev), torch.randn(9, 3, 40, device=dev)
    cos, sin = (t.to(dev) for t in tables(12, 20))
    positions = torch.randint(0, 12, (9,), device=dev)
    f = lambda x: rotary(x, None, cos, sin, positions, interleaved=True)[0]
    gq, = torch.autograd.grad(f(q), q, g)
    moved = (f(q.detach() + d) - f(q.detach() - d)).double() / 2
    # values of up to 6 units, each of 9 x 3 x 40 within 2^-22 of them
    assert abs(float((moved * g.double()).sum() - (gq.double() * d.double()).sum())) <= 1080 * 6 * 6 * 2.0 ** -22
    go = g.clone().requires_grad_()
    out = rotary(q, k, cos, sin, positions, interleaved=True)
    first, = torch.autograd.grad(out[0], q, go, create_graph=True)
    second, = torch.autograd.grad(first, go, d)
    assert torch.equal(second, f(d))
    only, = torch.autograd.grad(rotary(q, k, cos, sin, positions)[1].sum(), k)
    assert only.shape == k.shape


@pytest.mark.gpu
def test_captured_and_other_streams(dev):
    torch.manual_seed(4)
    cos, sin = (t.to(dev) for t in tables(64, 96))
    q, k, gq, gk = (torch.randn(40, h, 96, device=dev).to(BF) for h in (8, 4, 8, 4))
    positions = torch.randint(0, 64, (40,), device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaves = [q.clone().requires_grad_(), k.clone().requires_grad_()]
        for _ in range(2):
            torch.autograd.grad(rotary(*leaves, cos, sin, positions), leaves, (gq, gk))
        graph = torch.cuda.CUDAGraph()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = rotary(*leaves, cos, sin, positions)
        grads = torch.autograd.grad(out, leaves, (gq, gk))
    for i in range(4):
        with torch.no_grad():
            for t in (*leaves, gq, gk):
                t.copy_(torch.randn_like(t.float()).to(BF))
            positions.copy_(torch.randint(0, 64, (40,), device=dev))
        graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            want = rotary(*leaves, cos, sin, positions) + rotary(gq, gk, cos, -sin, positions)
        assert all(torch.equal(a, b) for a, b in zip((*out, *grads), want)), i


@pytest.mark.gpu
def test_many_rows(dev):
    """More rows than one line of a launch holds, and offsets past 2^31 elements."""
    rows = (1 << 23) * 32 + 5
    q = torch.zeros(rows, 1, 16, dtype=BF, device=dev)
    cos, sin = (t.to(dev) for t in tables(4, 16))
    q[-3:] = torch.randn(3, 1, 16, device=dev).to(BF)
    q[0] = 1.0
    positions = torch.ones(rows, dtype=torch.int32, device=dev)
    out = rotary(q, None, cos, sin, positions)[0]
    for at in (slice(0, 2), slice(-4, None)):
        close(out[at], exact(q[at], cos, sin, positions[at], False), BF)
    assert not bool(out[1:-3].any())
