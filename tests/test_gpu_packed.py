"""Attention over packed sequences against the formula in float64 on the CPU: lengths
around the kernels' tiles, empty and single-token sequences, slots that are partly used,
rows that see no key, strides, head layouts, both 16-bit types; gradients against the
formula's."""
from __future__ import annotations

import math

import pytest
import torch

from model.packed import packed_attention

BF, F16 = torch.bfloat16, torch.float16
EPS = {BF: 2.0 ** -8, F16: 2.0 ** -11}  # half a step of each type


def _cu(lengths, dev):
    return torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device=dev)


def exact(q, k, v, new, slots, used, scale, g=None):
    """Outputs (and gradients for g) of the packed tensors, the size of each: the same
    sums over absolute values, which the roundings are relative to, and the sums over the
    other factor alone, which roundings of an absolute size are multiplied by."""
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    out, gq, gk, gv = (torch.zeros_like(t) for t in (q, q, k, v))
    size, other = ([torch.zeros_like(t) for t in (q, q, k, v)] for _ in range(2))
    rep = q.shape[1] // k.shape[1]
    qa = ka = 0
    for n, slot, m in zip(new, slots, used):
        for h in range(q.shape[1] if n and m else 0):
            qs, ks = slice(qa, qa + n), slice(ka, ka + m)
            Q, K, V = q[qs, h], k[ks, h // rep], v[ks, h // rep]
            hidden = torch.ones(n, m, dtype=torch.bool).triu(m - n + 1)
            S = (Q @ K.t() * scale).masked_fill(hidden, -math.inf)
            P = torch.nan_to_num(torch.softmax(S, -1), 0.0)  # rows without a key
            out[qs, h] = P @ V
            size[0][qs, h] = P @ V.abs()
            if g is None:
                continue
            G = g[qs, h].detach().double().cpu()
            dP = G @ V.t()
            D = (G * out[qs, h]).sum(-1, keepdim=True)
            dS = P * (dP - D) * scale
            W = P * (G.abs() @ V.abs().t() + (G.abs() * size[0][qs, h]).sum(-1, keepdim=True)) * scale
            gq[qs, h] = dS @ K
            gk[ks, h // rep] += dS.t() @ Q
            gv[ks, h // rep] += P.t() @ G
            size[1][qs, h] = W @ K.abs()
            size[2][ks, h // rep] += W.t() @ Q.abs()
            size[3][ks, h // rep] += P.t() @ G.abs()
            other[1][qs, h] = (~hidden).double() @ K.abs() * scale
            other[2][ks, h // rep] += (~hidden).double().t() @ Q.abs() * scale
        qa, ka = qa + n, ka + slot
    return (out, gq, gk, gv), [*zip(size, other)]


def close(got, want, sizes, dtype, roundings):
    """Within `roundings` half steps of the type of the terms' absolute sum, and a last one
    of the result itself.  fp16 rounds to multiples of 2^-24 below 2^-14: half of that for
    the result, and for each dS of a gradient of q or k times its factor of K or Q."""
    got, (size, other) = got.detach().double().cpu(), sizes
    assert got.shape == want.shape and torch.isfinite(got).all()
    bar = EPS[dtype] * (roundings * size + want.abs()) + (2.0 ** -25 * (1 + other) if dtype == F16 else 0.0)
    worst = ((got - want).abs() - bar).max().item() if got.numel() else 0.0
    assert worst <= 0.0, worst


def _make(dev, dtype, rows, krows, heads, kv, hd, seed=0):
    torch.manual_seed(seed)
    q = torch.randn(rows, heads, hd).mul_(1.5).to(dtype)
    k = torch.randn(krows, kv, hd).mul_(1.5).to(dtype)
    v, g = torch.randn(krows, kv, hd).to(dtype), torch.randn(rows, heads, hd).to(dtype)
    return tuple(t.to(dev) for t in (q, k, v, g))


# Roundings, in half steps of the type on the absolute sums.  Output: the probabilities' one
# (fp32 scores of up to 60 units with 2^-24 relative errors add 2^-17 and less: under half a
# fp16 step).  Gradients of q and k: dS's one, and what the output's two roundings and the
# probabilities' one leave in D (half a step of |G . O|).  Gradient of v: the probabilities' one.
OUT, GRAD = 1.5, 2.5

TRAIN = [
    (96, 8, 4, BF, [1]), (96, 8, 4, BF, [63, 1, 65]), (96, 4, 2, F16, [128, 0, 127, 129]),
    (64, 4, 4, BF, [257, 31, 33]), (64, 3, 1, F16, [64, 64, 1, 1, 95]), (128, 8, 2, BF, [200, 311]),
    (128, 4, 1, F16, [32, 1, 0, 0, 160]), (96, 6, 2, BF, [5] * 70), (64, 12, 4, BF, [1] * 130 + [300]),
    (128, 2, 2, BF, [0, 0]), (96, 16, 1, BF, [77, 130]),
    # long chains on few key tiles: dK and dV from several ranges of rows
    (64, 8, 1, BF, [1100, 37]), (128, 8, 1, F16, [900, 300]), (96, 8, 1, BF, [0, 1300, 1]),
    # more sequences than the tiles are ranked for
    (64, 2, 1, BF, [3] * 300 + [150]), (128, 2, 2, F16, [1, 0, 2] * 120)]


@pytest.mark.gpu
@pytest.mark.parametrize("hd,heads,kv,dtype,lengths", TRAIN)
@pytest.mark.parametrize("behind", [0, 37])
def test_forward_and_gradients(dev, hd, heads, kv, dtype, lengths, behind):
    T = sum(lengths) + behind
    q, k, v, g = _make(dev, dtype, T, T, heads, kv, hd)
    cu = _cu(lengths, dev)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = packed_attention(*leaves, cu)
    grads = torch.autograd.grad(out, leaves, g)
    with torch.no_grad():
        plain = packed_attention(q, k, v, cu)
    want, size = exact(q, k, v, lengths, lengths, lengths, hd ** -0.5, g)
    close(out, want[0], size[0], dtype, OUT)
    close(plain, want[0], size[0], dtype, OUT)
    for got, w, s in zip(grads, want[1:], size[1:]):
        close(got, w, s, dtype, GRAD)
    if behind:  # rows of no sequence
        assert not any(bool(t[-behind:].any()) for t in (out, plain, *grads))
    again = torch.autograd.grad(packed_attention(*leaves, cu), leaves, g)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


SLOTS = [
    # (head_dim, heads, kv heads, type, new tokens, rows of the slots, rows in use)
    (96, 8, 4, BF, [1, 1, 1], [40, 320, 1], [33, 320, 1]),
    (96, 8, 4, BF, [1] * 9, [700] * 9, [1, 2, 31, 32, 33, 64, 65, 699, 700]),
    (128, 16, 2, F16, [1], [9001], [8777]),
    (64, 8, 1, BF, [1, 0, 1], [130, 64, 5], [129, 64, 0]),
    (64, 34, 1, BF, [1, 2], [500, 77], [400, 70]),
    (128, 4, 4, F16, [2, 1, 3], [300, 40, 64], [257, 40, 2]),      # more queries than keys
    (96, 8, 4, BF, [70, 1, 130], [500, 333, 130], [450, 300, 130]),  # chunks beside single tokens
    (64, 6, 2, F16, [33], [5000], [4567]),
    (128, 8, 2, BF, [200], [4000], [0])]


@pytest.mark.gpu
@pytest.mark.parametrize("hd,heads,kv,dtype,new,slots,used", SLOTS)
def test_slots(dev, hd, heads, kv, dtype, new, slots, used):
    q, k, v, g = _make(dev, dtype, sum(new), sum(slots), heads, kv, hd)
    want, size = exact(q, k, v, new, slots, used, 0.11, g)
    at = 0
    for slot, m in zip(slots, used):  # what lies behind a slot's length is not read
        k[at + m:at + slot], v[at + m:at + slot] = math.nan, math.inf
        at += slot
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    args = dict(cu_seqlens_k=_cu(slots, dev), scale=0.11,
                key_lengths=torch.tensor(used, dtype=torch.int32, device=dev))
    with torch.no_grad():
        close(packed_attention(q, k, v, _cu(new, dev), **args), want[0], size[0], dtype, OUT)
    out = packed_attention(*leaves, _cu(new, dev), **args)
    close(out, want[0], size[0], dtype, OUT)
    for got, w, s in zip(torch.autograd.grad(out, leaves, g), want[1:], size[1:]):
        close(got, w, s, dtype, GRAD)


@pytest.mark.gpu
def test_strides(dev):
    """Slices of one fused projection, a transposed tensor, rows off 16-byte boundaries and
    broadcast heads."""
    T, heads, kv, hd, cu = 150, 4, 2, 64, [100, 50]
    q, k, v, g = _make(dev, BF, T, T, heads, kv, hd)
    want = packed_attention(q, k, v, _cu(cu, dev))
    fused = torch.cat([q, k, v], 1)
    got = packed_attention(fused[:, :heads], fused[:, heads:heads + kv], fused[:, heads + kv:], _cu(cu, dev))
    assert torch.equal(got, want)
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(packed_attention(*turned, _cu(cu, dev)), want)
    odd = [torch.empty(t.numel() + 3, dtype=BF, device=dev)[3:].view(t.shape).copy_(t) for t in (q, k, v)]
    assert torch.equal(packed_attention(*odd, _cu(cu, dev)), want)
    one = [t.clone().requires_grad_() for t in (q, k[:, :1], v[:, :1])]
    out = packed_attention(one[0], one[1].expand(-1, kv, -1), one[2].expand(-1, kv, -1), _cu(cu, dev))
    got = torch.autograd.grad(out, one, g)
    wide = [t.detach().expand(-1, h, -1).contiguous().requires_grad_() for t, h in zip(one, (heads, kv, kv))]
    full = torch.autograd.grad(packed_attention(*wide, _cu(cu, dev)), wide, g)
    assert torch.equal(got[0], full[0])
    for a, b in zip(got[1:], full[1:]):
        assert torch.equal(a, b.sum(1, keepdim=True))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40])
def test_offsets_past_32_bits(dev, new):
    """The second sequence's keys lie past 2^31 elements."""
    kv, hd, n = 4, 96, 500
    rows = (1 << 31) // (kv * hd) + 3000
    torch.manual_seed(0)
    q, g = (torch.randn(2 * new, 8, hd, device=dev).to(BF) for _ in range(2))
    small = [torch.randn(10 + n, kv, hd, device=dev).to(BF) for _ in range(2)]
    big = [torch.empty(rows, kv, hd, dtype=BF, device=dev) for _ in range(2)]
    for b, s in zip(big, small):
        b[:10], b[-n:] = s[:10], s[10:]
    used = torch.tensor([10, n], dtype=torch.int32, device=dev)
    res = []
    for kvs, ends in ((small, [0, 10, 10 + n]), (big, [0, rows - n, rows])):
        leaves = [t.requires_grad_() for t in (q.clone(), *kvs)]
        out = packed_attention(*leaves, _cu([new, new], dev), key_lengths=used,
                               cu_seqlens_k=torch.tensor(ends, dtype=torch.int32, device=dev))
        gq, gk, gv = torch.autograd.grad(out, leaves, g)
        res.append([out, gq, gk[:10], gv[:10], gk[-n:], gv[-n:]])
        if kvs is big:
            assert not bool(gk[10:1000].any()) and not bool(gv[-n - 1000:-n].any())
    (want, size) = exact(q, *small, [new, new], [10, n], [10, n], hd ** -0.5)
    for r in res:  # the key ranges may be cut otherwise
        close(r[0], want[0], size[0], BF, OUT)
    for a, b in zip(res[0][1:], res[1][1:]):
        assert float((a.float() - b.float()).norm()) <= 2.0 ** -6 * float(a.float().norm())


@pytest.mark.gpu
def test_bounds_that_make_no_sense(dev):
    """Bounds outside the tensors, and decreasing ones, are cut to them: such a call ends, and
    the next one is right."""
    T = 200
    q, k, v, g = _make(dev, BF, T, T, 4, 2, 64)
    good = packed_attention(q, k, v, _cu([120, 80], dev))
    for ends in ([-5, 500, 2 ** 31 - 1], [0, 150, 20], [0, -2 ** 31, 200], [9, 9, 9]):
        cu = torch.tensor(ends, dtype=torch.int32, device=dev)
        for more in ({}, {"cu_seqlens_k": cu.flip(0).contiguous()},
                     {"key_lengths": torch.tensor([-7, 2 ** 31 - 1], dtype=torch.int32, device=dev)}):
            leaves = [t.clone().requires_grad_() for t in (q, k, v)]
            out = packed_attention(*leaves, cu, **more)
            assert out.shape == q.shape
            assert [x.shape for x in torch.autograd.grad(out, leaves, g)] == [q.shape, k.shape, v.shape]
            packed_attention(q[:2], k, v, cu, **{"cu_seqlens_k": cu, **more})
    assert torch.equal(packed_attention(q, k, v, _cu([120, 80], dev)), good)


def hd_scale(hd):
    return 1.01 * hd ** -0.5  # and the roundings of the products with it


@pytest.mark.gpu
@pytest.mark.parametrize("rows,keys,bounds", [(0, 0, [0]), (0, 5, [0, 0]), (7, 7, [0]), (3, 0, [0, 3]), (1, 1, [0, 1])])
def test_smallest(dev, rows, keys, bounds):
    q, k, v, g = _make(dev, BF, rows, keys, 4, 2, 64)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    cu = torch.tensor(bounds, dtype=torch.int32, device=dev)
    ends = torch.tensor(bounds, dtype=torch.int32, device=dev).clamp_max(keys)
    out = packed_attention(*leaves, cu, cu_seqlens_k=ends)
    grads = torch.autograd.grad(out, leaves, g)
    if (rows, keys) == (1, 1):  # one key: its value, whatever the score
        assert torch.equal(out, v.repeat_interleave(2, 1))
        # dS = G . v - D, the same sum of 64 products in fp32 twice, in two orders: each is
        # within 64 half steps (2^-24) of its absolute sum, so dS is under 2^-17 of it
        bar = 2.0 ** -17 * (g.float() * out.float()).abs().sum(-1, keepdim=True) * hd_scale(64)
        assert bool((grads[0].float().abs() <= bar * k.float().abs().repeat_interleave(2, 1)).all())
        assert bool((grads[1].float().abs() <= (bar * q.float().abs()).view(1, 2, 2, 64).sum(2)).all())
    else:
        assert not any(bool(t.any()) for t in (out, *grads))


@pytest.mark.gpu
@pytest.mark.parametrize("hd,dtype", [(96, BF), (64, F16)])
def test_extreme_scores(dev, hd, dtype):
    """Rows of hugely negative, hugely positive and of equal scores: a maximum that is far
    from 0 loses nothing."""
    q, k, v, _ = _make(dev, dtype, 90, 90, 2, 2, hd)
    big = 2.0 ** (60 if dtype == BF else 7)
    q[:30], k[:, 0] = big, -big       # head 0: every score the same, far below 0
    q[30:60] = -big                   # far above
    q[60:] = 0.0
    k[:, 1] = big
    out = packed_attention(q, k, v, _cu([90], dev))
    want = v.double().cumsum(0) / torch.arange(1, 91, device=dev, dtype=torch.float64)[:, None, None]
    size = v.double().abs().cumsum(0) / torch.arange(1, 91, device=dev, dtype=torch.float64)[:, None, None]
    close(out, want.cpu(), (size.cpu(), torch.zeros_like(size).cpu()), dtype, OUT)
