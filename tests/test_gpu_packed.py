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
    (64, 8, 1, BF, [1100, 37]), (128, 8, 1, F16, [900, 300]), (96, 8, 1, BF, [0, 1300, 1])]


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
