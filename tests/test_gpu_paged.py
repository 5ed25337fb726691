"""The cache of pages: appending, attention of single tokens, trees and chunks, and keeping an
accepted branch, each against the formula in float64 on the CPU."""
from __future__ import annotations

import math
import random

import pytest
import torch

from model.paged import paged_append, paged_attention, paged_keep
from test_gpu_rotary import exact as exact_rotary, tables

BF, F16 = torch.bfloat16, torch.float16
EPS = {BF: 2.0 ** -8, F16: 2.0 ** -11}  # half a step of each type


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def starts(n):
    return [0] + torch.tensor(n, dtype=torch.int64).cumsum(0).tolist()


class Pool:
    """Pages in random order for sequences of so many keys, everything else in them NaN."""

    def __init__(self, dev, dtype, keys, page, kv, hd, planes=2, wide=2, seed=0):
        rng = random.Random(seed)
        need = [(n + page - 1) // page for n in keys]
        self.width = max(need, default=0) + wide
        order = list(range(sum(need) + 2))
        rng.shuffle(order)
        self.rows, at = [], 0
        for n in need:
            self.rows.append(order[at:at + n] + [-1] * (self.width - n))
            at += n
        self.page, self.dtype = page, dtype
        self.table = ints(self.rows, dev) if keys else torch.zeros(0, self.width, dtype=torch.int32, device=dev)
        self.planes = torch.full((planes, len(order), page, kv, hd), math.nan, dtype=dtype, device=dev)
        self.k, self.v = self.planes[0], self.planes[1]

    def at(self, seq, a, b):
        x = torch.arange(a, b)
        return torch.tensor([self.rows[seq][i // self.page] * self.page + i % self.page for i in x.tolist()],
                            dtype=torch.int64, device=self.planes.device)


def make(dev, dtype, past, new, page, heads, kv, hd, seed=0, behind=0):
    """A pool that holds random keys of every sequence's first past + new positions, and queries."""
    torch.manual_seed(seed)
    pool = Pool(dev, dtype, [a + b for a, b in zip(past, new)], page, kv, hd, seed=seed)
    for i, (a, b) in enumerate(zip(past, new)):
        rows = pool.at(i, 0, a + b)
        pool.k.flatten(0, 1)[rows] = torch.randn(a + b, kv, hd).mul_(1.5).to(dtype).to(dev)
        pool.v.flatten(0, 1)[rows] = torch.randn(a + b, kv, hd).to(dtype).to(dev)
    q = torch.randn(sum(new) + behind, heads, hd).mul_(1.5).to(dtype).to(dev)
    return pool, q


def random_tree(new, seed, words=None, empty=False):
    """(bits [rows, words], which of its sequence's rows each row sees) of random trees; empty: some
    rows see nothing of it."""
    rng = random.Random(seed)
    words = words or (max(new + [1]) + 63) // 64
    sees = []
    for n in new:
        rows = []
        for j in range(n):
            p = rng.randrange(max(-1, j - 5), j) if j else -1
            rows.append((rows[p] if p >= 0 else 0) | 1 << j)
        if empty:
            rows = [0 if rng.random() < 0.3 else r for r in rows]
        sees += rows
    full = (1 << 64) - 1
    signed = [[(w - (1 << 64) if w >> 63 else w) for w in ((r >> 64 * i) & full for i in range(words))] for r in sees]
    return torch.tensor(signed, dtype=torch.int64).view(len(sees), words), sees


def exact(pool, q, past, new, scale, sees=None, lost=()):
    """(outputs, the sums of their terms' absolute values); lost: (sequence, page slot) not there."""
    q = q.double().cpu()
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    k, v = (t.flatten(0, 1).double().cpu() for t in (pool.k, pool.v))
    rep, at = q.shape[1] // k.shape[1], 0
    for i, (a, b) in enumerate(zip(past, new)):
        rows = pool.at(i, 0, a + b).cpu()
        hidden = torch.ones(b, a + b, dtype=torch.bool).triu(a + 1)
        for j in range(b if sees is not None else 0):
            hidden[j, a:] = torch.tensor([not sees[at + j] >> x & 1 for x in range(b)], dtype=torch.bool)
        for seq, slot in lost:
            if seq == i:
                hidden[:, slot * pool.page:(slot + 1) * pool.page] = True
        for h in range(q.shape[1] if b else 0):
            S = (q[at:at + b, h] @ k[rows, h // rep].t() * scale).masked_fill(hidden, -math.inf)
            P = torch.nan_to_num(torch.softmax(S, -1), 0.0)
            V = torch.where(hidden.all(0)[:, None], 0.0, v[rows, h // rep])
            out[at:at + b, h], size[at:at + b, h] = P @ V, P @ V.abs()
        at += b
    return out, size


def close(got, want, dtype):
    """The probabilities' one rounding and what the fp32 scores (up to 60 units, 2^-24 each) add to
    them, under half a step more, on the terms' sizes; the result's own on itself."""
    out, size = want
    got = got.double().cpu()
    assert got.shape == out.shape and torch.isfinite(got).all()
    bar = EPS[dtype] * (1.5 * size + out.abs()) + (2.0 ** -25 if dtype == F16 else 0.0)
    worst = ((got - out).abs() - bar).max().item() if got.numel() else 0.0
    assert worst <= 0.0, worst


ATTEND = [
    # head_dim, heads, kv heads, type, page, keys before, new rows
    (96, 8, 4, BF, 16, [33], [1]), (96, 8, 4, BF, 64, [0, 1, 31, 32, 63, 64, 65, 700], [1] * 8),
    (128, 16, 2, F16, 256, [9001], [1]), (64, 8, 1, BF, 16, [5, 0, 200], [2, 0, 1]),
    (96, 8, 4, BF, 32, [100, 0, 257], [16, 7, 16]), (64, 4, 4, F16, 16, [777], [33]),
    (128, 8, 8, BF, 64, [300, 17], [64, 63]), (96, 12, 4, F16, 16, [500, 40], [100, 3]),
    (64, 34, 1, BF, 128, [400, 70], [1, 2]), (96, 6, 2, BF, 16, [0], [300]), (128, 8, 2, BF, 64, [4000], [200]),
    (64, 2, 2, BF, 16, [50] * 70, [1] * 70), (64, 2, 1, F16, 16, [3, 20] * 150, [1, 2] * 150),
    (96, 8, 4, BF, 16, [2000, 10, 10, 10], [5, 5, 5, 5]), (128, 16, 2, F16, 16, [5001], [64]),
    (64, 3, 1, BF, 4096, [100, 4200], [1, 9]), (96, 8, 4, BF, 64, [20, 30], [0, 0]), (128, 5, 1, BF, 32, [0, 0], [1, 1])]


@pytest.mark.gpu
@pytest.mark.parametrize("hd,heads,kv,dtype,page,past,new", ATTEND)
@pytest.mark.parametrize("tree", [None, "tree", "empty"])
def test_attention(dev, hd, heads, kv, dtype, page, past, new, tree):
    behind = 0 if tree is None else 5
    pool, q = make(dev, dtype, past, new, page, heads, kv, hd, behind=behind)
    bits, sees = (None, None) if tree is None else random_tree(new, 7, empty=tree == "empty")
    if bits is not None:
        bits = torch.cat([bits, torch.full((behind, bits.shape[1]), -1)]).to(dev)
    want = exact(pool, q, past, new, 0.11, sees)
    args = (pool.k, pool.v, pool.table, ints(past, dev), ints(starts(new), dev))
    got = paged_attention(q, *args, tree=bits, scale=0.11)
    close(got, want, dtype)
    assert torch.equal(got, paged_attention(q, *args, tree=bits, scale=0.11))
    if behind:  # rows of no sequence
        assert not bool(got[-behind:].any())


@pytest.mark.gpu
def test_chain_as_a_tree_is_causal(dev):
    past, new = [130, 5], [40, 70]
    pool, q = make(dev, BF, past, new, 16, 8, 4, 96)
    chain = torch.tensor([[((1 << (j + 1)) - 1) & ((1 << 63) - 1) if j < 63 else -1,
                           0 if j < 64 else (1 << (j - 63)) - 1] for n in new for j in range(n)], dtype=torch.int64)
    args = (pool.k, pool.v, pool.table, ints(past, dev), ints(starts(new), dev))
    assert torch.equal(paged_attention(q, *args), paged_attention(q, *args, tree=chain.to(dev)))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 20, 150])
def test_pages_that_are_not_there(dev, new):
    """Page numbers outside the pages: their keys are not seen, and nothing is read of them."""
    past, n = [200, 90], [new, new]
    pool, q = make(dev, BF, past, n, 16, 8, 4, 64)
    full = paged_attention(q, pool.k, pool.v, pool.table, ints(past, dev), ints(starts(n), dev))
    lost = [(0, 2), (0, 5), (1, 0), (0, 12)]
    pool.k[0], pool.v[0] = math.nan, math.inf  # what a wrong read would fetch
    keep = pool.table.clone()
    for value in (-1, len(pool.k), 2 ** 31 - 1, -2 ** 31):
        for seq, slot in lost:
            pool.table[seq, slot] = value
        dropped = [(s, p) for s, p in lost] + [(s, p) for s in range(2) for p, x in enumerate(pool.rows[s]) if x == 0]
        pool.table[keep == 0] = value
        got = paged_attention(q, pool.k, pool.v, pool.table, ints(past, dev), ints(starts(n), dev))
        close(got, exact(pool, q, past, n, 64 ** -0.5, None, dropped), BF)
    assert torch.isfinite(full).all()


@pytest.mark.gpu
def test_lengths_and_bounds_that_make_no_sense(dev):
    """Clamped: such calls end, and the next one is right."""
    past, new = [100, 50], [30, 10]
    pool, q = make(dev, BF, past, new, 16, 4, 2, 64)
    rows = pool.planes.clone()
    good_args = (pool.k, pool.v, pool.table, ints(past, dev), ints(starts(new), dev))
    good = paged_attention(q, *good_args)
    cos, sin = (t.to(dev) for t in tables(300, 64))
    k = torch.randn(40, 2, 64, device=dev).to(BF)
    for ends in ([-5, 500, 2 ** 31 - 1], [0, 35, 20], [0, -2 ** 31, 40], [9, 9, 9]):
        for lens in ([-7, 2 ** 31 - 1], [2 ** 31 - 1, 2 ** 31 - 1], [0, -2 ** 31]):
            assert paged_attention(q, pool.k, pool.v, pool.table, ints(lens, dev), ints(ends, dev)).shape == q.shape
            out = paged_append(q, k, k, pool.k, pool.v, pool.table, ints(lens, dev), ints(ends, dev), cos, sin)
            assert out.shape == q.shape
            paged_keep(pool.planes, pool.table, ints(lens, dev), ints(ends, dev), ints([50, -3], dev),
                       torch.randint(-50, 50, (40,), dtype=torch.int32, device=dev))
    pool.planes.copy_(rows)
    assert torch.equal(paged_attention(q, *good_args), good)
    # many sequences whose bounds go back and forth
    for B in (200, 300):
        ends = ints([0, 40] * (B // 2) + [0], dev)
        table, lens = pool.table[:1].expand(B, -1).contiguous(), ints([70] * B, dev)
        assert paged_attention(q, pool.k, pool.v, table, lens, ends).shape == q.shape


@pytest.mark.gpu
@pytest.mark.parametrize("rows,B,pages,width", [(0, 0, 3, 2), (0, 2, 3, 2), (4, 0, 3, 2), (4, 2, 0, 2), (4, 2, 3, 0)])
def test_smallest(dev, rows, B, pages, width):
    q = torch.randn(rows, 4, 64, device=dev).to(BF)
    k = torch.randn(rows, 2, 64, device=dev).to(BF)
    planes = torch.zeros(2, pages, 16, 2, 64, dtype=BF, device=dev)
    table = torch.zeros(B, width, dtype=torch.int32, device=dev)
    lens = torch.zeros(B, dtype=torch.int32, device=dev)
    cu = ints([0] + [min(2 * (i + 1), rows) for i in range(B)], dev)
    cos, sin = (t.to(dev) for t in tables(9, 64))
    out = paged_attention(q, planes[0], planes[1], table, lens, cu)
    assert out.shape == q.shape and not bool(out.any())
    turned = paged_append(q, k, k, planes[0], planes[1], table, lens, cu, cos, sin)
    assert turned.shape == q.shape and (B > 0 or not bool(turned.any()))
    assert not bool(planes.any())
    kept = torch.ones(B, dtype=torch.int32, device=dev)
    path = torch.zeros(rows, dtype=torch.int32, device=dev)
    new = paged_keep(planes, table, lens, cu, kept, path)
    room = width * 16
    assert new.tolist() == [min(1, room, int(cu[i + 1] - cu[i])) for i in range(B)]


@pytest.mark.gpu
def test_strides(dev):
    """Queries cut from a projection, pages as views of a larger pool or in another order of heads."""
    past, new = [90, 33], [20, 7]
    pool, q = make(dev, BF, past, new, 16, 8, 4, 96)
    args = (pool.table, ints(past, dev), ints(starts(new), dev))
    want = paged_attention(q, pool.k, pool.v, *args)
    fused = torch.cat([q, q], 1)
    odd = torch.empty(q.numel() + 3, dtype=BF, device=dev)[3:].view(q.shape).copy_(q)
    for x in (fused[:, :8], fused[:, 8:], odd, q.transpose(0, 1).contiguous().transpose(0, 1)):
        assert torch.equal(paged_attention(x, pool.k, pool.v, *args), want)
    both = torch.stack([pool.k, pool.v], 3)  # [pages, page, kv, 2, hd]
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (pool.k, pool.v)]
    for k, v in ((both[:, :, :, 0], both[:, :, :, 1]), heads_first):
        assert torch.equal(paged_attention(q, k, v, *args), want)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 40])
def test_offsets_past_32_bits(dev, new):
    """Pages past 2^31 elements."""
    kv, hd, page, past = 4, 128, 256, [300, 500]
    pages = (1 << 32) // (kv * hd * page) + 8
    big = [torch.empty(pages, page, kv, hd, dtype=BF, device=dev) for _ in range(2)]
    torch.manual_seed(0)
    q = torch.randn(2 * new, 8, hd, device=dev).to(BF)
    k, v = (torch.randn(2 * new, kv, hd, device=dev).to(BF) for _ in range(2))
    cos, sin = (t.to(dev) for t in tables(600, 128))
    res = []
    for ps, table in ((big, [[pages - 1, 0, pages - 2], [pages - 5, pages - 3, 1]]), ([t[:6] for t in big], [[3, 0, 2], [5, 4, 1]])):
        for t, seed in zip(ps, (1, 2)):
            for i, row in enumerate(table):
                for j, p in enumerate(row):
                    t[p] = torch.randn(page, kv, hd, generator=torch.Generator().manual_seed(100 * seed + 10 * i + j)).to(BF).to(dev)
        args = (*ps, ints(table, dev), ints(past, dev), ints([0, new, 2 * new], dev))
        turned = paged_append(q, k, v, *args, cos, sin)
        res.append((turned, paged_attention(turned, *args)))
    assert all(torch.equal(a, b) for a, b in zip(*res))


@pytest.mark.gpu
@pytest.mark.parametrize("hd,dtype", [(96, BF), (64, F16)])
def test_extreme_scores(dev, hd, dtype):
    """Hugely negative, positive and equal scores lose nothing."""
    past, new = [80], [12]
    pool, q = make(dev, dtype, past, new, 16, 2, 2, hd)
    rows = pool.at(0, 0, 92)
    big = 2.0 ** (60 if dtype == BF else 7)
    pool.k.flatten(0, 1)[rows, 0], pool.k.flatten(0, 1)[rows, 1] = -big, big
    q[:4], q[4:8], q[8:] = big, -big, 0.0
    got = paged_attention(q, pool.k, pool.v, pool.table, ints(past, dev), ints([0, 12], dev))
    v = pool.v.flatten(0, 1)[rows].double().cpu()
    n = torch.arange(1, 93, dtype=torch.float64)[:, None, None]
    close(got, ((v.cumsum(0) / n)[80:], (v.abs().cumsum(0) / n)[80:]), dtype)


@pytest.mark.gpu
def test_a_sequence_does_not_reach_another(dev):
    past, new = [40, 60], [3, 3]
    pool, q = make(dev, BF, past, new, 16, 4, 2, 64)
    args = (pool.table, ints(past, dev), ints(starts(new), dev))
    want = paged_attention(q, pool.k, pool.v, *args)
    pool.k.flatten(0, 1)[pool.at(0, 5, 9)] = math.nan
    pool.v.flatten(0, 1)[pool.at(0, 5, 9)] = math.inf
    got = paged_attention(q, pool.k, pool.v, *args)
    assert torch.equal(got[3:], want[3:]) and not bool(torch.isfinite(got[:3]).all())


# ------------------------------------------------------------------ appending

APPEND = [
    # head_dim, rotary_dim, heads, kv heads, type, page, keys before, new rows
    (96, 96, 8, 4, BF, 64, [5, 0, 63, 64], [1, 1, 1, 1]), (128, 64, 16, 2, F16, 16, [3, 50], [40, 17]),
    (64, 16, 6, 2, BF, 32, [0], [1]), (96, 24, 8, 1, BF, 16, [0, 9, 100], [33, 0, 2]), (80, 80, 4, 4, F16, 16, [7], [30]),
    (64, 64, 12, 12, BF, 256, [250] * 70, [9] * 70), (40, 6, 2, 1, BF, 16, [1], [20]), (96, 0, 8, 4, BF, 16, [2], [5]),
    (256, 128, 2, 1, F16, 16, [10], [10]), (200, 40, 2, 2, BF, 16, [3], [4])]


@pytest.mark.gpu
@pytest.mark.parametrize("hd,rd,heads,kv,dtype,page,past,new", APPEND)
@pytest.mark.parametrize("norm", ["", "q", "qk"])
@pytest.mark.parametrize("inter", [False, True])
def test_append(dev, hd, rd, heads, kv, dtype, page, past, new, norm, inter):
    torch.manual_seed(hd + rd)
    T, behind = sum(new), 3
    pool = Pool(dev, dtype, [a + b for a, b in zip(past, new)], page, kv, hd)
    pool.planes.normal_()
    before = pool.planes.clone()
    q = torch.randn(T + behind, heads, hd).to(dtype).to(dev)
    k, v = (torch.randn(T + behind, kv, hd).to(dtype).to(dev) for _ in range(2))
    gains = {n: (1 + 0.2 * torch.randn(hd)).to(dtype if n == "q" else torch.float32).to(dev) for n in "qk" if n in norm}
    cos, sin = (t.to(dev) for t in tables(max(a + b for a, b in zip(past, new)), rd))
    got = paged_append(q, k, v, pool.k, pool.v, pool.table, ints(past, dev), ints(starts(new), dev), cos, sin,
                       q_gain=gains.get("q"), k_gain=gains.get("k"), eps=1e-5, interleaved=inter)
    at = torch.cat([torch.arange(a, a + b) for a, b in zip(past, new)])
    rows = torch.cat([pool.at(i, a, a + b) for i, (a, b) in enumerate(zip(past, new))])

    def check(have, x, gain):
        x = x[:T].double().cpu()
        if gain is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * gain.double().cpu()
        want, size = exact_rotary(x, cos, sin, at, inter)
        # the square sum of 256 at most in fp32: 2^-17 of it, half of that in its root; a few roundings more
        bar = EPS[dtype] * want.abs() + 2.0 ** -17 * torch.maximum(size, want.abs()) + (2.0 ** -25 if dtype == F16 else 0)
        worst = ((have.double().cpu() - want).abs() - bar).max().item()
        assert worst <= 0.0, worst
    check(got[:T], q, gains.get("q"))
    check(pool.k.flatten(0, 1)[rows], k, gains.get("k"))
    assert torch.equal(pool.v.flatten(0, 1)[rows], v[:T])
    assert not bool(got[T:].any())
    pool.planes.flatten(1, 2)[:, rows] = before.flatten(1, 2)[:, rows]
    assert torch.equal(pool.planes, before)  # nothing else changed


@pytest.mark.gpu
def test_append_depths_places_and_tables(dev):
    """Positions of a tree, tokens without room or a page, positions outside the tables."""
    torch.manual_seed(5)
    pool = Pool(dev, BF, [30, 20], 16, 2, 64, wide=0)
    pool.planes.normal_()
    before = pool.planes.clone()
    q, k, v = (torch.randn(14, h, 64).to(BF).to(dev) for h in (4, 2, 2))
    depths = ints([0, 1, 1, 2, 2, 3, -20, 2 ** 31 - 1, 0, 1, 2, 3, 4, 5], dev)
    pool.table[1, 1] = len(pool.k)
    past, cu = ints([29, 10], dev), ints([0, 8, 14], dev)  # rows 3 and on of the first have no room
    cos, sin = (t.to(dev) for t in tables(31, 64))
    got = paged_append(q, k, v, pool.k, pool.v, pool.table, past, cu, cos, sin, depths=depths)
    at = torch.cat([29 + depths[:8].long().cpu(), 10 + depths[8:].long().cpu()])
    want, size = exact_rotary(q, cos, sin, at, False)
    assert torch.equal(got.isnan().cpu(), want.isnan()) and bool(want.isnan().any())
    bar = EPS[BF] * want.abs() + 2.0 ** -22 * size
    assert bool(((got.double().cpu() - want).abs() <= bar)[~want.isnan()].all())
    stored = torch.cat([pool.at(0, 29, 32), pool.at(1, 10, 16)])
    rows = torch.tensor([0, 1, 2, 8, 9, 10, 11, 12, 13], device=dev)
    assert torch.equal(pool.v.flatten(0, 1)[stored], v[rows])
    want, size = exact_rotary(k[rows], cos, sin, at[rows.cpu()], False)
    have = pool.k.flatten(0, 1)[stored].double().cpu()
    assert torch.equal(have.isnan(), want.isnan())
    assert bool(((have - want).abs() <= EPS[BF] * want.abs() + 2.0 ** -22 * size)[~want.isnan()].all())
    pool.planes.flatten(1, 2)[:, stored] = before.flatten(1, 2)[:, stored]
    assert torch.equal(pool.planes, before)


@pytest.mark.gpu
def test_append_strides(dev):
    torch.manual_seed(6)
    past, new = [20, 3], [9, 30]
    fused = torch.randn(39, 16, 96).to(BF).to(dev)
    q, k, v = fused[:, :8], fused[:, 8:12], fused[:, 12:]
    cos, sin = (t.to(dev) for t in tables(60, 96))
    res = []
    for how in range(4):
        pool = Pool(dev, BF, [29, 33], 16, 4, 96)
        pool.planes.zero_()
        ks, vs = pool.k, pool.v
        if how == 1:
            ks, vs = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (ks, vs))
        if how == 2:
            odd = [torch.empty(t.numel() + 1, dtype=BF, device=dev)[1:].view(t.shape).copy_(t) for t in (q, k, v)]
        if how == 3:
            odd = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
        xs = (q, k, v) if how < 2 else odd
        out = paged_append(*xs, ks, vs, pool.table, ints(past, dev), ints(starts(new), dev), cos, sin)
        res.append((out, ks, vs))
    for r in res[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, res[0]))


# -------------------------------------------------------------------- keeping

@pytest.mark.gpu
@pytest.mark.parametrize("past,new,page,planes,dtype", [
    ([0], [1], 16, 2, BF), ([5, 0, 30, 16], [7, 16, 0, 40], 16, 6, F16), ([100] * 70, [20] * 70, 64, 4, BF),
    ([9001], [64], 256, 48, torch.float32)])
def test_keep(dev, past, new, page, planes, dtype):
    rng = random.Random(3)
    pool = Pool(dev, dtype, [a + b for a, b in zip(past, new)], page, 2, 64, planes=planes)
    pool.planes.normal_()
    want, paths, kept = pool.planes.clone(), [], []
    for i, (a, b) in enumerate(zip(past, new)):
        path = sorted(rng.sample(range(b), rng.randint(1, b))) if b else []
        path = [0] + path[1:] if path else path
        src = pool.at(i, a, a + b)[path] if b else None
        if b:
            want.flatten(1, 2)[:, pool.at(i, a, a + len(path))] = pool.planes.flatten(1, 2)[:, src]
        paths += path + [-1] * (b - len(path))
        kept.append(len(path))
    new_lengths = paged_keep(pool.planes, pool.table, ints(past, dev), ints(starts(new), dev), ints(kept, dev), ints(paths, dev))
    assert torch.equal(pool.planes, want)
    assert new_lengths.tolist() == [a + b for a, b in zip(past, kept)]


@pytest.mark.gpu
def test_keep_senseless_paths_and_no_pages(dev):
    pool = Pool(dev, BF, [40], 16, 2, 64, planes=2, wide=0)
    pool.planes.normal_()
    before = pool.planes.clone()
    new = paged_keep(pool.planes, pool.table, ints([30], dev), ints([0, 8], dev), ints([99], dev),
                     ints([0, 0, 1, 8, 2 ** 31 - 1, -5, 6, 7], dev))
    assert torch.equal(pool.planes, before) and new.tolist() == [38]
    pool.table[0, 2] = -1  # keys 32 and on
    paged_keep(pool.planes, pool.table, ints([30], dev), ints([0, 8], dev), ints([4], dev), ints([1, 5, 6, 7, 0, 0, 0, 0], dev))
    pool.planes.flatten(1, 2)[:, pool.at(0, 30, 32)[:1]] = before.flatten(1, 2)[:, pool.at(0, 30, 32)[:1]]
    assert torch.equal(pool.planes, before)


# ------------------------------------------------------------------- refusals

@pytest.mark.gpu
def test_refusals(dev):
    """Wrong shapes, types and layouts raise, and write nothing."""
    from model.rotary import rotary
    from model.speculative import verify_drafts
    pool, q = make(dev, BF, [20, 5], [3, 2], 16, 4, 2, 64)
    k = torch.randn(5, 2, 64, device=dev).to(BF)
    cu, lens, table = ints([0, 3, 5], dev), ints([20, 5], dev), pool.table
    cos, sin = (t.to(dev) for t in tables(40, 64))
    before = pool.planes.clone()

    def app(q=q, k=k, v=k, kp=pool.k, vp=pool.v, table=table, lens=lens, cu=cu, cos=cos, sin=sin, **kw):
        return paged_append(q, k, v, kp, vp, table, lens, cu, cos, sin, **kw)

    def att(q=q, kp=pool.k, vp=pool.v, table=table, lens=lens, cu=cu, **kw):
        return paged_attention(q, kp, vp, table, lens, cu, **kw)
    odd = torch.empty(2 * 6 * 16 * 2 * 64 + 1, dtype=BF, device=dev)[1:].view(2, 6, 16, 2, 64)
    grad = q.clone().requires_grad_()
    wide = torch.zeros(6, 16, 2, 68, dtype=BF, device=dev)[..., :64]
    bad = [
        lambda: app(q=q.float()), lambda: app(k=k.to(F16)), lambda: app(v=k[:4]), lambda: app(q=q[:, :, :32]),
        lambda: app(lens=lens.long()), lambda: app(lens=lens[:1]), lambda: app(cu=cu.cpu()), lambda: app(table=table[:1]),
        lambda: app(table=table.long()), lambda: app(table=table[0]), lambda: app(cos=cos[0]), lambda: app(cos=cos[:, :16]),
        lambda: app(sin=sin.to(BF)), lambda: app(depths=ints([0, 1], dev)), lambda: app(q_gain=torch.ones(32, device=dev)),
        lambda: app(kp=odd[0], vp=odd[1]), lambda: app(kp=pool.k[:, :8], vp=pool.v[:, :8]), lambda: app(vp=pool.v[:2]),
        lambda: app(kp=wide, vp=wide), lambda: app(q=grad), lambda: app(kp=pool.k.float(), vp=pool.v.float()),
        lambda: att(q=q.float()), lambda: att(q=grad), lambda: att(q=q[:, :3]), lambda: att(q=q[0]), lambda: att(scale=0.0),
        lambda: att(scale=-1.0), lambda: att(scale=math.nan), lambda: att(tree=torch.ones(5, 1, dtype=torch.int32, device=dev)),
        lambda: att(tree=torch.ones(4, 1, dtype=torch.int64, device=dev)), lambda: att(tree=torch.ones(5, 0, dtype=torch.int64, device=dev)),
        lambda: att(tree=torch.ones(5, 1, dtype=torch.int64)), lambda: att(kp=pool.k[..., :32], vp=pool.v[..., :32]),
        lambda: paged_keep(pool.planes[:, ::2], table, lens, cu, lens, lens), lambda: paged_keep(pool.k, table, lens, cu, lens, lens),
        lambda: paged_keep(pool.planes, table, lens, cu, lens.long(), lens),
        lambda: paged_keep(pool.planes[..., :1].contiguous()[..., :1, :], table, lens, cu, lens, lens),
        lambda: rotary(q, k.float(), cos, sin, torch.arange(5, device=dev)), lambda: rotary(q, k[:4], cos, sin, torch.arange(5, device=dev)),
        lambda: rotary(q, k, cos, sin, torch.arange(4, device=dev)), lambda: rotary(q, k, cos, sin, torch.arange(5, device=dev).float()),
        lambda: rotary(q, k, cos.repeat(1, 2), sin.repeat(1, 2), torch.arange(5, device=dev)),
        lambda: rotary(q, k, cos.clone().requires_grad_(), sin, torch.arange(5, device=dev)),
        lambda: rotary(q.double(), None, cos, sin, torch.arange(5, device=dev)),
    ]
    p, t = torch.rand(5, 9, device=dev), torch.zeros(5, dtype=torch.int64, device=dev)
    bad += [lambda: verify_drafts(p[0], t, cu), lambda: verify_drafts(p.double(), t, cu), lambda: verify_drafts(p, t.int(), cu),
            lambda: verify_drafts(p, t[:4], cu), lambda: verify_drafts(p, t, cu, parents=t), lambda: verify_drafts(p, t, cu, draft_probs=p),
            lambda: verify_drafts(p, t, cu, draft_probs=p[:, :8], uniforms=p[:, 0]), lambda: verify_drafts(p, t, cu.long()),
            lambda: verify_drafts(p, t, cu, uniforms=t), lambda: verify_drafts(p, t, cu, uniforms=p[:4, 0])]
    for i, f in enumerate(bad):
        with pytest.raises((TypeError, ValueError, RuntimeError), match="mhc_amd"):
            f()
            print("not refused:", i)
    assert torch.equal(pool.planes.isnan(), before.isnan()) and torch.equal(pool.planes.nan_to_num(), before.nan_to_num())
