"""More of the operators on a cache of pages: how near outputs are to the formula whatever the
number of rows, and bounds that make no sense."""
from __future__ import annotations

import pytest
import torch

from model import _hip as H
from model.paged import paged_attention
from test_gpu_paged import BF, EPS, F16, close, exact, ints, make, random_tree, starts


@pytest.mark.gpu
@pytest.mark.parametrize("hd,heads,kv,page,past,new", [
    (96, 8, 4, 16, [30], [1]), (96, 8, 4, 16, [30], [9]), (64, 4, 4, 16, [20, 70], [40, 50]), (128, 16, 2, 64, [40], [64]),
    (96, 8, 4, 16, [50, 3], [100, 70]), (64, 8, 1, 16, [300], [33]), (128, 4, 2, 16, [700], [150])])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("tree", [False, True])
def test_probabilities_lose_nothing_to_16_bits(dev, hd, heads, kv, page, past, new, dtype, tree):
    """The outputs are rounded once, and nothing before them to 16 bits alone.  A probability is two 16-bit
    operands, off by at most EPS^2 <= 2^-16 of itself.  Its score is a sum of head_dim <= 128 products in fp32: with these
    inputs it stays under 32 (five standard deviations of 0.375 x 1.5 x 128^0.5), so each step rounds by 2^-19 at
    most; at random, three standard deviations of 128 steps are 20 x 2^-19, and times 0.11 log2 e they move the
    probability by less than 2^-17 of itself.  Both together, in the row's sum too: 2^-14 of the terms' sizes."""
    pool, q = make(dev, dtype, past, new, page, heads, kv, hd)
    q /= 4  # scores of some units: many keys count in each row
    bits, sees = random_tree(new, 3) if tree else (None, None)
    got = paged_attention(q, pool.k, pool.v, pool.table, ints(past, dev), ints(starts(new), dev),
                          tree=None if bits is None else bits.to(dev), scale=0.11).double().cpu()
    out, size = exact(pool, q, past, new, 0.11, sees)
    bar = EPS[dtype] * out.abs() + 2.0 ** -14 * size + (2.0 ** -25 if dtype == F16 else 0.0)
    worst = ((got - out).abs() - bar).max().item()
    assert worst <= 0.0, worst


@pytest.mark.gpu
@pytest.mark.parametrize("record", [
    (-2 ** 30, 2 ** 26, 1, 2), (-2 ** 31, 0, 1, 2 ** 31 - 1), (0, -1000, 1, 5), (2 ** 31 - 1, 3, 2, 2), (0, 2 ** 31 - 1, 2 ** 31 - 1, 9),
    (0, 5, 0, 3), (0, 5, -7, 3), (0, 5, 2 ** 31 - 1, 2 ** 31 - 1), (0, 0, 1, -1), (0, 0, 1, 2 ** 31 - 1)])
def test_bounds_that_decrease_read_nothing_outside_the_workspace(dev, record):
    """Sequence 1 begins behind its end: no workgroup writes its record for the join, which rows 0 to 29 come out
    at.  Whatever stands there, NaN before and behind the workspace does not reach an output."""
    heads, kv, hd, page, width, cu = 8, 4, 64, 16, 64, [0, 40, 0, 30]
    T, B = 45, 3
    torch.manual_seed(0)
    q = torch.randn(T, heads, hd, device=dev).to(BF)
    k, v = (torch.randn(B * width, page, kv, hd, device=dev).to(BF) for _ in range(2))
    table = torch.arange(B * width, dtype=torch.int32, device=dev).view(B, width)
    lens, cu = ints([900] * B, dev), ints(cu, dev)
    lib = H.load()
    nbytes = lib.mhc_paged_attn_workspace_bytes(B, T, heads, kv, hd)
    assert nbytes > 0 and nbytes % 16 == 0
    room = 1 << 20  # floats before and behind
    buf = torch.full((2 * room + nbytes // 4,), float("nan"), device=dev)
    ws = buf[room:room + nbytes // 4]
    ws.zero_()
    ws.view(torch.int32)[-4 * B:].view(B, 4).copy_(ints([record] * B, dev))
    out = torch.full_like(q, 7.0)
    assert lib.mhc_paged_attn_fwd(
        q.data_ptr(), heads * hd, hd, k.data_ptr(), v.data_ptr(), page * kv * hd, kv * hd, hd, table.data_ptr(), lens.data_ptr(),
        cu.data_ptr(), None, 0, out.data_ptr(), ws.data_ptr(), nbytes, B, T, heads, kv, hd, width, B * width, page, 1, 0.1,
        H.stream(dev)) == 0
    assert bool(torch.isfinite(out).all())
    assert bool(buf[:room].isnan().all()) and bool(buf[room + nbytes // 4:].isnan().all())


@pytest.mark.gpu
def test_workspace_sizes_are_kept_for_each_device(dev, monkeypatch):
    """The split follows the device's compute units: a size that one device was asked for is not another's."""
    from model import paged
    seen, ask = [], paged._workspace
    monkeypatch.setattr(paged, "_workspace", lambda *a: seen.append(a) or ask(*a))
    pool, q = make(dev, BF, [900], [1], 16, 8, 4, 96)
    paged_attention(q, pool.k, pool.v, pool.table, ints([900], dev), ints([0, 1], dev))
    assert seen == [(dev.index, 1, 1, 8, 4, 96)]


@pytest.mark.gpu
@pytest.mark.parametrize("past,new", [
    ([3000] + [i % 40 for i in range(255)], [1] * 256), ([i % 40 for i in range(199)] + [3000] + [5] * 60, [1] * 260),
    ([700, 90, 0, 1500, 33] * 4, [1, 1, 200, 1, 1] * 4), ([20, 500] * 3 + [900], [1, 2] * 3 + [400]),
    ([i % 70 for i in range(290)], [1] * 100 + [130] + [1] * 100 + [0] * 60 + [3] * 29)])
@pytest.mark.parametrize("tree", [False, True])
def test_sequences_that_are_not_alike(dev, past, new, tree):
    """One long sequence among many short ones, on both sides of 256; single tokens and chunks in one call."""
    pool, q = make(dev, BF, past, new, 16, 8, 4, 64)
    bits, sees = random_tree(new, 5) if tree else (None, None)
    got = paged_attention(q, pool.k, pool.v, pool.table, ints(past, dev), ints(starts(new), dev),
                          tree=None if bits is None else bits.to(dev), scale=0.11)
    close(got, exact(pool, q, past, new, 0.11, sees), BF)
