"""Packed sequences on the GPU, where a call's sequences, rows, types and lengths are not the
usual ones: values that are not finite, rows behind the last sequence, caches of another
type, gradients of very different sizes."""
from __future__ import annotations

import math

import pytest
import torch

from model.packed import PackedBatch

BF, F16 = torch.bfloat16, torch.float16


@pytest.mark.gpu
def test_sums_of_sequences(dev):
    """Each sequence's by itself, the same bits in a replayed graph, and their gradient."""
    lengths = [700, 0, 1, 2048, 333]
    b = PackedBatch.from_lengths(lengths, rows=sum(lengths) + 9, device=dev)
    torch.manual_seed(0)
    x = (-10.0 * torch.rand(b.rows, device=dev)).requires_grad_()
    w = torch.tensor([1.0, 2.0, 3.0, 4.0, 5.0], dtype=torch.float64, device=dev)
    want = torch.stack([t.double().cpu().sum() for t in x.detach()[:-9].split(lengths)])
    got = b.sums(x)
    torch.testing.assert_close(got.detach().cpu(), want, rtol=2048 * 2.0 ** -53, atol=0.0)
    g, = torch.autograd.grad(got, x, w)
    assert torch.equal(g, torch.cat([w.repeat_interleave(torch.tensor(lengths, device=dev)), w.new_zeros(9)]).float())
    y = x.detach().clone()
    y[800] = -math.inf
    y[-20] = math.nan
    s = b.sums(y).cpu()
    assert torch.equal(s[:3], got.detach().cpu()[:3]) and s[3] == -math.inf and s[4].isnan()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.sums(y)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b.sums(y)
    for i in range(4):
        y.copy_(x.detach() * (i + 1))
        eager = b.sums(y)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
