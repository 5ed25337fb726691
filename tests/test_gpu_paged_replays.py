"""Captured steps over a cache of pages: rounds of reserving and replaying, and eager calls between them, against a
cache that only eager calls have filled."""
from __future__ import annotations

import pytest
import torch

from model.packed import PackedBatch
from model.paged import PagedCache
from test_gpu_paged_model import _model


def same(cache, other):
    """The sequences' keys and values in both caches, whatever their pages."""
    assert torch.equal(cache.lengths, other.lengths)
    for s, n in enumerate(other.lengths.tolist()):
        key = torch.arange(n, device=cache.lengths.device)
        a, b = (c.planes.flatten(1, 2)[:, c.rows_of(torch.full_like(key, s), key)] for c in (cache, other))
        assert torch.equal(a, b), s


@pytest.mark.gpu
def test_rounds_of_reserve_replays_and_eager_calls(dev):
    m = _model(dev).eval()
    cache, other = (PagedCache(m.config, 2, 400, 16, pages=50, device=dev) for _ in range(2))
    g = torch.Generator(device=dev).manual_seed(3)
    ids = lambda n: torch.randint(0, 500, (1, n), generator=g, device=dev)
    one, token = PackedBatch.from_lengths([1, 1], device=dev), ids(2)
    prompt, chunk = PackedBatch.from_lengths([30, 3], device=dev), PackedBatch.from_lengths([0, 20], device=dev)
    first, more = ids(33), ids(20)
    with torch.inference_mode():
        for c in (cache, other):
            m(first, packed=prompt, past_key_values=c)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # warm up on the cache that is not captured
            m(token, packed=one, past_key_values=other)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        other.lengths.copy_(cache.lengths)
        other.settle()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(token, packed=one, past_key_values=cache)
        for turn in range(3):
            cache.reserve(18)
            for _ in range(18):
                token.copy_(ids(2))
                graph.replay()
                want = m(token, packed=one, past_key_values=other)
                torch.cuda.synchronize()
                assert torch.equal(out.logits, want.logits), turn
            got, want = (m(more, packed=chunk, past_key_values=c) for c in (cache, other))
            assert torch.equal(got.logits, want.logits), turn
            same(cache, other)
        assert cache.lengths.tolist() == [84, 117] and [len(x) for x in cache.owned] == [6, 8]


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["greedy", "certain", "draft", "wide draft"])
def test_verify_step_of_a_64_bit_model(dev, mode):
    """What the kernel does not take is verified on the host; the results are on the GPU, as ever."""
    from model.speculative import plain_verify
    dtype = torch.float32 if mode == "wide draft" else torch.float64
    m = _model(dev, dtype, use_mhc=0).eval()
    cache = PagedCache(m.config, 2, 100, 16, dtype=dtype, device=dev)
    b = PackedBatch.from_lengths([5, 3], device=dev)
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(0, 500, (1, 8), generator=g).to(dev)
    u = None if mode == "greedy" else torch.rand(8, generator=g).to(dev)
    draft = torch.full((8, 500), 1 / 500, dtype=torch.float64, device=dev) if "draft" in mode else None
    with torch.inference_mode():
        m(ids[:, :7], packed=PackedBatch.from_lengths([4, 3], device=dev), past_key_values=cache)
        res = m.verify_step(ids, b, cache, None, draft, u)
        host = lambda t: None if t is None else t.cpu()
        logits = res.logits[0]
        probs = logits if u is None else torch.softmax(logits.float(), -1)
        want = plain_verify(host(probs), ids[0].cpu(), b.cu_seqlens.cpu(), None, host(draft), host(u))
    for got, w in zip((res.kept, res.path, res.next_tokens), want):
        assert got.device == dev and got.dtype == w.dtype and torch.equal(got.cpu(), w)
    assert cache.lengths.tolist() == [4 + int(want[0][0]), 3 + int(want[0][1])]


@pytest.mark.gpu
def test_rounds_of_captured_verify_steps(dev):
    """Whole steps with drafts in a graph, reserved for and settled between rounds, against eager steps on a cache whose
    host count is only a bound; both end where the pages do."""
    m = _model(dev).eval()
    cache, other = (PagedCache(m.config, 2, 160, 16, pages=14, device=dev) for _ in range(2))
    g = torch.Generator(device=dev).manual_seed(5)
    draw = lambda n: torch.randint(0, 500, (1, n), generator=g, device=dev)
    b, prompt = PackedBatch.from_lengths([4, 4], device=dev), PackedBatch.from_lengths([40, 9], device=dev)
    ids, u, first = draw(8), torch.rand(8, generator=g, device=dev), draw(49)
    with torch.inference_mode():
        for c in (cache, other):
            m(first, packed=prompt, past_key_values=c)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m.verify_step(ids, b, other, None, None, u)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        other.lengths.copy_(cache.lengths)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(RuntimeError, match="captured"):
                cache.reserve(4)
            res = m.verify_step(ids, b, cache, None, None, u)
        for turn in range(12):
            cache.reserve(12)  # three steps of four nodes at most
            for _ in range(3):
                ids.copy_(draw(8))
                u.copy_(torch.rand(8, generator=g, device=dev) * (0.005 if turn % 3 else 1.0))
                graph.replay()
                want = m.verify_step(ids, b, other, None, None, u)
                torch.cuda.synchronize()
                assert torch.equal(res.logits, want.logits) and torch.equal(res.next_tokens, want.next_tokens), turn
            same(cache, other)
            if turn % 2:
                cache.settle(spare=0)
        longest = max(cache.lengths.tolist())
        assert longest > 76
        for c in (cache, other):  # what does not fit is refused, by its true length
            with pytest.raises(ValueError, match=f"{longest} . {161 - longest} keys may not fit"):
                c.reserve([161 - longest] * 2 if c.lengths[0] >= c.lengths[1] else [0, 161 - longest])
