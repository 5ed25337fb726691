"""Drafting and verifying through the model on the GPU: prompts, steps and trees over a cache of
pages against each sequence alone, whole steps one after another, captured graphs, side streams,
other rotary layouts in training."""
from __future__ import annotations

import copy
import random

import pytest
import torch

from model import model_minimind, paged
from model.model_minimind import MiniMindConfig, MiniMindForCausalLM, init_normal_
from model.packed import PackedBatch
from model.paged import DraftTree, PagedCache
from model.speculative import verify_drafts

BF, F16 = torch.bfloat16, torch.float16


def _model(dev, dtype=BF, **kw):
    torch.manual_seed(0)
    cfg = MiniMindConfig(hidden_size=192, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                         head_dim=64, intermediate_size=256, vocab_size=500, max_position_embeddings=512,
                         **{"use_mhc": 1, **kw})
    return init_normal_(MiniMindForCausalLM(cfg), 0.05).to(dev).to(dtype)


def _far(got, ref):
    return float((got.double() - ref.double()).norm() / ref.double().norm())


def _taken(monkeypatch):
    """Counts the calls of the paged kernels."""
    seen = []
    for name in ("paged_append", "paged_attention"):
        run = getattr(paged, name)
        monkeypatch.setattr(paged, name, lambda *a, run=run, **k: seen.append(1) or run(*a, **k))
    return seen


def _batch(lengths, dev, rows=None):
    return PackedBatch.from_lengths(lengths, rows, device=dev)


def random_trees(lengths, seed):
    rng = random.Random(seed)
    return [[-1] + [rng.randrange(max(0, j - 3), j) for j in range(1, n)] for n in lengths]


@pytest.mark.gpu
@pytest.mark.parametrize("kw,page", [({}, 16), ({"rotary_dim": 32}, 64), ({"rope_interleaved": True}, 16),
                                     ({"rotary_dim": 24, "rope_interleaved": True, "use_mhc": 0}, 32),
                                     ({"use_moe": True, "num_experts": 1}, 16)])
def test_prompts_and_steps(dev, monkeypatch, kw, page):
    """As far from the fp32 model as the sequences alone are, twice over: both round the same steps
    to bf16, in kernels that differ."""
    m = _model(dev, **kw).eval()
    wide = copy.deepcopy(m).float()
    lengths, steps = [40, 3, 129, 1], 4
    ids = [torch.randint(0, 500, (n + steps,), device=dev) for n in lengths]
    cache = PagedCache(m.config, 4, 160, page, device=dev)
    seen = _taken(monkeypatch)
    with torch.inference_mode():
        out = m(torch.cat([x[:n] for x, n in zip(ids, lengths)] + [ids[0][:2]])[None],
                packed=_batch(lengths, dev, sum(lengths) + 2), past_key_values=cache)
        last = [o[-1:] for o in out.logits[0, :-2].split(lengths)]
        step = _batch([1] * 4, dev)
        for i in range(steps):
            out = m(torch.stack([x[n + i] for x, n in zip(ids, lengths)])[None], packed=step, past_key_values=cache)
            last = [torch.cat([a, o[None]]) for a, o in zip(last, out.logits[0])]
        assert len(seen) == 4 * (1 + steps) and cache.lengths.tolist() == [n + steps for n in lengths]
        for x, n, got in zip(ids, lengths, last):
            ref = wide(x[None]).logits[0, n - 1:]
            assert _far(got, ref) <= 2 * _far(m(x[None]).logits[0, n - 1:], ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cache_dtype", [(BF, BF), (F16, F16), (torch.float32, BF), (BF, torch.float32)])
def test_trees_and_kept_branches(dev, monkeypatch, dtype, cache_dtype):
    """A tree's rows against their branches alone, and the next tree behind the branch that is kept.
    A model of another type than its cache rounds more than the sequences alone do: its distance is
    bounded by that of the bf16 model."""
    m = _model(dev, dtype).eval()
    low = m if dtype in (BF, F16) and cache_dtype == dtype else copy.deepcopy(m).to(BF)
    wide = copy.deepcopy(m).float()
    cache = PagedCache(m.config, 3, 200, 16, dtype=cache_dtype, device=dev)
    seen = _taken(monkeypatch)
    tokens = [torch.randint(0, 500, (n,), device=dev) for n in (50, 7, 100)]
    with torch.inference_mode():
        m(torch.cat(tokens)[None], packed=_batch([50, 7, 100], dev), past_key_values=cache)
        for turn in range(3):
            sizes = [[9, 17, 1], [1, 2, 40], [5, 5, 5]][turn]
            b, trees = _batch(sizes, dev), random_trees(sizes, turn)
            ids = torch.randint(0, 500, (b.rows,), device=dev)
            up = torch.tensor(sum(trees, []), dtype=torch.int32, device=dev)
            got = m(ids[None], packed=b, past_key_values=cache, drafts=DraftTree(b, up)).logits[0]
            at, kept, path, far, alone = 0, [], [], 0.0, 0.0
            for s, parents in enumerate(trees):
                branches = []
                for j, p in enumerate(parents):
                    branches.append((branches[p] if p >= 0 else []) + [j])
                for j in (0, len(parents) // 2, len(parents) - 1):
                    full = torch.cat([tokens[s], ids[at:at + len(parents)][branches[j]]])[None]
                    ref = wide(full).logits[0, -1].double()
                    far += float((got[at + j].double() - ref).square().sum())
                    alone += float((low(full).logits[0, -1].double() - ref).square().sum())
                keep = branches[-1]
                tokens[s] = torch.cat([tokens[s], ids[at:at + len(parents)][keep]])
                kept.append(len(keep))
                path += keep + [-1] * (len(parents) - len(keep))
                at += len(parents)
            assert far <= 4 * alone
            cache.keep(b, torch.tensor(kept, dtype=torch.int32, device=dev), torch.tensor(path, dtype=torch.int32, device=dev))
            assert cache.lengths.tolist() == [len(t) for t in tokens]
            cache.settle()
        assert len(seen) == (16 if cache_dtype in (BF, F16) else 0)


@pytest.mark.gpu
@pytest.mark.parametrize("sampled", [False, True])
def test_verify_steps_together(dev, sampled):
    """Steps as they are used: append, attention, verification and keeping, one after another.  Each
    verdict is that of verify_drafts on the step's own logits, and the cache then holds the kept tokens: the
    logits of a last step are as near to the fp32 model on them as the sequences alone are, twice over."""
    m = _model(dev).eval()
    wide = copy.deepcopy(m).float()
    cache = PagedCache(m.config, 3, 300, 16, device=dev)
    tokens = [torch.randint(0, 500, (n,), device=dev) for n in (30, 2, 61)]
    rng = random.Random(1)
    with torch.inference_mode():
        m(torch.cat([t[:-1] for t in tokens])[None], packed=_batch([29, 1, 60], dev), past_key_values=cache)
        for turn in range(4):
            sizes = [rng.randint(1, 9) for _ in tokens]
            b, trees = _batch(sizes, dev), random_trees(sizes, turn)
            ids, at = torch.randint(0, 500, (b.rows,), device=dev), 0
            for s, n in enumerate(sizes):
                ids[at] = tokens[s][-1]
                if n > 1 and not sampled:  # a first draft that is right
                    ids[at + 1] = m(tokens[s][None]).logits[0, -1].argmax()
                at += n
            up = torch.tensor(sum(trees, []), dtype=torch.int32, device=dev)
            draft = torch.full((b.rows, 500), 1 / 500, device=dev) if sampled else None
            u = torch.rand(b.rows, device=dev) * 0.3 if sampled else None
            res = m.verify_step(ids[None], b, cache, up, draft, u, temperature=0.8)
            probs = res.logits[0] if u is None else torch.softmax(res.logits[0].float() / 0.8, -1)
            want = verify_drafts(probs, ids, b.cu_seqlens, up, draft, u)
            assert all(torch.equal(x, y) for x, y in zip((res.kept, res.path, res.next_tokens), want))
            at = 0
            for s, n in enumerate(sizes):
                nodes = [x for x in res.path[at:at + n].tolist() if x >= 0]
                tokens[s] = torch.cat([tokens[s], ids[at:at + n][nodes[1:]], res.next_tokens[s:s + 1]])
                at += n
            assert cache.lengths.tolist() == [len(t) - 1 for t in tokens]
        got = m(torch.stack([t[-1] for t in tokens])[None], packed=_batch([1] * 3, dev), past_key_values=cache).logits[0]
        for s, t in enumerate(tokens):
            ref = wide(t[None]).logits[0, -1]
            assert _far(got[s], ref) <= 2 * _far(m(t[None]).logits[0, -1], ref)


@pytest.mark.gpu
def test_captured_verify_step(dev):
    """A whole step in a graph, replayed with other tokens, trees and lengths, eager work between: each
    replay gives what the eager step on a copy of the cache gives."""
    m = _model(dev).eval()
    cache, other = (PagedCache(m.config, 2, 400, 16, device=dev) for _ in range(2))
    sizes = [6, 4]
    b = _batch(sizes, dev)
    g = torch.Generator(device=dev).manual_seed(3)
    new = lambda: (torch.randint(0, 500, (10,), generator=g, device=dev), torch.rand(10, generator=g, device=dev))
    ids, u = new()
    up = torch.tensor(sum(random_trees(sizes, 0), []), dtype=torch.int32, device=dev)
    with torch.inference_mode():
        prompt = torch.randint(0, 500, (1, 50), device=dev)
        for c in (cache, other):
            m(prompt, packed=_batch([30, 20], dev), past_key_values=c)
            c.reserve(100)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m.verify_step(ids[None], b, other, up, None, u)
        torch.cuda.current_stream().wait_stream(side)
        other.planes.copy_(cache.planes)
        other.lengths.copy_(cache.lengths)
        other.page_table.copy_(cache.page_table)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = m.verify_step(ids[None], b, cache, up, None, u)
        for turn in range(5):
            a, c = new()
            ids.copy_(a)
            u.copy_(c * (0.02 if turn % 2 else 1.0))
            up.copy_(torch.tensor(sum(random_trees(sizes, turn + 5), []), dtype=torch.int32))
            graph.replay()
            torch.cuda.synchronize()
            want = m.verify_step(ids[None], b, other, up, None, u)
            for x, y in ((res.kept, want.kept), (res.path, want.path), (res.next_tokens, want.next_tokens),
                         (res.logits, want.logits), (cache.lengths, other.lengths), (cache.planes, other.planes)):
                assert torch.equal(x, y), turn


@pytest.mark.gpu
def test_two_captured_graphs_and_a_side_stream(dev):
    """Graphs of two calls replayed at once on two streams do not share a workspace."""
    torch.manual_seed(2)
    from model.paged import paged_attention
    calls = []
    for i in range(2):
        q = torch.randn(12, 8, 96, device=dev).to(BF)
        k, v = (torch.randn(200, 16, 4, 96, device=dev).to(BF) for _ in range(2))
        table = torch.randperm(200, device=dev)[:198].to(torch.int32).view(3, 66)
        lens = torch.tensor([1000, 5, 700], dtype=torch.int32, device=dev)
        cu = torch.tensor([0, 4, 8, 12], dtype=torch.int32, device=dev)
        calls.append((q, k, v, table, lens, cu))
    want = [paged_attention(*c) for c in calls]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for c in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(paged_attention(*c))
    for _ in range(10):
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    with torch.cuda.stream(streams[0]):
        eager = paged_attention(*calls[1])
    streams[0].synchronize()
    assert torch.equal(eager, want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [{"rotary_dim": 32}, {"rope_interleaved": True}])
@pytest.mark.parametrize("packed", [False, True])
def test_training_with_other_pairs(dev, monkeypatch, kw, packed):
    """Losses and gradients of a training step under autocast: as far from the fp32 step as the
    same step with its rotation on torch ops is, twice over."""
    m = _model(dev, torch.float32, **kw).train()
    ids = torch.randint(0, 500, (1 if packed else 2, 60), device=dev)
    seen = []

    def step(model, x, where):
        more = {"packed": PackedBatch.from_lengths([20, 33, 7], device=where)} if packed else {}
        loss = model(x, labels=x, **more).loss
        grads = torch.autograd.grad(loss, list(model.parameters()))
        return loss.detach().cpu(), torch.cat([t.flatten() for t in grads]).cpu()
    run = model_minimind.rotary
    monkeypatch.setattr(model_minimind, "rotary", lambda *a, **k: seen.append(1) or run(*a, **k))
    with torch.autocast("cuda", BF):
        got = step(m, ids, dev)
    assert len(seen) == 2
    monkeypatch.setattr(model_minimind, "rotary", model_minimind.plain_rotary)
    with torch.autocast("cuda", BF):
        plain = step(m, ids, dev)
    ref = step(m, ids, dev)
    assert abs(float(got[0] - ref[0])) <= 2 * abs(float(plain[0] - ref[0])) + 2.0 ** -6
    assert _far(got[1], ref[1]) <= 2 * _far(plain[1], ref[1])
