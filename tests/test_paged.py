"""The cache of pages, drafted trees and their verification through the model on the CPU (torch
ops), and the refusals of the operators that need no GPU."""
from __future__ import annotations

import random

import pytest
import torch

from model.model_minimind import MiniMindConfig, MiniMindForCausalLM, init_normal_
from model.packed import PackedBatch, PackedCache
from model.paged import DraftTree, PagedCache, paged_append, paged_attention, paged_keep
from model.rotary import plain_rotary, rotary
from model.speculative import plain_verify, verify_drafts


def tiny(**more):
    torch.manual_seed(0)
    args = dict(hidden_size=64, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, vocab_size=50,
                intermediate_size=96, max_position_embeddings=128)
    return init_normal_(MiniMindForCausalLM(MiniMindConfig(**{**args, **more})), 0.3).eval()


def batch(lengths, rows=None):
    return PackedBatch.from_lengths(lengths, rows, device="cpu")


def pages(model, n, capacity=64, **more):
    return PagedCache(model.config, n, capacity, page=16, dtype=torch.float32, device="cpu", **more)


@pytest.mark.parametrize("more", [{}, {"rotary_dim": 8}, {"rope_interleaved": True}, {"rotary_dim": 4, "rope_interleaved": True},
                                  {"use_moe": True}])
def test_prompts_and_steps_as_without_a_cache(more):
    model = tiny(**more)
    prompts = [torch.randint(0, 50, (n,)) for n in (20, 1, 33)]
    cache = pages(model, 3)
    with torch.no_grad():
        got = model(torch.cat(prompts)[None], packed=batch([20, 1, 33]), past_key_values=cache).logits[0]
        want = [model(p[None]).logits[0] for p in prompts]
        assert torch.allclose(got, torch.cat(want), atol=1e-4)
        for _ in range(3):
            new = torch.randint(0, 50, (3,))
            got = model(new[None], packed=batch([1, 1, 1]), past_key_values=cache).logits[0]
            prompts = [torch.cat([p, t[None]]) for p, t in zip(prompts, new)]
            want = torch.stack([model(p[None]).logits[0, -1] for p in prompts])
            assert torch.allclose(got, want, atol=1e-4)
    assert cache.lengths.tolist() == [23, 4, 36] == cache.most


def test_a_tree_sees_its_branches_and_keep_goes_on_with_one():
    model = tiny()
    prompts = [torch.randint(0, 50, (n,)) for n in (15, 4)]
    parents = [[-1, 0, 0, 1, 2, 2, 4], [-1, 0, 1]]
    cache = pages(model, 2)
    flat = torch.tensor(sum(parents, []), dtype=torch.int32)
    with torch.no_grad():
        model(torch.cat(prompts)[None], packed=batch([15, 4]), past_key_values=cache)
        ids, b = torch.randint(0, 50, (10,)), batch([7, 3])
        tree = DraftTree(b, flat)
        assert tree.depths.tolist() == [0, 1, 1, 2, 2, 2, 3, 0, 1, 2]
        assert tree.mask[:, 0].tolist() == [1, 3, 5, 11, 21, 37, 85, 1, 3, 7]
        got = model(ids[None], packed=b, past_key_values=cache, drafts=tree).logits[0]
        assert cache.lengths.tolist() == [15, 4]
        for s, (at, ps) in enumerate(zip((0, 7), parents)):
            for j in range(len(ps)):
                branch, k = [], j
                while k >= 0:
                    branch.insert(0, k)
                    k = ps[k]
                full = torch.cat([prompts[s], ids[at:at + len(ps)][branch]])
                assert torch.allclose(got[at + j], model(full[None]).logits[0, -1], atol=1e-4)
        cache.keep(b, torch.tensor([4, 1], dtype=torch.int32),
                   torch.tensor([0, 2, 4, 6, -1, -1, -1, 0, -1, -1], dtype=torch.int32))
        assert cache.lengths.tolist() == [19, 5] and cache.most == [22, 7]
        cache.settle()
        assert cache.most == [19, 5] and [len(x) for x in cache.owned] == [2, 1]
        kept = [torch.cat([prompts[0], ids[[0, 2, 4, 6]]]), torch.cat([prompts[1], ids[7:8]])]
        new = torch.randint(0, 50, (2,))
        got = model(new[None], packed=batch([1, 1]), past_key_values=cache).logits[0]
        for s in range(2):
            assert torch.allclose(got[s], model(torch.cat([kept[s], new[s:s + 1]])[None]).logits[0, -1], atol=1e-4)


def test_greedy_decoding_with_drafts_is_greedy_decoding():
    """Whatever is drafted, the tokens are those of one step after another."""
    model = tiny(rope_interleaved=True)
    prompts = [torch.randint(0, 50, (n,)) for n in (9, 3)]
    rng = random.Random(0)
    with torch.no_grad():
        want = []
        for p in prompts:
            for _ in range(14):
                p = torch.cat([p, model(p[None]).logits[0, -1:].argmax(-1)])
            want.append(p)
        cache = pages(model, 2)
        model(torch.cat([p[:-1] for p in prompts])[None], packed=batch([8, 2]), past_key_values=cache)
        have = [p.clone() for p in prompts]
        while min(len(h) for h in have) < 17:
            n = [rng.randint(1, 6) for _ in have]
            parents = sum(([-1] + [rng.randrange(max(0, j - 2), j) for j in range(1, k)] for k in n), [])
            ids, at = [], 0
            for s, k in enumerate(n):
                row = [int(have[s][-1])]
                depth = [0]
                for j in range(1, k):
                    d = depth[parents[at + j]] + 1
                    depth.append(d)
                    there = len(have[s]) - 1 + d
                    right = int(want[s][there]) if there < len(want[s]) else 0
                    row.append(right if rng.random() < 0.7 else rng.randrange(50))
                ids += row
                at += k
            b = batch(n)
            res = model.verify_step(torch.tensor(ids)[None], b, cache, parents=torch.tensor(parents, dtype=torch.int32))
            at = 0
            for s, k in enumerate(n):
                nodes = [x for x in res.path[at:at + k].tolist() if x >= 0]
                assert len(nodes) == int(res.kept[s])
                have[s] = torch.cat([have[s], torch.tensor([ids[at + x] for x in nodes[1:]] + [int(res.next_tokens[s])], dtype=torch.int64)])
                at += k
            assert cache.lengths.tolist() == [len(h) - 1 for h in have]
        for h, w in zip(have, want):
            m = min(len(h), len(w))
            assert torch.equal(h[:m], w[:m])


def test_pages_are_handed_out_and_taken_back():
    model = tiny()
    cache = pages(model, 3, capacity=40, pages=5)
    cache.reserve([17, 1, 0])
    assert [len(x) for x in cache.owned] == [2, 1, 0] and len(cache.free_pages) == 2
    table = cache.page_table.tolist()
    assert table[0][2] == table[1][1] == table[2][0] == -1 and len({*table[0][:2], table[1][0]}) == 3
    with pytest.raises(RuntimeError, match="pages needed"):
        cache.reserve([0, 40, 1])
    with pytest.raises(ValueError, match="may not fit"):
        cache.reserve([41, 0, 0])
    with pytest.raises(ValueError, match="3"):
        cache.reserve([1, 1])
    assert cache.page_table.tolist() == table
    with torch.no_grad():
        model(torch.zeros(1, 18, dtype=torch.int64), packed=batch([17, 1, 0]), past_key_values=cache)
    assert cache.most == [17, 1, 0] and len(cache.free_pages) == 2
    cache.free(0)
    assert cache.lengths.tolist() == [0, 1, 0] and len(cache.free_pages) == 4 and cache.page_table[0].tolist() == [-1] * 3
    cache.clear()
    assert cache.lengths.tolist() == [0, 0, 0] and sorted(cache.free_pages) == list(range(5))


def test_a_refused_call_changes_nothing():
    model = tiny()
    cache = pages(model, 2, capacity=32, pages=2)
    with torch.no_grad():
        model(torch.zeros(1, 6, dtype=torch.int64), packed=batch([3, 3]), past_key_values=cache)
        before = cache.planes.clone()
        for n in ([1, 40], [20, 20]):
            with pytest.raises((ValueError, RuntimeError)):
                model(torch.zeros(1, sum(n), dtype=torch.int64), packed=batch(n), past_key_values=cache)
        with pytest.raises(ValueError, match="sequences"):
            model(torch.zeros(1, 3, dtype=torch.int64), packed=batch([1, 1, 1]), past_key_values=cache)
        other = DraftTree(batch([2, 1]))
        with pytest.raises(ValueError, match="another batch"):
            model(torch.zeros(1, 3, dtype=torch.int64), packed=batch([2, 1]), past_key_values=cache, drafts=other)
        slots = PackedCache(model.config, 2, 16, dtype=torch.float32, device="cpu")
        with pytest.raises(ValueError, match="PagedCache"):
            model(torch.zeros(1, 3, dtype=torch.int64), packed=other.batch, past_key_values=slots, drafts=other)
        with pytest.raises(ValueError, match="PagedCache"):
            model.verify_step(torch.zeros(1, 3, dtype=torch.int64), other.batch, slots)
        with pytest.raises(ValueError, match="temperature"):
            model.verify_step(torch.zeros(1, 3, dtype=torch.int64), other.batch, cache, temperature=0.0)
        with pytest.raises(ValueError, match="packed"):
            model(torch.zeros(1, 3, dtype=torch.int64), drafts=other)
    assert cache.lengths.tolist() == [3, 3] == cache.most and torch.equal(cache.planes, before)
    with pytest.raises(RuntimeError, match="no_grad"):
        model(torch.zeros(1, 2, dtype=torch.int64), packed=batch([1, 1]), past_key_values=cache)


def test_rows_without_a_page_and_past_the_table():
    model = tiny(max_position_embeddings=20)
    cache = pages(model, 2, capacity=40)
    free = PackedBatch(torch.tensor([0, 10, 20], dtype=torch.int32), 20)  # lengths the host does not know: no pages
    with torch.no_grad():
        out = model(torch.zeros(1, 20, dtype=torch.int64), packed=free, past_key_values=cache).logits
        assert torch.isfinite(out).all() and not bool(cache.planes.any())
        cache.clear()
        cache.reserve(25)
        cache.lengths[0] = 15
        out = model(torch.zeros(1, 20, dtype=torch.int64), packed=free, past_key_values=cache).logits[0]
        assert bool(out[5:10].isnan().all()) and torch.isfinite(out[:5]).all() and torch.isfinite(out[10:]).all()


def test_draft_tree_refusals_and_edges():
    b = batch([70, 0, 2], rows=75)
    tree = DraftTree(b, torch.cat([torch.arange(-1, 69), torch.tensor([5, 7]), torch.zeros(3)]).to(torch.int32))
    assert tree.mask.shape == (75, 2) and tree.depths[:70].tolist() == list(range(70))
    assert tree.mask[69].tolist() == [-1, 63]
    assert tree.mask[70:72].tolist() == [[1, 0], [2, 0]] and tree.depths[70:72].tolist() == [0, 0]
    assert DraftTree(b).mask is None
    for bad in (torch.zeros(75, dtype=torch.int64), torch.zeros(74, dtype=torch.int32)):
        with pytest.raises(ValueError, match="parents"):
            DraftTree(b, bad)
    assert DraftTree(batch([]), torch.zeros(0, dtype=torch.int32)).mask.shape == (0, 1)


@pytest.mark.parametrize("inter", [False, True])
def test_plain_rotary_gradients(inter):
    torch.manual_seed(0)
    q, k = (torch.randn(5, h, 12, dtype=torch.float64, requires_grad=True) for h in (3, 2))
    a = torch.rand(7, 4, dtype=torch.float64)
    at = torch.tensor([0, 6, 3, 3, 1])
    assert torch.autograd.gradcheck(lambda x, y: plain_rotary(x, y, a.cos(), a.sin(), at, inter), (q, k))
    y = plain_rotary(q, None, a.cos(), a.sin(), torch.tensor([0, 7, -1, 3, 1]), inter)[0]
    assert y[1:3, :, :8].isnan().all() and torch.equal(y[..., 8:], q[..., 8:]) and torch.isfinite(y[3:]).all()


def test_own_pairs_without_a_cache_and_padded():
    """Other rotary layouts on the dense paths: prefill, cached steps and a padded batch agree."""
    model = tiny(rotary_dim=8, rope_interleaved=True)
    ids = torch.randint(0, 50, (2, 11))
    with torch.no_grad():
        full = model(ids).logits
        first = model(ids[:, :6], use_cache=True)
        rest = model(ids[:, 6:], past_key_values=first.past_key_values, use_cache=True).logits
        assert torch.allclose(torch.cat([first.logits, rest], 1), full, atol=1e-4)
        slots = PackedCache(model.config, 2, 16, dtype=torch.float32, device="cpu")
        got = model(ids.reshape(1, 22), packed=batch([11, 11]), past_key_values=slots).logits
        assert torch.allclose(got.view(2, 11, -1), full, atol=1e-4)
    loss = model(ids, labels=ids).loss
    loss.backward()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters() if p.grad is not None)


def test_default_config_has_the_rotary_of_before():
    cfg = MiniMindConfig(hidden_size=64, num_attention_heads=4)
    assert cfg.rotary_dim == cfg.head_dim == 16 and not cfg.rope_interleaved
    for bad in (7, 18, 0):
        with pytest.raises(AssertionError, match="rotary_dim"):
            MiniMindConfig(hidden_size=64, num_attention_heads=4, rotary_dim=bad)


def test_cpu_tensors_are_refused():
    q, pool = torch.zeros(2, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 16, 2, 64, dtype=torch.bfloat16)
    one, cu, table = torch.zeros(1, dtype=torch.int32), torch.tensor([0, 2], dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    ang = torch.zeros(4, 32)
    for call in (lambda: rotary(q, q, ang, ang, torch.zeros(2, dtype=torch.int64)),
                 lambda: paged_append(q, q, q, pool, pool, table, one, cu, ang, ang),
                 lambda: paged_attention(q, pool, pool, table, one, cu),
                 lambda: paged_keep(pool[None], table, one, cu, one, one),
                 lambda: verify_drafts(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64), cu)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_plain_verify_against_the_walk():
    from test_gpu_drafts import make, walk
    for mode in ("sample", "certain", "greedy"):
        lens = [5, 1, 0, 9, 12]
        p, q, tokens, parents, u = make("cpu", torch.float32, lens, 60, 3, mode, seed=4)
        cu = torch.tensor([0, 5, 6, 6, 15, 27], dtype=torch.int32)
        kept, path, following = plain_verify(p, tokens, cu, torch.tensor(parents, dtype=torch.int32), q, u)
        at = 0
        for i, n in enumerate(lens):
            if n:
                sl = slice(at, at + n)
                want, token = walk(p[sl].double(), None if q is None else q[sl].double(), tokens[sl].tolist(),
                                   parents[at:at + n], None if u is None else u[sl].double().tolist())
                assert path[sl].tolist() == want + [-1] * (n - len(want)) and int(following[i]) == token
                assert int(kept[i]) == len(want)
            at += n
