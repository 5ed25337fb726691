"""What a cache of pages hands out and takes back: replays that the host does not see, reservations, lengths that
the host only knows a bound of.  On the CPU; a replay is a call in which Python counts nothing."""
from __future__ import annotations

import contextlib

import pytest
import torch

from model import paged
from model.paged import PagedCache
from test_paged import batch, pages, tiny


@contextlib.contextmanager
def replayed():
    """The call inside moves the cache's lengths on and stores its rows, as a replay does; the host
    neither hands out pages nor counts."""
    with pytest.MonkeyPatch.context() as m:
        m.setattr(paged, "_capturing", lambda t: True)
        yield


def step(model, cache, tokens):
    """One new token for each sequence; the logits of all."""
    new = torch.randint(0, 50, (len(tokens),))
    got = model(new[None], packed=batch([1] * len(tokens)), past_key_values=cache).logits[0]
    for i in range(len(tokens)):
        tokens[i] = torch.cat([tokens[i], new[i:i + 1]])
    return got


def as_without_a_cache(model, got, tokens):
    want = torch.stack([model(t[None]).logits[0, -1] for t in tokens])
    assert torch.allclose(got, want, atol=1e-4)


def begin(model, lengths, **more):
    tokens = [torch.randint(0, 50, (n,)) for n in lengths]
    cache = pages(model, len(lengths), **more)
    model(torch.cat(tokens)[None], packed=batch(lengths), past_key_values=cache)
    return cache, tokens


def test_rounds_of_reserve_and_replays():
    model = tiny()
    with torch.no_grad():
        cache, tokens = begin(model, [30, 3], capacity=120)
        for _ in range(4):
            cache.reserve(16)
            for _ in range(16):
                with replayed():
                    got = step(model, cache, tokens)
            as_without_a_cache(model, got, tokens)
        assert cache.lengths.tolist() == [94, 67]
        assert [len(x) for x in cache.owned] == [6, 5]


def test_calls_after_replays_hand_out_pages_and_raise_where_none_are_left():
    model = tiny(max_position_embeddings=256)
    with torch.no_grad():
        cache, tokens = begin(model, [30], capacity=200, pages=10)
        cache.reserve(100)
        for _ in range(100):
            with replayed():
                step(model, cache, tokens)
        more = torch.randint(0, 50, (20,))
        got = model(more[None], packed=batch([20]), past_key_values=cache).logits[0, -1:]
        tokens = [torch.cat([tokens[0], more])]
        as_without_a_cache(model, got, tokens)
        assert cache.lengths.tolist() == [150] and len(cache.owned[0]) == 10
        with pytest.raises(RuntimeError, match="pages needed"):
            model(torch.zeros(1, 20, dtype=torch.int64), packed=batch([20]), past_key_values=cache)
        for _ in range(10):
            with replayed():
                step(model, cache, tokens)
        with pytest.raises(ValueError, match="may not fit"):
            model(torch.zeros(1, 41, dtype=torch.int64), packed=batch([41]), past_key_values=cache)
        assert cache.lengths.tolist() == [160]


def test_dropped_rows_are_noticed():
    """Replays past what was reserved: settling says so, and so does the next call of that sequence."""
    model = tiny()
    with torch.no_grad():
        cache, tokens = begin(model, [30, 10])
        cache.reserve(2)
        for _ in range(3):  # the first sequence's 33rd key has no page
            with replayed():
                step(model, cache, tokens)
        assert cache.lengths.tolist() == [33, 13]
        for call in (cache.settle, lambda: cache.reserve(1), lambda: cache.reserve([1, 0]),
                     lambda: model(torch.zeros(1, 1, dtype=torch.int64), packed=batch([1, 0]), past_key_values=cache)):
            with pytest.raises(RuntimeError, match="sequence 0 has 33 keys and pages for 32"):
                call()
        assert [len(x) for x in cache.owned] == [2, 1] and cache.lengths.tolist() == [33, 13]
        model(torch.zeros(1, 1, dtype=torch.int64), packed=batch([0, 1]), past_key_values=cache)  # not that sequence's
        cache.lengths[0] = 32  # rolled back to what is there
        cache.settle()
        tokens[0] = tokens[0][:32]
        tokens[1] = torch.cat([tokens[1], torch.zeros(1, dtype=torch.int64)])
        as_without_a_cache(model, step(model, cache, tokens), tokens)
        cache.reserve(1)
        for _ in range(20):
            with replayed():
                step(model, cache, tokens)
        with pytest.raises(RuntimeError, match="rows were dropped"):
            cache.settle()
        cache.free(0)
        cache.free(1)
        cache.settle()
        with replayed():  # a slot that is not in use: nothing of it is kept, and nothing is amiss
            step(model, cache, tokens)
        cache.settle()
        assert cache.lengths.tolist() == [1, 1] and cache.owned == [[], []]


def drafts(model, cache, n, seed):
    """A verify_step of n nodes for each sequence whose drafts are mostly wrong; its kept rows."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, 50, (1, n * cache.sequences), generator=g)
    return model.verify_step(ids, batch([n] * cache.sequences), cache).kept


@pytest.mark.parametrize("sizes", [dict(capacity=64), dict(capacity=120, pages=6)])
def test_many_drafts_without_settling(sizes):
    """What the host counts at most no longer fits; what is there does, for as long as it does."""
    model = tiny(max_position_embeddings=256)
    with torch.no_grad():
        cache, _ = begin(model, [8, 3], **sizes)
        have, steps = [8, 3], 0
        while max(have) + 8 <= 64 and steps < 14:
            kept = drafts(model, cache, 8, steps)
            have = [a + b for a, b in zip(have, kept.tolist())]
            assert cache.lengths.tolist() == have
            steps += 1
        assert steps == 14 or max(have) + 8 > 64
        assert sum(len(x) for x in cache.owned) + len(cache.free_pages) == cache.planes.shape[1]
        cache.settle()
        assert cache.most == have
        free = len(cache.free_pages)
        with pytest.raises(ValueError, match="may not fit"):  # that one is true
            cache.reserve([cache.capacity - have[0] + 1, 0])
        if free * 16 < cache.capacity - have[0] - 16:
            with pytest.raises(RuntimeError, match="pages needed"):
                cache.reserve([cache.capacity - have[0], 0])
        assert len(cache.free_pages) == free and cache.most == have


def test_lengths_that_the_host_does_not_know_are_looked_at():
    """A batch whose lengths only the device knows counts all its rows for every sequence."""
    from model.packed import PackedBatch
    model = tiny()
    with torch.no_grad():
        cache, tokens = begin(model, [4, 4], capacity=48, pages=6)
        cache.reserve(4)
        free = PackedBatch(torch.tensor([0, 4, 8], dtype=torch.int32), 8)
        new = torch.randint(0, 50, (8,))
        for _ in range(5):  # far more than fits, if every row were each sequence's
            cache.lengths.fill_(4)
            model(new[None], packed=free, past_key_values=cache)
        tokens = [torch.cat([t, n]) for t, n in zip(tokens, new.split(4))]
        as_without_a_cache(model, step(model, cache, tokens), tokens)
        more = torch.randint(0, 50, (60,))
        got = model(more[None], packed=batch([30, 30]), past_key_values=cache).logits[0, [29, 59]]
        as_without_a_cache(model, got, [torch.cat([t, n]) for t, n in zip(tokens, more.split(30))])


def test_what_is_not_taken_back_for_another_sequence():
    """Pages that were reserved, and those of drafts that are not kept yet."""
    model = tiny()
    with torch.no_grad():
        cache, tokens = begin(model, [5, 5, 5], capacity=64, pages=6)
        cache.reserve([0, 0, 20])  # sequence 2: a page more
        b = batch([30, 0, 0])
        ids = torch.randint(0, 50, (30,))
        model(ids[None], packed=b, past_key_values=cache, drafts=paged.DraftTree(b))  # sequence 0: two more, the last
        assert not cache.free_pages
        with pytest.raises(RuntimeError, match="1 pages needed, 0 left"):
            model(torch.zeros(1, 20, dtype=torch.int64), packed=batch([0, 20, 0]), past_key_values=cache)
        cache.settle()  # takes back what was reserved, not the drafts
        assert [len(x) for x in cache.owned] == [3, 1, 1]
        more = torch.randint(0, 50, (20,))
        model(more[None], packed=batch([0, 20, 0]), past_key_values=cache)
        cache.keep(b, torch.tensor([30, 0, 0], dtype=torch.int32), torch.arange(30, dtype=torch.int32))
        tokens[0], tokens[1] = torch.cat([tokens[0], ids]), torch.cat([tokens[1], more])
        assert cache.lengths.tolist() == [35, 25, 5] == cache.most
        as_without_a_cache(model, step(model, cache, tokens), tokens)
        cache.clear()
        cache.reserve([1, 1, 1])
        cache.settle()
        assert cache.owned == [[], [], []] and len(cache.free_pages) == 6


def test_settling_between_replays_keeps_what_was_reserved_for_them():
    model = tiny()
    with torch.no_grad():
        cache, tokens = begin(model, [14, 2], capacity=100)
        cache.reserve(40)
        for turn in range(40):
            with replayed():
                got = step(model, cache, tokens)
            if turn % 10 == 5:
                cache.settle()
        as_without_a_cache(model, got, tokens)
        assert cache.lengths.tolist() == [54, 42] and [len(x) for x in cache.owned] == [4, 3]
        cache.reserve([30, 1])
        assert [len(x) for x in cache.owned] == [6, 3]
        cache.settle(spare=[10, 0])
        assert [len(x) for x in cache.owned] == [4, 3] and cache.held == [64, 42]
        cache.settle(spare=100)  # what there is: it hands out none
        assert [len(x) for x in cache.owned] == [4, 3]
        with pytest.raises(ValueError, match="rows of 3"):
            cache.settle(spare=[1, 2, 3])
        cache.lengths.copy_(torch.tensor([20, 3]))
        cache.settle(spare=0)
        assert [len(x) for x in cache.owned] == [2, 1]


def test_captured_drafts_that_are_kept_outside_the_graph():
    """The forward pass of a tree in a graph, verification and keeping outside: its replays need their pages too."""
    model = tiny()
    with torch.no_grad():
        cache, tokens = begin(model, [14], capacity=100)
        cache.reserve(20)
        b, ids = batch([10]), torch.randint(0, 50, (10,))
        for turn in range(2):
            with replayed():
                model(ids[None], packed=b, past_key_values=cache, drafts=paged.DraftTree(b))
            cache.settle()
            assert len(cache.owned[0]) == 3
            cache.keep(b, torch.tensor([10], dtype=torch.int32), torch.arange(10, dtype=torch.int32))
            tokens[0] = torch.cat([tokens[0], ids])
        cache.settle()
        as_without_a_cache(model, step(model, cache, tokens), tokens)


def test_a_call_that_reaches_past_the_tables_hands_out_nothing():
    model = tiny(max_position_embeddings=20)
    with torch.no_grad():
        cache, _ = begin(model, [3, 3], capacity=64, pages=6)
        table = cache.page_table.clone()
        with pytest.raises(ValueError, match="max_position_embeddings is 20"):
            model(torch.zeros(1, 42, dtype=torch.int64), packed=batch([2, 40]), past_key_values=cache)
        assert torch.equal(cache.page_table, table) and len(cache.free_pages) == 4 and cache.most == [3, 3]


def test_pages_are_not_handed_out_or_taken_back_while_capturing():
    """The host's part would happen once and the device's with every replay."""
    model = tiny()
    with torch.no_grad():
        cache, _ = begin(model, [14, 2])
        state = lambda: (cache.most, cache.held, cache.owned, cache.free_pages, cache.lengths.tolist(), cache.page_table.tolist())
        before = repr(state())
        for call in (lambda: cache.reserve(40), cache.settle, lambda: cache.free(0), cache.clear):
            with replayed(), pytest.raises(RuntimeError, match="captur"):
                call()
        assert repr(state()) == before
        with replayed():
            assert pages(model, 2).owned == [[], []]
