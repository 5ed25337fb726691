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
