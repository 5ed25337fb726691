"""Packed sequences without a GPU, where a call's sequences, rows, types and lengths are not
the usual ones: values that are not finite, rows behind the last sequence, bounds past the
rows, caches of another type, slots that fill up unevenly."""
from __future__ import annotations

import math

import pytest
import torch

from model.model_minimind import MiniMindForCausalLM
from model.packed import PackedBatch, PackedCache, _plain_attention
from tests.test_packed import _ints, _model


# ------------------------------------------------- log-probabilities of sequences

def _rows_of(m, monkeypatch, lp):
    """m, whose rows' log-probabilities are lp wherever a label counts."""
    monkeypatch.setattr(MiniMindForCausalLM, "_token_logprobs",
                        staticmethod(lambda logits, y: torch.where(y != -100, lp, 0.0)))
    return m


@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("bad", [-math.inf, math.nan])
def test_sequence_logprobs_keep_to_their_sequence(monkeypatch, bad, average):
    lengths = [3, 0, 4, 1, 5]
    b = PackedBatch.from_lengths(lengths, rows=15, device="cpu")
    lp = -torch.rand(15)
    lp[4] = bad  # of the third
    got = _rows_of(_model(), monkeypatch, lp).sequence_logprobs(
        torch.zeros(1, 15, dtype=torch.int64), torch.zeros(1, 15, dtype=torch.int64), b, average)
    want, at = [], 0
    for n in lengths:  # a sequence's last row predicts nothing
        s = sum(float(x) for x in lp[at:at + max(n - 1, 0)])
        want.append(s / max(n - 1, 1) if average else s)
        at += n
    assert got.dtype == torch.float32
    # 64-bit sums, rounded once
    torch.testing.assert_close(got, torch.tensor(want, dtype=torch.float64).float(), rtol=2.0 ** -23, atol=0.0,
                               equal_nan=True)
    assert torch.isfinite(got[[0, 1, 3, 4]]).all() and not math.isfinite(got[2])


@pytest.mark.parametrize("cu", [(0, 5, 20), (0, -3, 12), (0, 9, 4)])
def test_sequence_logprobs_of_bounds_past_the_rows(monkeypatch, cu):
    """Clamped to the rows, as everywhere (the last: decreasing, any values, but no error)."""
    b = PackedBatch(_ints(*cu), 12)
    lp = -torch.rand(12)
    ids = torch.zeros(1, 12, dtype=torch.int64)
    got = _rows_of(_model(), monkeypatch, lp).sequence_logprobs(ids, ids, b)
    assert got.shape == (2,)
    if cu[1] == 5:
        torch.testing.assert_close(got, torch.stack([lp[:4].double().sum(), lp[5:11].double().sum()]).float())


def test_sequence_logprobs_gradient():
    m = _model()
    b = PackedBatch.from_lengths([4, 1, 6], rows=13, device="cpu")
    ids = torch.randint(0, 50, (1, 13))
    s = m.sequence_logprobs(ids, ids, b)
    got = torch.autograd.grad((s * torch.tensor([1.0, 5.0, -2.0])).sum(), list(m.parameters()))
    ref = []
    for a, n in ((0, 4), (5, 6)):
        lp = torch.log_softmax(m(ids[:, a:a + n]).logits[0], -1)
        ref.append(lp[:-1].gather(1, ids[0, a + 1:a + n, None]).sum())
    want = torch.autograd.grad(ref[0] - 2.0 * ref[1], list(m.parameters()))
    for x, y in zip(got, want):
        torch.testing.assert_close(x, y, rtol=1e-3, atol=1e-4)


# ------------------------------------------------- slots that fill up unevenly

def _step(m, cache, lengths, **kw):
    b = PackedBatch.from_lengths(lengths, device="cpu") if not isinstance(lengths, PackedBatch) else lengths
    with torch.no_grad():
        return m(torch.zeros(1, b.rows, dtype=torch.int64), packed=b, past_key_values=cache, **kw)


def test_uneven_batches_that_fit():
    m = _model().eval()
    cache = PackedCache(m.config, 2, 10, torch.float32, "cpu")
    _step(m, cache, [8, 1])
    _step(m, cache, [1, 8])
    _step(m, cache, [1, 0])
    assert cache.lengths.tolist() == [10, 9]
    for lengths in ([1, 0], [0, 2]):
        with pytest.raises(ValueError, match="10 rows"):
            _step(m, cache, lengths)
    _step(m, cache, [0, 1])
    assert cache.lengths.tolist() == [10, 10]
    cache.clear()
    _step(m, cache, [10, 10])


def test_failed_calls_take_no_room(monkeypatch):
    m = _model().eval()
    cache = PackedCache(m.config, 2, 10, torch.float32, "cpu")
    _step(m, cache, [2, 1])
    with monkeypatch.context() as c:
        c.setattr(m.model.layers[1].mlp, "forward", lambda z: 1 / 0)
        for _ in range(3):
            with pytest.raises(ZeroDivisionError):
                _step(m, cache, [8, 4])
    assert cache.lengths.tolist() == [2, 1]
    _step(m, cache, [8, 8])
    assert cache.lengths.tolist() == [10, 9]


def test_batches_of_unknown_lengths_between():
    """What the host has not seen refuses nothing; what it has seen still does."""
    m = _model().eval()
    cache = PackedCache(m.config, 2, 10, torch.float32, "cpu")
    _step(m, cache, [6, 2])
    _step(m, cache, PackedBatch(_ints(0, 1, 4), 4))
    _step(m, cache, [3, 5])
    assert cache.lengths.tolist() == [10, 10]
    with pytest.raises(ValueError, match="10 rows"):
        _step(m, cache, [2, 0])


def test_lengths_from_an_iterator():
    b = PackedBatch.from_lengths((n for n in (3, 5)), device="cpu")
    assert b.longest == 5 and b.cu_seqlens.tolist() == [0, 3, 8]
    assert PackedBatch.from_lengths(torch.tensor([3, 5]), device="cpu").longest == 5


# ------------------------------------------------- positions past the rotary table

def test_positions_past_the_table_are_refused():
    """Where the host knows the lengths; the dense call raises too."""
    m = _model(max_position_embeddings=16).eval()
    ids = torch.randint(0, 50, (1, 20))
    with pytest.raises(RuntimeError):
        m(ids)
    for lengths in ([17, 3], [3, 17]):
        with pytest.raises(ValueError, match="17 positions.*16"):
            m(ids, packed=PackedBatch.from_lengths(lengths, device="cpu"))
    b = PackedBatch.from_lengths([16, 1], rows=20, device="cpu")  # 3 rows of no sequence
    torch.testing.assert_close(m(ids, packed=b).logits[:, :16], m(ids[:, :16]).logits, rtol=1e-4, atol=1e-4)


def test_cached_positions_past_the_table_are_refused():
    m = _model(max_position_embeddings=16).eval()
    cache = PackedCache(m.config, 2, 20, torch.float32, "cpu")
    ids = torch.randint(0, 50, (1, 14))
    with torch.no_grad():
        m(ids, packed=PackedBatch.from_lengths([10, 4], device="cpu"), past_key_values=cache)
        with pytest.raises(ValueError, match="17 positions.*16"):
            m(ids[:, :10], packed=PackedBatch.from_lengths([7, 3], device="cpu"), past_key_values=cache)
        assert cache.lengths.tolist() == [10, 4]
        out = m(ids[:, :10], packed=PackedBatch.from_lengths([6, 4], device="cpu"), past_key_values=cache)
    assert cache.lengths.tolist() == [16, 8] and torch.isfinite(out.logits).all()


def test_positions_the_host_does_not_know():
    """Not a number behind the table's end instead of the last position's angles again: in that
    sequence alone."""
    m = _model(max_position_embeddings=16).eval()
    ids = torch.randint(0, 50, (1, 40))
    out = m(ids, packed=PackedBatch(_ints(0, 9, 29), 40)).logits[0]  # the second has 20 tokens
    torch.testing.assert_close(out[:9], m(ids[:, :9]).logits[0], rtol=1e-4, atol=1e-4)
    assert out[25:29].isnan().all() and torch.isfinite(out[29:]).all()
    cache = PackedCache(m.config, 2, 20, torch.float32, "cpu")
    with torch.no_grad():
        for n in (9, 7):
            out = m(ids[:, :n + 1], packed=PackedBatch(_ints(0, n, n + 1), n + 1), past_key_values=cache).logits[0]
            assert torch.isfinite(out).all()
        out = m(ids[:, :3], packed=PackedBatch(_ints(0, 2, 3), 3), past_key_values=cache).logits[0]
    assert out[:2].isnan().all() and torch.isfinite(out[2]).all()


# ------------------------------------------------- the router's balance loss

@pytest.mark.parametrize("lengths", [[3], [6, 6], [0, 4, 0], []])
def test_rows_of_no_sequence_are_not_balanced(lengths):
    """The loss over all tokens takes the sequences' tokens alone: the same loss and
    gradients whatever the rows behind them hold, and those of the sequences without such rows."""
    m = _model(use_moe=True, num_experts_per_tok=2, router_aux_loss_coef=0.5).train()
    moe, n = m.model.layers[0].mlp, sum(lengths)
    res = []
    ids = torch.randint(0, 50, (1, n + 8))
    for rows, seed in ((n + 8, 1), (n + 8, 2), (n, None)):
        x = ids.clone()
        if seed is not None:
            x[0, n:] = torch.randint(0, 50, (8,), generator=torch.Generator().manual_seed(seed))
        m.zero_grad()
        if rows == 0:
            continue
        out = m(x[:, :rows], packed=PackedBatch.from_lengths(lengths, rows=rows, device="cpu"))
        out.aux_loss.backward()
        res.append((out.aux_loss.detach(), moe.gate.weight.grad.clone()))
    for other in res[1:]:
        # other numbers of rows add up in other orders: 64 terms of a product 64 x 2^-24, some four
        # products one after another before the gate's gradient, whose elements also cancel
        for a, b in zip(res[0], other):
            torch.testing.assert_close(a, b, rtol=0.0, atol=2.0 ** -16 * float(a.abs().max()))
    assert n or (float(res[0][0]) == 0.0 and float(res[0][1].abs().max()) == 0.0)


def test_expert_counts_belong_to_their_call():
    """Counted wherever the balance loss is formed, and none of an earlier call elsewhere."""
    m = _model(use_moe=True, num_experts_per_tok=2).train()
    ids = torch.randint(0, 50, (3, 7))
    moe = m.model.layers[1].mlp
    m(ids)
    assert moe.expert_counts.dtype == torch.int64
    assert moe.expert_counts.shape == (4,) and int(moe.expert_counts.sum()) == 42
    m.eval()(ids)
    assert moe.expert_counts is None


@pytest.mark.parametrize("cu", [(0, 5, 20), (0, -3, 12)])
def test_balance_of_each_sequence_clamps_its_bounds(cu):
    m = _model(use_moe=True, num_experts_per_tok=2, router_aux_loss_per_sequence=True, router_aux_loss_coef=0.5).train()
    ids = torch.randint(0, 50, (1, 12))
    got = m(ids, packed=PackedBatch(_ints(*cu), 12))
    lengths = [5, 7] if cu[1] == 5 else [0, 12]
    assert m.model.layers[0].mlp.expert_counts.sum(1).tolist() == [2 * n for n in lengths]
    want = m(ids, packed=PackedBatch.from_lengths(lengths, device="cpu"))
    torch.testing.assert_close(got.aux_loss, want.aux_loss, rtol=1e-6, atol=0.0)


# ------------------------------------------------- a cache of another type than the model

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kept", [torch.float32, torch.bfloat16, torch.float16, None])
def test_cache_of_another_type(dtype, kept):
    """A model takes a cache of any type (None: the default): its outputs stay in its own."""
    m = _model().to(dtype).eval()
    cache = PackedCache(m.config, 2, 8, device="cpu", **({} if kept is None else {"dtype": kept}))
    ids = torch.randint(0, 50, (1, 8))
    with torch.no_grad():
        out = m(ids[:, :6], packed=PackedBatch.from_lengths([2, 4], device="cpu"), past_key_values=cache)
        out = m(ids[:, 6:], packed=PackedBatch.from_lengths([1, 1], device="cpu"), past_key_values=cache)
        ref = m(ids[:, [0, 1, 6]]).logits[0, -1], m(ids[:, [2, 3, 4, 5, 7]]).logits[0, -1]
    assert out.logits.dtype == dtype and cache.layers[0][0].dtype == (kept or torch.bfloat16)
    assert float(cache.layers[0][0].float().abs().sum()) > 0
    # the right tokens' keys: some 20 roundings of 2^-8 one after another are 0.08, other keys are of order 1
    for got, want in zip(out.logits[0], ref):
        assert float((got - want).float().norm() / want.float().norm()) < 0.1


# ------------------------------------------------- the preference loss on torch ops

@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("smoothing", [0.0, 0.2])
def test_preference_loss_without_a_gpu(average, smoothing):
    """The model's step on the torch path, against each sequence alone."""
    m = _model()
    lengths = [5, 3, 1, 7]
    b = PackedBatch.from_lengths(lengths, rows=19, device="cpu")
    ids = torch.randint(0, 50, (1, 19))
    labels = ids.clone()
    labels[0, :2] = -100
    ref = torch.tensor([-12.0, -8.0, 0.5, -20.0])
    out = m.preference_loss(ids, labels, b, ref, beta=0.2, label_smoothing=smoothing, average=average)
    S, at = [], 0
    for n in lengths:
        lp = torch.log_softmax(m(ids[:, at:at + n]).logits[0], -1)
        y = labels[0, at + 1:at + n]
        rows = [lp[i, t] for i, t in enumerate(y) if t != -100]
        S.append(sum(rows, torch.zeros(())) / (max(len(rows), 1) if average else 1))
        at += n
    r = 0.2 * (torch.stack(S) - ref)
    z, ls = r[:2] - r[2:], torch.nn.functional.logsigmoid
    want = -((1 - smoothing) * ls(z) + smoothing * ls(-z)).mean()
    torch.testing.assert_close(out.loss, want, rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(torch.cat([out.chosen_rewards, out.rejected_rewards]), r.detach(), rtol=1e-4, atol=1e-5)
    assert out.loss.dtype == torch.float32 and not out.chosen_rewards.requires_grad
    got = torch.autograd.grad(out.loss, list(m.parameters()))
    # sums of 64 terms in other orders, 2^-18 each, in up to 16 products one after another
    for a, w in zip(got, torch.autograd.grad(want, list(m.parameters()))):
        torch.testing.assert_close(a, w, rtol=0.0, atol=2.0 ** -14 * float(w.abs().max()))
    for bad, kw in ((ref[:3], {}), (ref[:2], {}), (ref[None], {}), (ref, {"label_smoothing": 1.0})):
        with pytest.raises(ValueError):
            m.preference_loss(ids, labels, b, bad, **kw)


def test_preference_loss_traces():
    m = _model()
    b = PackedBatch.from_lengths([5, 3], device="cpu")
    ids = torch.randint(0, 50, (1, 8))
    ref = torch.tensor([-12.0, -8.0])
    got = torch.compile(lambda i: m.preference_loss(i, i, b, ref).loss, backend="eager")(ids)
    torch.testing.assert_close(got, m.preference_loss(ids, ids, b, ref).loss, rtol=1e-5, atol=1e-6)


def test_preference_pairs_of_impossible_answers(monkeypatch):
    """A rejected answer of log-probability -inf costs nothing without label smoothing."""
    lp = -torch.rand(8)
    lp[6] = -math.inf
    m = _rows_of(_model(), monkeypatch, lp)
    b, ids = PackedBatch.from_lengths([2] * 4, device="cpu"), torch.zeros(1, 8, dtype=torch.int64)
    out = m.preference_loss(ids, ids, b, torch.zeros(4))
    z = 0.1 * (lp[0] - lp[4])
    torch.testing.assert_close(out.loss, -torch.nn.functional.logsigmoid(z) / 2)
    assert float(out.rejected_rewards[1]) == -math.inf
    assert float(m.preference_loss(ids, ids, b, torch.zeros(4), label_smoothing=0.1).loss) == math.inf


def test_batches_without_sequences():
    for each in (False, True):
        m = _model(use_moe=True, num_experts_per_tok=2, router_aux_loss_per_sequence=each).train()
        b, ids = PackedBatch.from_lengths([], rows=5, device="cpu"), torch.randint(0, 50, (1, 5))
        out = m(ids, packed=b)
        assert out.logits.shape == (1, 5, 50) and float(out.aux_loss) == 0.0
        assert m.model.layers[0].mlp.expert_counts.shape == ((0, 4) if each else (4,))
        assert m.sequence_logprobs(ids, ids, b).shape == (0,)
        out.aux_loss.backward()


# ------------------------------------------------- attention on torch ops

@pytest.mark.parametrize("where", ["q", "k", "v"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_plain_attention_keeps_to_its_sequence(where, bad):
    """Values that are not finite reach the rows that see them, and no other sequence."""
    torch.manual_seed(0)
    q, k, v = torch.randn(12, 4, 16), torch.randn(12, 2, 16), torch.randn(12, 2, 16)
    cu = _ints(0, 4, 9, 11)
    good = _plain_attention(q, k, v, cu, cu, None, 0.0)
    t = {"q": q, "k": k, "v": v}[where].clone()
    t[6, 0, 3] = bad
    args = {"q": q, "k": k, "v": v, where: t.requires_grad_()}
    out = _plain_attention(args["q"], args["k"], args["v"], cu, cu, None, 0.0)
    keep = [0, 1, 2, 3, 4, 5, 9, 10, 11]
    torch.testing.assert_close(out[keep], good[keep], rtol=1e-6, atol=1e-6)
    assert not torch.isfinite(out[6, 0]).all()
    g, = torch.autograd.grad(out[keep].sum(), t)
    assert torch.isfinite(g[:4]).all() and torch.isfinite(g[9:]).all()


# ------------------------------------------------- launches of 2^32 threads

def test_library_refuses_what_a_launch_cannot_hold():
    """Such a launch would wrap without an error.  Nothing of these calls reaches a device."""
    import ctypes
    from model import _hip
    lib, p = _hip.load(), ctypes.c_void_p(16)

    def refused(rc):
        return rc != 0 and b"too large" in lib.mhc_last_error()
    for B, Tq, heads, kv in ((1 << 24, 8, 2, 1), (1 << 22, 1 << 22, 16, 16), (1 << 21, 1 << 23, 32, 32)):
        sizes = (B, Tq, Tq, heads, kv, 64)
        assert lib.mhc_packed_attn_workspace_bytes(*sizes) == -1
        assert lib.mhc_packed_attn_bwd_workspace_bytes(*sizes) == -1
        assert refused(lib.mhc_packed_attn_fwd(p, 64, 64, p, 64, 64, p, 64, 64, p, p, None, p, None, None, p, 1 << 60,
                                               *sizes, 1, 0.1, None))
        assert refused(lib.mhc_packed_attn_bwd(p, 64, 64, p, 64, 64, p, 64, 64, p, p, None, p, p, p, p, p, p, p, p,
                                               1 << 60, *sizes, 1, 0.1, None))
    assert refused(lib.mhc_preference_fwd(p, p, -100, p, p, p, p, p, p, p, 4, 1 << 24, 0.1, 0.0, 0, None))
    assert lib.mhc_balance_workspace_bytes(4, 1, 1 << 24) == -1
    assert refused(lib.mhc_balance_fwd(p, 1, 0, p, p, p, p, p, p, 1 << 60, 4, 1, 1, 1 << 24, 0.1, None))
    # the largest that are not
    assert lib.mhc_packed_attn_workspace_bytes(1 << 20, 1 << 20, 1 << 20, 8, 4, 64) >= 0
    assert lib.mhc_packed_attn_bwd_workspace_bytes(1 << 20, 1 << 20, 1 << 20, 8, 4, 64) > 0
    assert lib.mhc_balance_workspace_bytes(1 << 20, 64, 1 << 20) > 0


# ------------------------------------------------- bounds that make no sense, and the cache

@pytest.mark.parametrize("ends", [(9, 9, 9), (3, 5, 8), (0, 150, 20), (-5, 500, 2 ** 31 - 1), (0, -2 ** 31, 8), (0, 6, 2)])
def test_cache_under_bounds_that_make_no_sense(ends):
    """They are taken as the kernels take them: no row lands outside its slots, no length leaves
    them, and the next call is right."""
    m = _model().eval()
    cache = PackedCache(m.config, 2, 10, torch.float32, "cpu")
    ids = torch.randint(0, 50, (1, 8))
    with torch.no_grad():
        for _ in range(3):
            m(ids, packed=PackedBatch(_ints(*ends), 8), past_key_values=cache)
            assert 0 <= int(cache.lengths.min()) and int(cache.lengths.max()) <= 10
        m(ids, packed=PackedBatch(_ints(*ends), 8), labels=ids)
        cache.clear()
        out = m(ids, packed=PackedBatch.from_lengths([5, 3], device="cpu"), past_key_values=cache).logits[0]
        torch.testing.assert_close(out[:5], m(ids[:, :5]).logits[0], rtol=1e-4, atol=1e-4)
    assert cache.lengths.tolist() == [5, 3]


def test_batch_takes_bounds_as_the_kernels_do():
    b = PackedBatch(_ints(3, 5, 500), 8)
    assert b.cu_seqlens.tolist() == [0, 5, 8] and b.positions.tolist() == [0, 1, 2, 3, 4, 0, 1, 2]
    cu = _ints(0, 2, 4)
    b = PackedBatch(cu, 4)
    cu.fill_(1)  # a batch keeps its own
    assert b.cu_seqlens.tolist() == [0, 2, 4]


def test_slots_that_are_freed_or_rolled_back():
    """lengths may be set from outside: what the host has counted no longer refuses anything."""
    m = _model().eval()
    cache = PackedCache(m.config, 2, 10, torch.float32, "cpu")
    ids = torch.randint(0, 50, (1, 9))
    with torch.no_grad():
        m(ids, packed=PackedBatch.from_lengths([8, 1], device="cpu"), past_key_values=cache)
        cache.lengths[0] = 0  # another conversation takes the slot
        out = m(ids, packed=PackedBatch.from_lengths([9, 0], device="cpu"), past_key_values=cache).logits[0]
        torch.testing.assert_close(out, m(ids).logits[0], rtol=1e-4, atol=1e-4)
        assert cache.lengths.tolist() == [9, 1]
        for _ in range(12):  # the last token of both, again and again
            m(ids[:, :2], packed=PackedBatch.from_lengths([1, 1], device="cpu"), past_key_values=cache)
            cache.lengths.sub_(1)
        assert cache.lengths.tolist() == [9, 1]
        m(ids[:, :2], packed=PackedBatch.from_lengths([1, 1], device="cpu"), past_key_values=cache)
        m(ids[:, :8], packed=PackedBatch.from_lengths([0, 8], device="cpu"), past_key_values=cache)
        with pytest.raises(ValueError, match="10 rows"):  # counted anew since then: 1 and 1 + 8, and 9 more
            m(ids, packed=PackedBatch.from_lengths([0, 9], device="cpu"), past_key_values=cache)


def test_cache_made_in_inference_mode():
    """Is a cache as any other: used outside, and its lengths set from outside."""
    m = _model().eval()
    ids = torch.randint(0, 50, (1, 9))
    b = PackedBatch.from_lengths([8, 1], device="cpu")
    with torch.inference_mode():
        cache = PackedCache(m.config, 2, 10, torch.float32, "cpu")
        for _ in range(3):
            m(ids, packed=b, past_key_values=cache)
            cache.lengths.zero_()
    with torch.no_grad():
        m(ids, packed=b, past_key_values=cache)
    assert cache.lengths.tolist() == [8, 1]


def test_batch_made_in_inference_mode():
    """Serves a training step afterwards: the reference model's pass comes first."""
    m = _model(use_moe=True, num_experts_per_tok=2).train()
    ids = torch.randint(0, 50, (1, 16))
    with torch.inference_mode():
        b = PackedBatch.from_lengths([5, 3, 1, 7], device="cpu")
        c = PackedBatch(_ints(0, 5, 8, 9, 16), 16)
        ref = m.sequence_logprobs(ids, ids, b)
    for batch in (b, c):
        m.preference_loss(ids, ids, batch, ref).loss.backward()
        m(ids, packed=batch, labels=ids).loss.backward()


def test_library_refuses_more_experts_and_sequences_than_are_joined():
    """2^31 less 128 pairs of them: the join counts in 32 bits, some past the last."""
    from model import _hip
    lib = _hip.load()
    assert lib.mhc_balance_workspace_bytes(4, 128, (1 << 24) - 1) == -1
    assert lib.mhc_balance_workspace_bytes(4, 64, 1 << 23) > 0
