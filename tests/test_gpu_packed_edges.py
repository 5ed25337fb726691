"""Packed sequences on the GPU, where a call's sequences, rows, types and lengths are not the
usual ones: values that are not finite, rows behind the last sequence, caches of another
type, gradients of very different sizes."""
from __future__ import annotations

import copy
import math

import pytest
import torch

from model import packed
from model.losses import balance_loss, preference_loss, token_logprobs
from model.packed import PackedBatch, PackedCache
from tests.test_gpu_losses import EPS, F32, _exact_logprobs, _logits
from tests.test_gpu_packed import _cu, exact
from tests.test_gpu_packed_model import _far, _model, _taken

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


# ------------------------------------------------- the router's balance loss

@pytest.mark.gpu
@pytest.mark.parametrize("each", [False, True])
@pytest.mark.parametrize("lengths", [[60, 1, 33], [0, 5, 0], [0]])
def test_rows_of_no_sequence_are_not_balanced(dev, lengths, each):
    """Whatever the rows behind the sequences hold: the loss, counts and gradients are those of
    a batch without such rows (to the sums' order)."""
    m = _model(dev, torch.float32, use_moe=True, num_experts_per_tok=2, use_mhc=0, router_aux_loss_coef=0.5,
               router_aux_loss_per_sequence=each).train()
    moe, n = m.model.layers[0].mlp, sum(lengths)
    ids = torch.randint(0, 500, (1, n + 70), device=dev)
    res = []
    for tail in (0, 70, 70):
        x = torch.cat([ids[:, :n], torch.randint(0, 500, (1, tail), device=dev)], 1)
        if x.numel() == 0:
            continue
        m.zero_grad()
        m(x, packed=PackedBatch.from_lengths(lengths, rows=x.shape[1], device=dev)).aux_loss.backward()
        assert moe.expert_counts.shape == ((len(lengths), 4) if each else (4,))
        assert int(moe.expert_counts.sum()) == 2 * n
        res.append((moe.aux_loss.detach().clone(), moe.expert_counts, moe.gate.weight.grad.clone()))
    for other in res[1:]:
        assert torch.equal(res[0][1], other[1])
        torch.testing.assert_close(res[0][0], other[0], rtol=1e-5, atol=0.0)
        torch.testing.assert_close(res[0][2], other[2], rtol=1e-3, atol=1e-3 * float(res[0][2].abs().max()))
    assert n or (float(res[0][0]) == 0.0 and float(res[0][2].abs().max()) == 0.0)


# ------------------------------------------------- a cache of another type than the model

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF, F16])
@pytest.mark.parametrize("kept", [torch.float32, BF, F16, None])
def test_cache_of_another_type(dev, monkeypatch, dtype, kept):
    """A model takes a cache of any type (None: the default), on the kernels where that has 16
    bits; its outputs stay in its own type."""
    m = _model(dev).eval()
    wide = copy.deepcopy(m).float()
    m = m.to(dtype)
    cache = PackedCache(m.config, 2, 64, device=dev, **({} if kept is None else {"dtype": kept}))
    ids = torch.randint(0, 500, (1, 52), device=dev)
    seen = _taken(monkeypatch)
    with torch.inference_mode():
        m(ids[:, :50], packed=PackedBatch.from_lengths([20, 30], device=dev), past_key_values=cache)
        out = m(ids[:, 50:], packed=PackedBatch.from_lengths([1, 1], device=dev), past_key_values=cache).logits
        ref = wide(ids[:, [*range(20), 50]]).logits[0, -1], wide(ids[:, [*range(20, 50), 51]]).logits[0, -1]
    assert len(seen) == (0 if kept == torch.float32 else 4) and out.dtype == dtype
    # some 20 roundings of 2^-8 one after another are 0.08, other keys than the right ones are of order 1
    for got, want in zip(out[0], ref):
        assert _far(got, want) < 0.1


@pytest.mark.gpu
@pytest.mark.parametrize("cast", [BF, F16])
def test_cache_is_read_in_place_under_autocast(dev, monkeypatch, cast):
    """Also where the autocast's type is not the cache's: no step copies the slots."""
    m = _model(dev, torch.float32).eval()
    cache = PackedCache(m.config, 2, 64, BF, dev)
    read, run = [], packed._forward
    monkeypatch.setattr(packed, "_forward", lambda q, k, v, *a: read.append((k.data_ptr(), v.data_ptr())) or run(q, k, v, *a))
    ids = torch.randint(0, 500, (1, 52), device=dev)
    with torch.inference_mode(), torch.autocast("cuda", cast):
        m(ids[:, :50], packed=PackedBatch.from_lengths([20, 30], device=dev), past_key_values=cache)
        out = m(ids[:, 50:], packed=PackedBatch.from_lengths([1, 1], device=dev), past_key_values=cache).logits
    assert read == 2 * [(k.data_ptr(), v.data_ptr()) for k, v in cache.layers]
    with torch.inference_mode():
        for i, rows in enumerate(([*range(20), 50], [*range(20, 50), 51])):
            assert _far(out[0, i], m(ids[:, rows]).logits[0, -1]) < 0.1  # as above


# ------------------------------------------------- the preference loss

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF, F16])
@pytest.mark.parametrize("V", [33, 500])
def test_preference_rows_behind_the_last_sequence(dev, dtype, V):
    """Count for nothing, though their labels count and their logits are no numbers: the same
    bits as without them, and zeros as their gradients."""
    torch.manual_seed(0)
    ends, rows = [0, 7, 20, 21, 40], 46
    x = torch.randn(rows, V, device=dev).to(dtype)
    y = torch.randint(0, V, (rows,), device=dev)
    cu = torch.tensor(ends, dtype=torch.int32, device=dev)
    ref = torch.randn(4, device=dev)
    short = x[:40].clone().requires_grad_()
    want = preference_loss(short, y[:40], cu, ref)
    g, = torch.autograd.grad(want[0], short)
    x[40:], x[41], x[42, 3] = math.nan, -math.inf, math.inf
    y[44] = V + 5
    x.requires_grad_()
    got = preference_loss(x, y, cu, ref)
    d, = torch.autograd.grad(got[0], x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(d[:40], g) and torch.equal(d[40:], torch.zeros_like(d[40:]))


# ------------------------------------------------- attention

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("new,keys", [(1, 32), (1, 2000), (3, 1000), (60, 60), (200, 333)])
def test_weights_add_up_to_one(dev, dtype, hd, new, keys):
    """Values of 1 everywhere come out as 1: the sums are those of the probabilities as the
    product takes them, rounded.  Here all but a sequence's first are just under half a step above
    a number of the type, so sums of the unrounded ones would be off by nearly that.  (fp32 sums of n terms
    are off by n 2^-24 at most, under the half step below 1, 2^-9 and 2^-12, for these lengths.)"""
    n, step = 24, 2.0 ** -7 if dtype == BF else 2.0 ** -10
    q, k = torch.zeros(n * new, 8, hd, device=dev), torch.zeros(n, keys, 4, hd, device=dev)
    q[..., 0], k[:, 1:, :, 0] = 1.0, -1.0
    k = k.flatten(0, 1).to(dtype)
    cu, ck = (torch.arange(n + 1, dtype=torch.int32, device=dev) * m for m in (new, keys))
    out = packed.packed_attention(q.to(dtype), k, torch.ones_like(k), cu, cu_seqlens_k=ck,
                                  scale=-math.log(0.5 * (1.0 + 0.49 * step)))
    assert torch.equal(out, torch.ones_like(out))


@pytest.mark.gpu
@pytest.mark.parametrize("new,slots,used,heads,kv,hd", [
    ([64, 16], [8192, 3000], [8192, 2999], 2, 1, 64), ([300, 40], [4100, 90], [3500, 77], 2, 2, 96),
    ([33], [6000], [5999], 4, 1, 128), ([1, 17, 64, 129, 300],) * 3 + (6, 2, 64), ([700, 90],) * 3 + (2, 1, 128),
    ([1200, 5],) * 3 + (4, 2, 96)])
@pytest.mark.parametrize("g_size,v_size", [(1.0, 1.0), (1e-2, 1.0), (1e-3, 1.0), (1e-4, 1.0), (1e-3, 2000.0),
                                           (300.0, 1.0), (2.0, 1e-3)])
def test_fp16_gradients_of_any_size(dev, new, slots, used, heads, kv, hd, g_size, v_size):
    """The terms of dQ and dK keep fp16's 11 bits whatever the size of g and v, and however many
    keys share a row's weight.  The bar is that of one rounding of each term and one of the result,
    with no term that grows with the keys: half a step (2^-11) of the result, half of the smallest
    number (2^-25), half a step of the terms' sizes; fp32 scores and sums are some 2^-18 of them."""
    torch.manual_seed(0)
    q, k, v, g = (torch.randn(rows, h, hd, device=dev) for rows, h in (
        (sum(new), heads), (sum(slots), kv), (sum(slots), kv), (sum(new), heads)))
    # gradients of very different sizes beside each other
    g *= g_size * torch.exp2(torch.randint(-3, 4, (sum(new), heads, 1), device=dev).float())
    q, k, v, g = (t.to(F16) for t in (q, k, v * v_size, g))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = packed.packed_attention(*leaves, _cu(new, dev), cu_seqlens_k=_cu(slots, dev),
                                  key_lengths=torch.tensor(used, dtype=torch.int32, device=dev))
    grads = torch.autograd.grad(out, leaves, g)
    want, size = exact(q, k, v, new, slots, used, 1.0 / math.sqrt(hd), g)
    for name, got, ref, (sz, _) in zip("qkv", grads, want[1:], size[1:]):
        got = got.double().cpu()
        assert torch.isfinite(got).all()
        bar = 2.0 ** -11 * ref.abs() + 2.0 ** -25 + (2.0 ** -11 + 2.0 ** -18) * sz
        assert ((got - ref).abs() <= bar).all(), (name, float(((got - ref).abs() / bar).max()))
        # over all of it the terms' roundings, each relative to a term, are as large as the result's
        # in a sum of independent terms, so together 1.42 times the result's own
        rms, own = float((got - ref).norm()), float((ref.half().double() - ref).norm())
        assert rms <= 1.5 * own + 2.0 ** -18 * float(ref.norm()), (name, rms / own)


@pytest.mark.gpu
def test_fp16_gradients_captured(dev):
    """A captured step replayed on gradients of other sizes: the eager bits, twice over."""
    torch.manual_seed(0)
    lengths = [1500, 0, 70, 1030]
    q, k, v, g = (torch.randn(sum(lengths), h, 64, device=dev).to(F16) for h in (4, 2, 2, 4))
    cu = _cu(lengths, dev)

    def step(q, k, v, g):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        return torch.autograd.grad(packed.packed_attention(*leaves, cu), leaves, g)
    state = [t.clone() for t in (q, k, v, g)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*state)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(*state)
    for size in (1.0, 1e-4, 30.0, 1e-4):
        state[3].copy_(g * size)
        want = step(q, k, v, state[3])
        assert all(torch.equal(a, b) for a, b in zip(want, step(q, k, v, state[3])))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, want)), size


@pytest.mark.gpu
@pytest.mark.parametrize("ends", [[-5, 500, 2 ** 31 - 1], [0, 150, 20], [0, -2 ** 31, 200], [9, 9, 9]])
def test_fp16_bounds_that_make_no_sense(dev, ends):
    """Such a backward pass ends, and the next one is right."""
    torch.manual_seed(0)
    q, k, v, g = (torch.randn(200, h, 64, device=dev).to(F16) for h in (4, 2, 2, 4))

    def step(cu, **more):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        return torch.autograd.grad(packed.packed_attention(*leaves, cu, **more), leaves, g)
    good, cu = step(_cu([120, 80], dev)), torch.tensor(ends, dtype=torch.int32, device=dev)
    for more in ({}, {"cu_seqlens_k": cu.flip(0).contiguous()},
                 {"key_lengths": torch.tensor([-7, 2 ** 31 - 1], dtype=torch.int32, device=dev)}):
        assert [t.shape for t in step(cu, **more)] == [q.shape, k.shape, v.shape]
    assert all(torch.equal(a, b) for a, b in zip(step(_cu([120, 80], dev)), good))


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["v", "g"])
def test_fp16_gradients_beside_values_that_are_not_finite(dev, what):
    """An infinite value or gradient in one sequence leaves the others' bits alone."""
    torch.manual_seed(0)
    lengths = [300, 200, 77]
    q, k, v, g = (torch.randn(577, h, 64, device=dev).to(F16) for h in (4, 2, 2, 4))

    def step():
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        return torch.autograd.grad(packed.packed_attention(*leaves, _cu(lengths, dev)), leaves, g)
    good = step()
    (v if what == "v" else g)[350, 0, 5] = math.inf
    for a, b in zip(step(), good):
        assert torch.equal(a[:300], b[:300]) and torch.equal(a[500:], b[500:])
    (v if what == "v" else g)[350, 0, 5] = 0.0  # and none at all
    q[300:500] = 0.0
    g[300:500] = 0.0
    assert not any(bool(t[300:500].any()) for t in step())


@pytest.mark.gpu
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_preference_pairs_of_impossible_answers(dev, smoothing):
    """A rejected answer that the model rules out (log-probability -inf) costs nothing without
    label smoothing, and does not reach the other pairs; with it, and where the chosen answer
    is ruled out, the loss is infinite."""
    torch.manual_seed(0)
    x, y = torch.randn(40, 50, device=dev), torch.randint(0, 50, (40,), device=dev)
    cu = torch.tensor([0, 10, 20, 30, 40], dtype=torch.int32, device=dev)
    ref = torch.randn(4, device=dev)
    x[33].scatter_(0, y[33:34], -math.inf)  # of the second pair's rejected answer
    leaf = x.clone().requires_grad_()
    loss, chosen, rejected = preference_loss(leaf, y, cu, ref, label_smoothing=smoothing)
    assert float(rejected[1]) == -math.inf and torch.isfinite(chosen).all()
    first = preference_loss(torch.cat([x[:10], x[20:30]]), torch.cat([y[:10], y[20:30]]), cu[:3],
                            ref[[0, 2]], label_smoothing=smoothing)[0]
    if smoothing:
        assert float(loss) == math.inf
    else:
        torch.testing.assert_close(loss.detach(), first / 2, rtol=2.0 ** -22, atol=0.0)
        g, = torch.autograd.grad(loss, leaf)
        assert torch.isfinite(g).all() and not bool(g[10:20].any()) and not bool(g[30:].any())
    swapped = preference_loss(x[[*range(20, 40), *range(20)]], y[[*range(20, 40), *range(20)]], cu,
                              ref[[2, 3, 0, 1]], label_smoothing=smoothing)[0]
    assert float(swapped) == math.inf


@pytest.mark.gpu
def test_preference_takes_64_bit_references(dev):
    """A reference of 64 bits is not rounded: where it is the policy's own sums, the rewards are 0 up
    to the order of 64-bit sums (2000 terms of 10 units).  In 32 bits half a step of a sum of -10000 is 5e-4."""
    torch.manual_seed(0)
    rows, V = 8000, 30
    x, y = 5.0 * torch.randn(rows, V, device=dev), torch.randint(0, V, (rows,), device=dev)
    b = PackedBatch.from_lengths([2000, 1999, 2001, 2000], device=dev)
    own = b.sums(token_logprobs(x, y))
    loss, chosen, rejected = preference_loss(x, y, b.cu_seqlens, own)
    bar = 0.1 * 2000 * 2.0 ** -53 * float(own.abs().max())
    assert chosen.dtype == torch.float32 and float(torch.cat([chosen, rejected]).abs().max()) <= bar
    torch.testing.assert_close(float(loss), math.log(2.0), rtol=2.0 ** -23, atol=0.0)
    low = preference_loss(x, y, b.cu_seqlens, own.float())
    high = preference_loss(x, y, b.cu_seqlens, own.float().double())
    assert all(torch.equal(a, c) for a, c in zip(low, high)) and float(low[1].abs().max()) > bar


@pytest.mark.gpu
def test_model_preference_in_64_bits(dev):
    """sequence_logprobs hands its 64-bit sums on where it is asked to."""
    m = _model(dev, torch.float32).eval()
    b = PackedBatch.from_lengths([200, 150, 60, 90], device=dev)
    ids = torch.randint(0, 500, (1, b.rows), device=dev)
    with torch.no_grad():
        own = m.sequence_logprobs(ids, ids, b, dtype=torch.float64)
        assert own.dtype == torch.float64 and torch.equal(own.float(), m.sequence_logprobs(ids, ids, b))
        out = m.preference_loss(ids, ids, b, own)
    assert float(torch.cat([out.chosen_rewards, out.rejected_rewards]).abs().max()) <= 1e-10


# ------------------------------------------------- second derivatives

@pytest.mark.gpu
def test_second_derivatives_raise(dev):
    """A gradient penalty through what is differentiable once raises; the first derivatives are
    the same with create_graph as without."""
    torch.manual_seed(0)
    q, k, g = (torch.randn(60, h, 64, device=dev).to(BF) for h in (4, 2, 4))
    x, y = torch.randn(60, 50, device=dev), torch.randint(0, 50, (60,), device=dev)
    cu = torch.tensor([0, 20, 60], dtype=torch.int32, device=dev)
    calls = [(lambda q, k, v: (packed.packed_attention(q, k, v, cu) * g).sum(), (q, k, k.flip(0))),
             (lambda x: token_logprobs(x, y).sum(), (x,)),
             (lambda x: preference_loss(x, y, cu, torch.zeros(2, device=dev))[0], (x,))]
    for call, inputs in calls:
        w = [torch.ones((), device=dev, requires_grad=True) for _ in inputs]
        leaves = [t.clone().requires_grad_() for t in inputs]
        plain = torch.autograd.grad(call(*leaves), leaves)
        grads = torch.autograd.grad(call(*[(t * s).to(t.dtype) for t, s in zip(leaves, w)]), leaves, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(grads, plain))
        with pytest.raises(RuntimeError, match="differentiable once"):
            sum((d.float() ** 2).sum() for d in grads).backward()


@pytest.mark.gpu
@pytest.mark.parametrize("each", [False, True])
def test_balance_loss_in_a_gradient_penalty(dev, each):
    """The routers' balance loss differentiates as often as its torch ops do, also where it is a
    factor of something else: against the CPU's torch path."""
    torch.manual_seed(0)
    m = _model(dev, torch.float32, use_moe=True, num_experts_per_tok=2, use_mhc=0, router_aux_loss_coef=0.5,
               router_aux_loss_per_sequence=each).train()
    x, res = torch.randn(3, 40, 192, device=dev), []
    for moe, z in ((m.model.layers[0].mlp, x), (copy.deepcopy(m.model.layers[0].mlp).cpu(), x.cpu())):
        moe(z)
        w = moe.gate.weight
        loss = moe.aux_loss ** 2 * w.square().mean()
        g, = torch.autograd.grad(loss, w, create_graph=True)
        res.append((g.detach().cpu(), *(t.cpu() for t in torch.autograd.grad(g.square().sum(), w))))
    for a, b in zip(*res):
        # fp32 sums of 120 tokens and 192 dims in other orders, 2^-16, twice differentiated
        assert _far(a, b) <= 2.0 ** -13


@pytest.mark.gpu
def test_router_of_very_many_experts(dev):
    """More experts than the kernels count: torch ops, as before."""
    m = _model(dev, torch.float32, use_moe=True, num_experts_per_tok=2, use_mhc=0, router_aux_loss_coef=0.5)
    moe = m.model.layers[0].mlp.train()
    scores = torch.randn(20, 5000, device=dev).softmax(-1)
    idx = scores.topk(2).indices
    moe.config.num_experts = 5000
    for each in (False, True):
        moe.config.router_aux_loss_per_sequence = each
        loss, counts = moe._balance(scores, idx, 2, 10, None)
        want, n = moe._balance(scores.cpu(), idx.cpu(), 2, 10, None)
        torch.testing.assert_close(loss.cpu(), want, rtol=1e-5, atol=0.0)
        assert torch.equal(counts.cpu(), n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, BF])
def test_batches_without_sequences(dev, dtype):
    for each in (False, True):
        m = _model(dev, dtype, use_moe=True, num_experts_per_tok=2, use_mhc=0, router_aux_loss_per_sequence=each).train()
        b, ids = PackedBatch.from_lengths([], rows=5, device=dev), torch.randint(0, 500, (1, 5), device=dev)
        out = m(ids, packed=b)
        assert out.logits.shape == (1, 5, 500) and float(out.aux_loss.detach()) == 0.0
        assert m.model.layers[0].mlp.expert_counts.shape == ((0, 4) if each else (4,))
        assert m.sequence_logprobs(ids, ids, b).shape == (0,)
        out.aux_loss.backward()


@pytest.mark.gpu
def test_model_of_64_bits(dev):
    """No kernel takes fp64: the packed calls run on torch ops, as the dense ones do."""
    m = _model(dev, torch.float64, use_moe=True, num_experts_per_tok=2, use_mhc=0,
               router_aux_loss_per_sequence=True).train()
    cpu = copy.deepcopy(m).cpu()
    lengths = [20, 7, 1, 30]
    ids, ref = torch.randint(0, 500, (1, 58)), torch.randn(4)
    res = []
    for net, d in ((m, dev), (cpu, "cpu")):
        b = PackedBatch.from_lengths(lengths, device=d)
        x = ids.to(d)
        out = net.preference_loss(x, x, b, ref.to(d))
        res.append((net(x, packed=b, labels=x).loss, net.sequence_logprobs(x, x, b), out.loss, out.aux_loss))
    for a, w in zip(*res):  # the rows' log-probabilities are fp32
        torch.testing.assert_close(a.detach().cpu().double(), w.detach().double(), rtol=1e-5, atol=1e-5)


# ------------------------------------------------- gradients of logits, each element by its own size

def _each_close(got, dlp, f, dtype, factor=0.0):
    """f ([hot] - p) element by element: half a step of the type, an error of the log-probability
    (2^-15) on p and one of the factor on all, and at the label, where 1 - p is rounded, four half steps
    of fp32.  (2^-25: half of fp16's smallest number; 2^-120: fp32's smallest exponentials are flushed.)"""
    got, want = got.detach().double().cpu(), dlp * f
    p = torch.where(dlp > 0, 1 - dlp, -dlp)  # 0 in rows that do not count, whose bar stays exact
    bar = (EPS[dtype] + factor) * want.abs() + 2.0 ** -15 * p * f.abs() + (dlp > 0) * 2.0 ** -22 * f.abs() \
        + (dlp != 0) * ((2.0 ** -25 if dtype == F16 else 0.0) + 2.0 ** -120)
    bad = (got - want).abs() > bar
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:5].tolist())


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,dtype,pad,offset", [
    (7, 7, F16, 0, 1), (5, 64, BF, 0, 3), (33, 6400, BF, 0, 0), (9, 6401, F16, 0, 0), (4, 6400, F32, 3, 1),
    (6, 50257, F32, 0, 0), (5, 50257, BF, 0, 5), (300, 100, F16, 28, 0), (2, 131072, BF, 0, 0), (17, 2050, BF, 6, 7),
    (3, 50257, F16, 3, 1), (2, 32001, F32, 1, 2)])
def test_gradients_of_logits_each(dev, T, V, dtype, pad, offset):
    x, labels = _logits(T, V, dtype, dev, pad=pad, offset=offset)
    labels[0] = V - 1
    dlp = _exact_logprobs(x, labels)[1]
    x = x.detach().requires_grad_()
    g = torch.randn(T) * (2.0 ** 12 if dtype == F16 else 1.0)
    got, = torch.autograd.grad(token_logprobs(x, labels), x, g.to(dev))
    _each_close(got, dlp, g.double()[:, None], dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("V,dtype,offset", [(6400, BF, 0), (6401, F32, 1), (50257, F16, 3), (100, BF, 1)])
def test_gradients_of_preference_each(dev, V, dtype, offset):
    lengths, behind = [5, 9, 1, 12], 3
    T = sum(lengths) + behind
    x, labels = _logits(T, V, dtype, dev, offset=offset)
    dlp = _exact_logprobs(x, labels)[1]
    lp = _exact_logprobs(x, labels)[0]
    ends = torch.tensor([0] + lengths).cumsum(0)
    S = torch.stack([lp[a:b].sum() for a, b in zip(ends, ends[1:])])
    ref = (S + torch.tensor([1.0, -2.0, 0.5, 3.0])).float()
    r = 0.3 * (S - ref.double())
    dz = -torch.sigmoid(r[2:] - r[:2]) * 0.3 / 2 * 2.0 ** 12
    f = torch.cat([torch.cat([dz, -dz]).repeat_interleave(torch.tensor(lengths)), torch.zeros(behind)])[:, None]
    x = x.detach().requires_grad_()
    loss = preference_loss(x, labels, ends.to(dev, torch.int32), ref.to(dev), 0.3)[0]
    got, = torch.autograd.grad(loss, x, torch.full((), 2.0 ** 12, device=dev))
    dlp[-behind:] = 0.0
    # z is off by 0.3 of 24 rows' errors of 2^-15, a sigmoid's relative slope is at most 1
    _each_close(got, dlp, f, dtype, factor=0.3 * 24 * 2.0 ** -15 + 2.0 ** -22)


@pytest.mark.gpu
def test_routed_experts_of_packed_rows(dev):
    """The routed layer of a packed inference call gives each sequence's rows what they get alone,
    where the second and third expert are not a rounding apart (half a step of bf16 on scores of up to
    1 is 2^-8 and less; 2^-5 leaves room for the gate's own)."""
    m = _model(dev, use_moe=True, num_experts=6, num_experts_per_tok=2, use_mhc=0).eval()
    moe, lengths = m.model.layers[0].mlp, [70, 1, 33, 150, 64]
    torch.manual_seed(0)
    moe.gate.weight.data.mul_(8.0)
    x = torch.randn(1, sum(lengths), 192, device=dev).to(BF)
    with torch.inference_mode():
        top = (x[0].double() @ moe.gate.weight.double().t()).softmax(-1).topk(3).values
        clear = top[:, 1] - top[:, 2] > 2.0 ** -5
        got, alone = moe(x)[0], torch.cat([moe(t)[0] for t in x.split(lengths, 1)])
    assert int(clear.sum()) > 150
    # both round the same steps (two products, an activation, the weighted sum) to bf16: 4 of 2^-8 each
    off = (got - alone).double().norm(dim=1) / alone.double().norm(dim=1)
    assert float(off[clear].max()) <= 8 * 2.0 ** -8


# ------------------------------------------------- more rows than one dimension of a launch takes

@pytest.mark.gpu
def test_rows_past_the_launch_limit(dev):
    """2^24 rows of 256 threads are 2^32 of them, one more than a dimension of a launch holds."""
    T, V = (1 << 24) + 5, 3
    torch.manual_seed(0)
    part = torch.randn(1 << 10, V, device=dev).to(BF)
    x = part.repeat(T // (1 << 10) + 1, 1)[:T].contiguous().requires_grad_()
    y = torch.randint(0, V, (1 << 10,), device=dev).repeat(T // (1 << 10) + 1)[:T].contiguous()
    small = x[:1 << 10].detach().requires_grad_()
    want = token_logprobs(small, y[:1 << 10])
    g, = torch.autograd.grad(want.sum(), small)
    lp = token_logprobs(x, y)
    got, = torch.autograd.grad(lp.sum(), x)
    for t, w in ((lp.detach(), want.detach()), (got, g)):
        assert torch.equal(t[:-5].view(-1, *w.shape), w.expand(T // (1 << 10), *w.shape))
        assert torch.equal(t[-5:], w[:5])


@pytest.mark.gpu
def test_balance_gradient_past_the_launch_limit(dev):
    """2^32 scores and some: every row's gradient."""
    E, T = 256, (1 << 24) + 3
    torch.manual_seed(0)
    row = torch.rand(1, E, device=dev).to(BF)
    index = torch.randint(0, E, (T, 1), device=dev)
    x = row.expand(T, E).requires_grad_()
    loss, counts = balance_loss(x, index, 1e6)
    g, = torch.autograd.grad(loss, x)
    assert torch.equal(counts, torch.bincount(index[:, 0], minlength=E))
    want = (1e6 * E * (counts.double() / T) / T).to(BF)  # the same of every row, rounded once
    torch.testing.assert_close(g[0], want, rtol=2.0 ** -7, atol=0.0)
    assert bool((g == g[0]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F16])
def test_recomputed_in_the_backward_pass(dev, dtype):
    """Under activation checkpointing (which lets a saved tensor be asked for once): the same bits."""
    from torch.utils.checkpoint import checkpoint
    torch.manual_seed(0)
    q, k, g = (torch.randn(60, h, 64, device=dev).to(dtype) for h in (4, 2, 4))
    x, y = torch.randn(60, 50, device=dev), torch.randint(0, 50, (60,), device=dev)
    s, index = torch.rand(60, 8, device=dev), torch.randint(0, 8, (60, 2), device=dev)
    cu = torch.tensor([0, 20, 60], dtype=torch.int32, device=dev)

    def call(q, k, v, x, s):
        return ((packed.packed_attention(q, k, v, cu) * g).float().sum() + token_logprobs(x, y).sum()
                + preference_loss(x * 2, y, cu, torch.zeros(2, device=dev))[0] + balance_loss(s, index, 1.0, cu)[0])
    leaves = [t.clone().requires_grad_() for t in (q, k, k.flip(0), x, s)]
    want = torch.autograd.grad(call(*leaves), leaves)
    got = torch.autograd.grad(checkpoint(call, *leaves, use_reentrant=False), leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_batch_formed_inside_a_graph(dev):
    """A captured call takes other lengths on its next replay where its batch is formed inside:
    forward, losses and the cache's places, also of bounds that make no sense."""
    m = _model(dev).eval()
    cache = PackedCache(m.config, 3, 120, BF, dev)
    ids = torch.randint(0, 500, (1, 90), device=dev)
    cu = torch.tensor([0, 30, 60, 90], dtype=torch.int32, device=dev)

    def call():
        b = PackedBatch(cu, 90)
        out = m(ids, packed=b, labels=ids)
        cache.clear()
        kept = m(ids, packed=b, past_key_values=cache).logits
        return out.logits, out.loss, m.sequence_logprobs(ids, ids, b), kept, cache.lengths.clone()
    with torch.inference_mode():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = call()
        for ends in ([0, 1, 2, 90], [0, 0, 45, 80], [0, 30, 60, 90], [7, 50, 20, 300], [0, -9, 2 ** 31 - 1, 5]):
            cu.copy_(torch.tensor(ends, dtype=torch.int32))
            want = call()
            graph.replay()
            torch.cuda.synchronize()
            used = min(max(ends[-1], 0), 90) if ends[1:] == sorted(ends[1:]) else 0
            for a, w in zip(res, want):
                a, w = (t[:, :used] if t.dim() == 3 else t for t in (a, w))  # rows of no sequence: anything
                assert torch.equal(a.nan_to_num(), w.nan_to_num()), ends


@pytest.mark.gpu
def test_batch_made_in_inference_mode(dev):
    """Serves a training step afterwards: the reference model's pass comes first."""
    m = _model(dev, use_moe=True, num_experts_per_tok=2, use_mhc=0, router_aux_loss_per_sequence=True).train()
    ids = torch.randint(0, 500, (1, 160), device=dev)
    with torch.inference_mode():
        b = PackedBatch.from_lengths([50, 30, 10, 70], device=dev)
        ref = m.sequence_logprobs(ids, ids, b)
    m.preference_loss(ids, ids, b, ref).loss.backward()
    m(ids, packed=b, labels=ids).loss.backward()
