"""Packed sequences through the model on the GPU: the mHC model against each sequence alone,
decode steps over cache slots, a preference step of a routed-expert model with its
gradients; captured graphs, side streams, another current device."""
from __future__ import annotations

import copy

import pytest
import torch
import torch.nn.functional as F

from model import _ops, packed
from model.losses import balance_loss, preference_loss, token_logprobs
from model.model_minimind import MiniMindConfig, MiniMindForCausalLM, init_normal_
from model.packed import PackedBatch, PackedCache, packed_attention

BF = torch.bfloat16
LENGTHS = [70, 1, 33, 0, 150, 64]


def _model(dev, dtype=BF, **kw):
    torch.manual_seed(0)
    cfg = MiniMindConfig(hidden_size=192, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                         head_dim=64, intermediate_size=256, vocab_size=500, max_position_embeddings=512,
                         **{"use_mhc": 1, **kw})
    return init_normal_(MiniMindForCausalLM(cfg), 0.05).to(dev).to(dtype)


def _far(got, ref):
    return float((got.double() - ref.double()).norm() / ref.double().norm())


def _taken(monkeypatch):
    """Counts the calls of the packed kernels."""
    seen, run = [], packed.packed_attention
    monkeypatch.setattr(packed, "packed_attention", lambda *a, **k: seen.append(1) or run(*a, **k))
    return seen


@pytest.mark.gpu
@pytest.mark.parametrize("moe", [False, True])
def test_inference_matches_each_sequence(dev, monkeypatch, moe):
    """As far from the fp32 model as the sequences alone are: both round the same steps to
    bf16, in kernels that differ, so twice their distance bounds the packed call's."""
    m = _model(dev, use_moe=moe, num_experts=1 if moe else 4).eval()
    wide = copy.deepcopy(m).float()
    b = PackedBatch.from_lengths(LENGTHS, rows=sum(LENGTHS) + 5, device=dev)
    ids = torch.randint(0, 500, (1, b.rows), device=dev)
    seen = _taken(monkeypatch)
    with torch.inference_mode():
        got = m(ids, packed=b).logits[0]
        assert len(seen) == 2
        at = 0
        for n in LENGTHS:
            if n:
                ref = wide(ids[:, at:at + n]).logits[0]
                alone = _far(m(ids[:, at:at + n]).logits[0], ref)
                assert _far(got[at:at + n], ref) <= 2 * alone
            at += n
        assert torch.isfinite(got).all()
        torch.testing.assert_close(wide(ids, packed=b).logits[0, :70], wide(ids[:, :70]).logits[0],
                                   rtol=1e-3, atol=1e-3)


@pytest.mark.gpu
def test_decode_over_slots(dev, monkeypatch):
    m = _model(dev).eval()
    wide = copy.deepcopy(m).float()
    lengths, steps = [40, 3, 129], 4
    ids = [torch.randint(0, 500, (n + steps,), device=dev) for n in lengths]
    cache = PackedCache(m.config, 3, 160, BF, dev)
    seen = _taken(monkeypatch)
    with torch.inference_mode():
        out = m(torch.cat([x[:n] for x, n in zip(ids, lengths)])[None],
                packed=PackedBatch.from_lengths(lengths, device=dev), past_key_values=cache)
        last = [o[-1:] for o in out.logits[0].split(lengths)]
        step = PackedBatch.from_lengths([1] * 3, device=dev)
        for i in range(steps):
            out = m(torch.stack([x[n + i] for x, n in zip(ids, lengths)])[None], packed=step, past_key_values=cache)
            last = [torch.cat([a, o[None]]) for a, o in zip(last, out.logits[0])]
        assert len(seen) == 2 * (1 + steps) and cache.lengths.tolist() == [n + steps for n in lengths]
        for x, n, got in zip(ids, lengths, last):
            ref = wide(x[None]).logits[0, n - 1:]
            assert _far(got, ref) <= 2 * _far(m(x[None]).logits[0, n - 1:], ref)


def _reference_loss(m, ids, b, ref, lengths):
    """The preference loss from each sequence alone, on torch ops."""
    S, aux, at = [], 0.0, 0
    for n in lengths:
        out = m(ids[:, at:at + n])
        lp = torch.log_softmax(out.logits[0].float(), -1)
        S.append(lp[:-1].gather(1, ids[0, at + 1:at + n, None]).sum())
        at += n
    r = 0.1 * (torch.stack(S) - ref)
    return -F.logsigmoid(r[:2] - r[2:]).mean()


@pytest.mark.gpu
def test_preference_step(dev, monkeypatch):
    """A preference step of a routed-expert model under the trainers' autocast: loss and
    gradients are as far from those of an fp32 run as the sequences alone are, twice over."""
    lengths = [60, 31, 45, 80]
    m = _model(dev, torch.float32, use_moe=True, num_experts_per_tok=2, router_aux_loss_coef=0.0).train()
    b = PackedBatch.from_lengths(lengths, device=dev)
    ids = torch.randint(0, 500, (1, b.rows), device=dev)
    with torch.no_grad():
        ref = m.sequence_logprobs(ids, ids, b) + torch.tensor([1.0, -2.0, 3.0, 0.5], device=dev)
    names = [n for n, _ in m.named_parameters()]

    def grads(loss):
        g = torch.autograd.grad(loss, list(m.parameters()), allow_unused=True)
        return torch.cat([x.flatten() for n, x in zip(names, g) if x is not None and ".gate." not in n])
    exact_loss = _reference_loss(m, ids, b, ref, lengths)
    exact = grads(exact_loss)
    seen = _taken(monkeypatch)
    with torch.autocast("cuda", BF):
        alone = _reference_loss(m, ids, b, ref, lengths)
        g_alone = grads(alone)
        out = m.preference_loss(ids, ids, b, ref)
    assert len(seen) == 2 and out.loss.dtype == torch.float32
    assert abs(float(out.loss - exact_loss)) <= 2 * abs(float(alone - exact_loss)) + 2.0 ** -6
    assert _far(grads(out.loss), exact) <= 2 * _far(g_alone, exact)


@pytest.mark.gpu
@pytest.mark.parametrize("each", [False, True])
def test_router_balance_in_training(dev, each):
    m = _model(dev, torch.float32, use_moe=True, num_experts_per_tok=2, use_mhc=0, router_aux_loss_coef=0.5,
               router_aux_loss_per_sequence=each).train()
    cpu = copy.deepcopy(m).cpu()
    b = PackedBatch.from_lengths(LENGTHS, device=dev)
    ids = torch.randint(0, 500, (1, b.rows), device=dev)
    out = m(ids, packed=b, labels=ids)
    ref = cpu(ids.cpu(), packed=PackedBatch.from_lengths(LENGTHS, device="cpu"), labels=ids.cpu())
    # an expert chosen otherwise (fp32 scores a rounding apart) moves one count of 318
    assert abs(float(out.aux_loss) - float(ref.aux_loss)) <= 0.01 * float(ref.aux_loss)
    assert abs(float(out.loss) - float(ref.loss)) <= 1e-3 * float(ref.loss)
    moe = m.model.layers[0].mlp
    assert moe.expert_counts.shape == ((6, 4) if each else (4,)) and int(moe.expert_counts.sum()) == 2 * b.rows
    (out.loss + out.aux_loss).backward()
    assert float(moe.gate.weight.grad.abs().sum()) > 0


def _case(dev, seed):
    torch.manual_seed(seed)
    T = 300
    q, g = (torch.randn(T, 4, 96, device=dev).to(BF) for _ in range(2))
    k, v = (torch.randn(T, 2, 96, device=dev).to(BF) for _ in range(2))
    logits, labels = torch.randn(T, 333, device=dev).to(BF), torch.randint(0, 333, (T,), device=dev)
    scores, index = torch.rand(T, 8, device=dev), torch.randint(0, 8, (T, 2), device=dev)
    ends = sorted(torch.randint(0, T + 1, (3,)).tolist())
    cu = torch.tensor([0, *ends, T], dtype=torch.int32, device=dev)
    return [q, k, v, g, logits, labels, scores, index, cu]


def _all(q, k, v, g, logits, labels, scores, index, cu):
    """Every operator, forward and backward."""
    leaves = [t.detach().requires_grad_() for t in (q, k, v, logits, scores)]
    q, k, v, x, s = leaves
    out = packed_attention(q, k, v, cu)
    a = torch.autograd.grad(out, (q, k, v), g)
    with torch.no_grad():
        step = packed_attention(q[:4], k, v, cu.new_tensor([0, 1, 2, 3, 4]) if not torch.cuda.is_current_stream_capturing()
                                else _all.steps, cu_seqlens_k=cu)
    lp = token_logprobs(x, labels)
    b = torch.autograd.grad(lp.sum(), x)
    loss, c, r = preference_loss(x, labels, cu, torch.zeros(4, device=cu.device))
    d = torch.autograd.grad(loss, x)
    bal, counts = balance_loss(s, index, 0.1, cu)
    e = torch.autograd.grad(bal, s)
    return [t.detach() for t in (out, *a, step, lp, *b, loss, c, r, *d, bal, counts, *e)]


@pytest.mark.gpu
def test_captured_and_replayed(dev):
    """One graph of every operator, replayed on other inputs and other lengths, with eager
    work between: each replay has the eager result's bits."""
    state = _case(dev, 0)
    _all.steps = torch.arange(5, dtype=torch.int32, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _all(*state)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = _all(*state)
    for seed in (1, 2, 1, 3):
        new = _case(dev, seed)
        for t, n in zip(state, new):
            t.copy_(n)
        want = _all(*new)  # eager, between the replays
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, want)), seed


@pytest.mark.gpu
def test_side_stream_and_two_at_once(dev):
    a, b = _case(dev, 4), _case(dev, 5)
    want = [_all(*a), _all(*b)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for i, (s, c) in enumerate(zip(streams, (a, b))):
        with torch.cuda.stream(s):
            for _ in range(3):
                got[i] = _all(*c)
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(w, g))


@pytest.mark.gpu
def test_another_device_current(dev, monkeypatch):
    """Tensors of a device that is not the current one: the launches go to theirs."""
    case = _case(dev, 6)
    want, switched = _all(*case), []

    class Seen(torch.cuda.device):
        def __init__(self, d):
            switched.append(d)
            super().__init__(d)
    monkeypatch.setattr(_ops, "_current_device", lambda: 1)
    monkeypatch.setattr(torch.cuda, "device", Seen)
    got = _all(*case)
    assert len(switched) >= 9 and all(torch.device(d).index == 0 for d in switched)
    assert all(torch.equal(x, y) for x, y in zip(want, got))


@pytest.mark.gpu
def test_captured_decode_step(dev):
    """A decode step over cache slots in a graph: the slots' lengths move on with each replay."""
    m = _model(dev).eval()
    prompt = PackedBatch.from_lengths([9, 30], device=dev)
    step = PackedBatch.from_lengths([1, 1], device=dev)
    ids = torch.randint(0, 500, (6, 1, 2), device=dev)
    start = torch.randint(0, 500, (1, 39), device=dev)

    def fresh():
        cache = PackedCache(m.config, 2, 64, BF, dev)
        m(start, packed=prompt, past_key_values=cache)
        return cache
    with torch.inference_mode():
        eager = fresh()
        want = [m(x, packed=step, past_key_values=eager).logits.clone() for x in ids]
        cache = fresh()
        x = ids[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m(x, packed=step, past_key_values=cache)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(x, packed=step, past_key_values=cache).logits
        cache.clear()
        m(start, packed=prompt, past_key_values=cache)
        for w, i in zip(want, ids):
            x.copy_(i)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, w)
        assert cache.lengths.tolist() == [15, 36]


@pytest.mark.gpu
def test_forward_mode_and_double_backward_are_refused(dev):
    q, k, v, g, logits, labels, scores, index, cu = _case(dev, 7)
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        x = fwd.make_dual(logits.float(), torch.ones_like(logits, dtype=torch.float32))
        with pytest.raises(Exception):
            token_logprobs(x, labels)
    x = logits.float().requires_grad_()
    d, = torch.autograd.grad(token_logprobs(x, labels).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()
