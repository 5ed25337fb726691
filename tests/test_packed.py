"""Packed sequences without a GPU: refusals, the batch's bookkeeping, the model's torch path
against each sequence alone, and the 64-bit oracle of the GPU tests against differences."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from model import losses
from model.model_minimind import Attention, MiniMindConfig, MiniMindForCausalLM, init_normal_
from model.packed import PackedBatch, PackedCache, PackedCall, _plain_attention, packed_attention
from tests.test_gpu_packed import exact


def _config(**kw):
    kw = {"hidden_size": 64, "num_hidden_layers": 2, "num_attention_heads": 4, "num_key_value_heads": 2,
          "head_dim": 16, "intermediate_size": 96, "vocab_size": 50, "max_position_embeddings": 128, **kw}
    return MiniMindConfig(**kw)


def _model(**kw):
    torch.manual_seed(0)
    return init_normal_(MiniMindForCausalLM(_config(**kw)), 0.2)


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32)


# ------------------------------------------------------------------- refusals

def test_no_cpu_path():
    q, kv = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.zeros(4, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        packed_attention(q, kv, kv, _ints(0, 4))
    x, y = torch.zeros(4, 10), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        losses.token_logprobs(x, y)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        losses.preference_loss(x, y, _ints(0, 2, 4), torch.zeros(2))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        losses.balance_loss(x, y[:, None], 0.1)


@pytest.fixture
def anywhere(monkeypatch):
    """The checks that come after the device's."""
    from model import _hip
    monkeypatch.setattr(_hip, "require_device", lambda *t: t[0].device)


@pytest.mark.parametrize("shape,kv,error", [
    ((4, 2, 80), (4, 1, 80), "head_dim"), ((4, 3, 64), (4, 2, 64), "no multiple"),
    ((4, 2, 64), (5, 2, 64), "need a cu_seqlens_k"), ((4, 2, 64), (4, 2, 96), "belong together"),
    ((4, 128), (4, 1, 64), "must be"), ((4, 2, 64), (4, 0, 64), "no multiple")])
def test_attention_refuses_shapes(anywhere, shape, kv, error):
    q, k = torch.zeros(shape, dtype=torch.bfloat16), torch.zeros(kv, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match=error):
        packed_attention(q, k, k, _ints(0, 4))


def test_attention_refuses(anywhere):
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    cu = _ints(0, 4)
    for bad in (q.float(), q.half()):
        with pytest.raises(TypeError, match="bf16 or fp16"):
            packed_attention(q, bad, bad, cu)
    with pytest.raises(TypeError, match="int32"):
        packed_attention(q, q, q, cu.long())
    with pytest.raises(TypeError, match="int32"):
        packed_attention(q, q, q, [0, 4])
    with pytest.raises(ValueError, match="at least 1"):
        packed_attention(q, q, q, cu[:0])
    with pytest.raises(ValueError, match="expected 2"):
        packed_attention(q, q, q, cu, cu_seqlens_k=_ints(0, 2, 4))
    with pytest.raises(ValueError, match="expected 1"):
        packed_attention(q, q, q, cu, key_lengths=_ints(2, 2))
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="scale"):
            packed_attention(q, q, q, cu, scale=scale)


def test_losses_refuse(anywhere):
    x, y, cu = torch.zeros(4, 10), torch.zeros(4, dtype=torch.int64), _ints(0, 2, 4)
    with pytest.raises(TypeError, match="int64"):
        losses.token_logprobs(x, y.int())
    with pytest.raises(ValueError, match="belong"):
        losses.token_logprobs(x, y[:3])
    with pytest.raises(TypeError, match="unsupported dtype"):
        losses.token_logprobs(x.double(), y)
    with pytest.raises(ValueError, match="n >= 1"):
        losses.token_logprobs(x[:, :0], y)
    with pytest.raises(ValueError, match="rows, V"):
        losses.preference_loss(x[None], y[None], cu, torch.zeros(2))
    for ref in (torch.zeros(3), torch.zeros(0), torch.zeros(2, 1)):
        with pytest.raises(ValueError, match="two values a pair"):
            losses.preference_loss(x, y, cu, ref)
    with pytest.raises(ValueError, match="expected 5"):
        losses.preference_loss(x, y, cu, torch.zeros(4))
    for e in (-0.1, 1.0, math.nan):
        with pytest.raises(ValueError, match="label_smoothing"):
            losses.preference_loss(x, y, cu, torch.zeros(2), label_smoothing=e)
    with pytest.raises(TypeError, match="int64"):
        losses.balance_loss(x, y[:, None].int(), 0.1)
    for index in (y, y[:3, None], y[:, None][:, :0]):
        with pytest.raises(ValueError, match="belong"):
            losses.balance_loss(x, index, 0.1)


def test_library_refuses():
    """Bad arguments come back as errors before any device work, not as aborts."""
    from model import _hip
    lib = _hip.load()
    p = ctypes.c_void_p(16)

    def attn(B=1, Tq=4, Tk=4, heads=2, kv=1, hd=64, dtype=1, scale=0.1, st=128, ptr=p, rest=None, lse=None):
        return lib.mhc_packed_attn_fwd(ptr, st, 64, ptr, 64, 64, ptr, 64, 64, p, p, None, ptr, rest, lse, None, 0, B,
                                       Tq, Tk, heads, kv, hd, dtype, scale, None)
    for kw in ({"B": -1}, {"Tq": -1}, {"Tq": 1 << 31}, {"Tk": (1 << 30) + 1}, {"heads": 3, "kv": 2}, {"hd": 80},
               {"dtype": 0}, {"scale": 0.0}, {"scale": float("nan")}, {"st": 12}, {"ptr": None},
               {"ptr": ctypes.c_void_p(8)}, {"lse": p}, {"st": 1 << 24}, {"Tq": 1 << 30, "heads": 64}):
        assert attn(**kw) != 0 and lib.mhc_last_error()
    assert lib.mhc_packed_attn_workspace_bytes(1, 4, 4, 2, 1, 80) == -1
    assert lib.mhc_logprobs_fwd(None, 10, 0, p, -100, p, None, 4, 10, None) != 0
    assert lib.mhc_logprobs_fwd(p, 10, 7, p, -100, p, None, 4, 10, None) != 0
    assert lib.mhc_logprobs_fwd(p, 10, 0, p, -100, p, None, 4, 0, None) != 0
    assert lib.mhc_logprobs_fwd(ctypes.c_void_p(18), 10, 0, p, -100, p, None, 4, 10, None) != 0
    assert lib.mhc_preference_fwd(p, p, -100, p, p, p, p, p, p, p, 4, 0, 0.1, 0.0, 0, None) != 0
    assert lib.mhc_balance_workspace_bytes(4, 4097, 1) == -1
    assert lib.mhc_balance_fwd(p, 8, 0, p, None, p, p, p, p, 1 << 20, 4, 8, 2, 2, 0.1, None) != 0
    assert lib.mhc_balance_fwd(p, 8, 0, p, None, p, p, p, p, 8, 4, 8, 2, 1, 0.1, None) != 0


# ------------------------------------------------------------------- bookkeeping

def test_batch():
    b = PackedBatch.from_lengths([3, 0, 2], rows=7, device="cpu")
    assert len(b) == 3 and b.longest == 3 and b.cu_seqlens.tolist() == [0, 3, 3, 5]
    assert b.sequence.tolist() == [0, 0, 0, 2, 2, 3, 3]
    assert b.positions.tolist()[:5] == [0, 1, 2, 0, 1]
    y = torch.arange(7)[None]
    assert b.next_labels(y).tolist() == [[1, 2, -100, 4, -100, -100, -100]]
    for bad in (dict(lengths=[3, -1]), dict(lengths=[3], rows=2)):
        with pytest.raises(ValueError):
            PackedBatch.from_lengths(**bad, device="cpu")
    with pytest.raises(ValueError):
        b.next_labels(y[:, :6])
    empty = PackedBatch.from_lengths([0], device="cpu")
    assert empty.next_labels(torch.zeros(1, 0, dtype=torch.int64)).shape == (1, 0)


def test_cache_rows():
    cfg = _config()
    cache = PackedCache(cfg, 2, 4, torch.float32, "cpu")
    call = PackedCall(PackedBatch.from_lengths([3, 1], rows=6, device="cpu"), cache)
    assert call.rows.tolist() == [0, 1, 2, 4, 8, 8] and call.lengths.tolist() == [3, 1]
    call.done()
    with pytest.raises(ValueError, match="may not fit"):
        PackedCall(PackedBatch.from_lengths([1, 2], device="cpu"), cache)
    call = PackedCall(PackedBatch(_ints(0, 2, 3), 3), cache)  # lengths the host does not know
    assert call.rows.tolist() == [3, 8, 5] and call.lengths.tolist() == [4, 2]  # the second has no room
    assert call.positions.tolist() == [3, 4, 1]
    with pytest.raises(ValueError, match="on a cache of 2"):
        PackedCall(PackedBatch.from_lengths([1], device="cpu"), cache)
    cache.clear()
    assert cache.lengths.tolist() == [0, 0]
    for bad in ((0, 4), (2, 0)):
        with pytest.raises(ValueError):
            PackedCache(cfg, *bad, device="cpu")


def test_model_refuses():
    m, ids = _model(), torch.zeros(1, 5, dtype=torch.int64)
    b = PackedBatch.from_lengths([2, 3], device="cpu")
    with pytest.raises(ValueError, match="PackedBatch of"):
        m(ids[:, :4], packed=b)
    with pytest.raises(ValueError, match="PackedBatch of"):
        m(ids.view(5, 1), packed=b)
    with pytest.raises(ValueError, match="attention_mask"):
        m(ids, packed=b, attention_mask=torch.ones(1, 5))
    with pytest.raises(ValueError, match="PackedCache"):
        m(ids, packed=b, past_key_values=[(ids, ids)] * 2)
    with pytest.raises(ValueError, match="every row"):
        m(ids, packed=b, labels=ids, logits_to_keep=1)
    with pytest.raises(RuntimeError, match="no_grad"):
        m(ids, packed=b, past_key_values=PackedCache(m.config, 2, 8, torch.float32, "cpu"))


# ------------------------------------------------- the torch path, each sequence alone

@pytest.mark.parametrize("moe", [False, True])
def test_model_matches_each_sequence(moe):
    m = _model(use_moe=moe, num_experts_per_tok=2).eval()
    lengths = [5, 1, 9, 0, 4]
    b = PackedBatch.from_lengths(lengths, rows=22, device="cpu")
    ids = torch.randint(0, 50, (1, 22))
    out = m(ids, packed=b, labels=ids)
    total, count, at = 0.0, 0, 0
    for n in lengths:
        if n:
            one = m(ids[:, at:at + n], labels=ids[:, at:at + n] if n > 1 else None)
            torch.testing.assert_close(out.logits[:, at:at + n], one.logits, rtol=1e-4, atol=1e-4)
            if n > 1:
                total, count = total + float(one.loss) * (n - 1), count + n - 1
        at += n
    assert float(out.loss) == pytest.approx(total / count, rel=1e-5)
    lp = m.sequence_logprobs(ids, ids, b)
    assert float(lp.sum()) == pytest.approx(-total, rel=1e-5) and float(lp[1]) == float(lp[3]) == 0.0


def test_cached_steps_match_the_whole():
    m = _model().eval()
    lengths, more = [4, 2, 7], 3
    ids = [torch.randint(0, 50, (n + more,)) for n in lengths]
    whole = [m(x[None]).logits[0] for x in ids]
    cache = PackedCache(m.config, 3, 11, torch.float32, "cpu")
    with torch.no_grad():
        first = PackedBatch.from_lengths(lengths, device="cpu")
        out = m(torch.cat([x[:n] for x, n in zip(ids, lengths)])[None], packed=first, past_key_values=cache)
        assert out.past_key_values is cache
        got = list(out.logits[0].split(lengths))
        step = PackedBatch.from_lengths([1, 1, 1], device="cpu")
        for i in range(more):
            out = m(torch.stack([x[n + i] for x, n in zip(ids, lengths)])[None], packed=step, past_key_values=cache)
            got = [torch.cat([g, o[None]]) for g, o in zip(got, out.logits[0])]
    for g, w in zip(got, whole):
        torch.testing.assert_close(g, w, rtol=1e-4, atol=1e-4)
    assert cache.lengths.tolist() == [n + more for n in lengths]


def test_per_sequence_balance_loss():
    m = _model(use_moe=True, num_experts_per_tok=2, router_aux_loss_per_sequence=True).train()
    plain = _model(use_moe=True, num_experts_per_tok=2).train()
    x = torch.randn(3, 6, 64)
    for layer in (m.model.layers[0].mlp, plain.model.layers[0].mlp):
        layer(x)
    each = []
    for row in x:
        plain.model.layers[0].mlp(row[None])
        each.append(plain.model.layers[0].mlp.aux_loss)
    moe = m.model.layers[0].mlp
    torch.testing.assert_close(moe.aux_loss, torch.stack(each).mean())
    assert moe.expert_counts.shape == (3, 4) and int(moe.expert_counts.sum()) == 3 * 6 * 2


def test_plain_attention_and_oracle():
    """The layer's torch path, and the 64-bit oracle's gradients against differences."""
    torch.manual_seed(0)
    new, slots, used = [3, 1, 0, 4], [5, 7, 2, 3], [4, 6, 1, 2]
    q = torch.randn(8, 4, 16, dtype=torch.float64)
    k, v = (torch.randn(17, 2, 16, dtype=torch.float64) for _ in range(2))
    g = torch.randn_like(q)
    (out, *grads), _ = exact(q, k, v, new, slots, used, 0.25, g)
    got = _plain_attention(q, k, v, _ints(0, 3, 4, 4, 8), _ints(0, 5, 12, 14, 17), _ints(*used), 0.0)
    torch.testing.assert_close(got, out)
    for i, (t, grad) in enumerate(zip((q, k, v), grads)):
        d = torch.randn_like(t)
        ends = []
        for s in (1e-5, -1e-5):
            moved = [x + s * d if x is t else x for x in (q, k, v)]
            ends.append(float((exact(*moved, new, slots, used, 0.25)[0][0] * g).sum()))
        assert (ends[0] - ends[1]) / 2e-5 == pytest.approx(float((grad * d).sum()), rel=1e-6)


def test_attention_layer_signature_keeps_its_order():
    import inspect
    assert list(inspect.signature(Attention.forward).parameters)[:6] == [
        "self", "x", "position_embeddings", "past_key_value", "use_cache", "attention_mask"]
