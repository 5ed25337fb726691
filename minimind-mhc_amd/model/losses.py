"""Losses of language models on HIP kernels: log-probabilities of labels, the preference
loss of pairs of answers, and the balance loss of a router.

The reference forms them with chains of torch ops (trainer/train_dpo.py,
model/model_minimind.py:290-297 and :421-425).
"""
from __future__ import annotations

import functools
from typing import Optional

import torch

from . import _hip as H
from . import _ops
from .packed import _bounds

IGNORE_INDEX = -100
MAX_EXPERTS = 4096  # of balance_loss
_TYPES = (torch.float32, *_ops.HALF)


def takes(t: torch.Tensor) -> bool:
    """Whether the kernels take these logits or scores, in a call that nothing traces."""
    return t.is_cuda and t.dtype in _TYPES and _ops.eager_call()


def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    """t [..., V] as rows one stride apart, its last dimension in order."""
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError(f"mhc_amd: {name} must be [..., n] with n >= 1, got {tuple(t.shape)}")
    H.dtype_tag(t)
    try:
        t = t.view(-1, t.shape[-1]) if t.dim() != 2 else t
    except RuntimeError:  # rows that no one stride joins
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _labels(labels: torch.Tensor, logits: torch.Tensor) -> torch.Tensor:
    if labels.dtype != torch.int64:
        raise TypeError(f"mhc_amd: labels must be int64, got {labels.dtype}")
    if labels.shape != logits.shape[:-1]:
        raise ValueError(f"mhc_amd: labels {tuple(labels.shape)} do not belong to logits "
                         f"{tuple(logits.shape)}")
    return labels.reshape(-1).contiguous()


def _scalar(g: torch.Tensor) -> torch.Tensor:
    return g if g.dtype == torch.float32 else g.to(torch.float32)


def _stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _logprobs(x, labels, ignore, lp: int, lse: Optional[int]):
    """Writes the log-probabilities (and the rows' sums) to these addresses."""
    H.check(H.load().mhc_logprobs_fwd(x.data_ptr(), _stride(x), H.dtype_tag(x), labels.data_ptr(), ignore,
                                      lp, lse, x.shape[0], x.shape[1], H.stream(x.device)), "mhc_logprobs_fwd")


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, labels, ignore):
        T, dev = x.shape[0], x.device
        lp = torch.empty(T, dtype=torch.float32, device=dev)
        lse = torch.empty((T, 2), dtype=torch.float32, device=dev) if ctx is not None else None
        with _ops.launch_device(x):
            _logprobs(x, labels, ignore, lp.data_ptr(), H.ptr(lse))
        if ctx is not None:
            ctx.save_for_backward(x, labels, lse)
            ctx.ignore = ignore
        return lp

    @staticmethod
    def backward(ctx, grad):
        x, labels, lse = ctx.saved_tensors
        T, V = x.shape
        g = grad.detach().to(torch.float32).contiguous()
        out = torch.empty((T, V), dtype=x.dtype, device=x.device)
        with _ops.launch_device(x):
            H.check(H.load().mhc_logprobs_bwd(
                x.data_ptr(), _stride(x), H.dtype_tag(x), labels.data_ptr(), ctx.ignore, lse.data_ptr(),
                g.data_ptr(), out.data_ptr(), T, V, H.stream(x.device)), "mhc_logprobs_bwd")
        return (*_ops.once((out,), x, grad), None, None)


def token_logprobs(logits: torch.Tensor, labels: torch.Tensor,
                   ignore_index: int = IGNORE_INDEX) -> torch.Tensor:
    """log softmax(logits)[label] of each row, fp32, in labels' shape.

    logits [..., V] fp32, bf16 or fp16 (rows any stride apart); labels [...] int64.  A row
    whose label is ignore_index gets 0 (and no gradient, and is not read); a label outside
    [0, V) otherwise gives NaN.  Differentiable once in logits; the gradient has logits' type.
    """
    H.require_device(logits, labels)
    x, y = _rows(logits, "logits"), _labels(labels, logits)
    if _ops.wants_graph(logits):
        lp = _TokenLogprobs.apply(x, y, int(ignore_index))
    else:
        lp = _TokenLogprobs.forward(None, x, y, int(ignore_index))
    return lp.view(labels.shape)


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, labels, cu, reference, beta, smoothing, average, ignore):
        T, P, dev = x.shape[0], reference.numel() // 2, x.device
        new, f32 = torch.empty, torch.float32
        loss, rewards = new((), dtype=f32, device=dev), new((2, P), dtype=f32, device=dev)
        rows = new((3 if ctx is not None else 1) * T, dtype=f32, device=dev)  # log-probabilities, and their sums
        seqs = new(4 * P, dtype=f32, device=dev)  # g_seq, and the pairs' losses (64 bits)
        lse = rows.data_ptr() + 4 * T if ctx is not None else None
        r, g = rewards.data_ptr(), seqs.data_ptr()
        with _ops.launch_device(x):
            _logprobs(x, labels, ignore, rows.data_ptr(), lse)
            H.check(H.load().mhc_preference_fwd(
                rows.data_ptr(), labels.data_ptr(), ignore, cu.data_ptr(), reference.data_ptr(),
                loss.data_ptr(), r, r + 4 * P, g, g + 8 * P, T, P, beta, smoothing,
                int(average) | (2 if reference.dtype == torch.float64 else 0),
                H.stream(dev)), "mhc_preference_fwd")
        chosen, rejected = rewards.unbind(0)
        if ctx is not None:
            ctx.save_for_backward(x, labels, cu, rows, seqs)
            ctx.ignore = ignore
            ctx.mark_non_differentiable(chosen, rejected)
            ctx.set_materialize_grads(False)
        return loss, chosen, rejected

    @staticmethod
    def backward(ctx, grad, *_):
        if grad is None:
            return (None,) * 8
        x, labels, cu, rows, seqs = ctx.saved_tensors
        T, V = x.shape
        g = _scalar(grad.detach())
        out = torch.empty((T, V), dtype=x.dtype, device=x.device)
        with _ops.launch_device(x):
            H.check(H.load().mhc_preference_bwd(
                x.data_ptr(), _stride(x), H.dtype_tag(x), labels.data_ptr(), ctx.ignore,
                rows.data_ptr() + 4 * T, cu.data_ptr(), seqs.data_ptr(), g.data_ptr(), out.data_ptr(), T, V,
                seqs.numel() // 4, H.stream(x.device)), "mhc_preference_bwd")
        return (*_ops.once((out,), x, grad),) + (None,) * 7


def _check_pairs(reference: torch.Tensor, label_smoothing: float) -> None:
    if reference.dim() != 1 or reference.numel() < 2 or reference.numel() % 2:
        raise ValueError(f"mhc_amd: reference must hold two values a pair, got {tuple(reference.shape)}")
    if not 0.0 <= label_smoothing < 1.0:
        raise ValueError(f"mhc_amd: label_smoothing must be in [0, 1), got {label_smoothing}")


def preference_loss(logits: torch.Tensor, labels: torch.Tensor, cu_seqlens: torch.Tensor,
                    reference: torch.Tensor, beta: float = 0.1, label_smoothing: float = 0.0,
                    average: bool = False, ignore_index: int = IGNORE_INDEX):
    """(loss, chosen rewards [n], rejected rewards [n]) of n pairs of packed answers, fp32.

    logits [rows, V] fp32, bf16 or fp16; labels [rows] int64, ignore_index where a row does
    not count (a prompt).  cu_seqlens [2 n + 1] int32: the first n sequences are the chosen
    answers, the last n the rejected ones, in the same order; sequence i has the rows
    cu_seqlens[i] to cu_seqlens[i + 1], beginning with row 0, and rows behind the last count
    for nothing.  reference [2 n]: the reference model's sums (average: means) of the
    sequences' token_logprobs, in 64 bits or taken to 32.

    With S a sequence's sum (mean over its counted rows) of token_logprobs, its reward is
    beta (S - reference); with z the chosen reward less the rejected one, the loss is the
    mean over the pairs of -((1 - e) log sigmoid(z) + e log sigmoid(-z)), e = label_smoothing.
    The sums are taken in 64 bits.  The loss is differentiable once, in logits; the rewards
    carry no gradient.
    """
    dev = H.require_device(logits, labels, reference)
    if logits.dim() != 2:
        raise ValueError(f"mhc_amd: logits must be [rows, V], got {tuple(logits.shape)}")
    x, y = _rows(logits, "logits"), _labels(labels, logits)
    _check_pairs(reference, label_smoothing)
    cu = _bounds("cu_seqlens", cu_seqlens, reference.numel() + 1, dev)
    ref = reference.detach()
    ref = (ref if ref.dtype == torch.float64 else ref.to(torch.float32)).contiguous()
    args = (x, y, cu, ref, float(beta), float(label_smoothing), bool(average), int(ignore_index))
    if _ops.wants_graph(logits):
        return _PreferenceLoss.apply(*args)
    return _PreferenceLoss.forward(None, *args)


@functools.lru_cache(maxsize=1024)
def _balance_workspace(T: int, E: int, B: int) -> int:
    return max(H.load().mhc_balance_workspace_bytes(T, E, B), 0)


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, index, cu, coef):
        T, E = scores.shape
        B = 1 if cu is None else cu.numel() - 1
        dev, new, lib = scores.device, torch.empty, H.load()
        loss = new((), dtype=torch.float32, device=dev)
        counts = new(E if cu is None else (B, E), dtype=torch.int64, device=dev)
        with _ops.launch_device(scores):
            nbytes = _balance_workspace(T, E, B)
            ws = new(nbytes + 16, dtype=torch.uint8, device=dev)  # the sequences with rows, then the partial sums
            H.check(lib.mhc_balance_fwd(
                scores.data_ptr(), _stride(scores), H.dtype_tag(scores), index.data_ptr(), H.ptr(cu),
                loss.data_ptr(), counts.data_ptr(), ws.data_ptr(), ws.data_ptr() + 16, nbytes,
                T, E, index.shape[1], B, coef, H.stream(dev)), "mhc_balance_fwd")
        if ctx is not None:
            ctx.save_for_backward(cu, counts, ws)
            ctx.shape, ctx.dtype, ctx.coef = (T, E), scores.dtype, coef
            ctx.mark_non_differentiable(counts)
            ctx.set_materialize_grads(False)
        return loss, counts

    @staticmethod
    def backward(ctx, grad, *_):
        if grad is None:
            return (None,) * 4
        cu, counts, ws = ctx.saved_tensors
        (T, E), g = ctx.shape, _scalar(grad.detach())
        again = torch.is_grad_enabled() and grad.requires_grad  # the scores do not enter, only grad does
        if again:
            g = torch.ones_like(g)
        out = torch.empty((T, E), dtype=torch.float32 if again else ctx.dtype, device=counts.device)
        with _ops.launch_device(counts):
            H.check(H.load().mhc_balance_bwd(
                H.ptr(cu), counts.data_ptr(), ws.data_ptr(), g.data_ptr(), out.data_ptr(),
                H.dtype_tag(out), T, E, counts.numel() // E, ctx.coef, H.stream(counts.device)),
                "mhc_balance_bwd")
        return (out * grad).to(ctx.dtype) if again else out, None, None, None


def balance_loss(scores: torch.Tensor, index: torch.Tensor, coef: float,
                 cu_seqlens: Optional[torch.Tensor] = None):
    """(loss, counts) of a router: coef E sum_e f_e P_e over E experts, f_e the times expert e
    was taken divided by the number of tokens, P_e its mean score.

    scores [..., E] fp32, bf16 or fp16, the router's probabilities; index [..., k] int64, the
    experts each token went to.  counts [E] int64: how often each was taken.  loss: fp32,
    differentiable in scores, as often as wanted (counts are constants).
    cu_seqlens [n + 1] int32: the mean over the sequences (rows cu_seqlens[i] to
    cu_seqlens[i + 1], beginning with row 0) of each one's own loss instead, and counts
    [n, E].  Sequences without rows do not enter the mean; rows behind the last are
    in none.  Without any row the loss is 0.
    """
    dev = H.require_device(scores, index)
    x = _rows(scores, "scores")
    if index.dtype != torch.int64:
        raise TypeError(f"mhc_amd: index must be int64, got {index.dtype}")
    if index.dim() != scores.dim() or index.shape[:-1] != scores.shape[:-1] or index.shape[-1] < 1:
        raise ValueError(f"mhc_amd: index {tuple(index.shape)} does not belong to scores {tuple(scores.shape)}")
    idx = index.reshape(-1, index.shape[-1]).contiguous()
    cu = None if cu_seqlens is None else _bounds("cu_seqlens", cu_seqlens, None, dev)
    if _ops.wants_graph(scores):
        return _BalanceLoss.apply(x, idx, cu, float(coef))
    return _BalanceLoss.forward(None, x, idx, cu, float(coef))
