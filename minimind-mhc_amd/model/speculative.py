"""Verification of drafted tokens against a target model's probabilities.

No reference counterpart: the reference decodes a token at a time
(eval_llm.py, trainer/train_grpo.py).
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _hip as H
from . import _ops
from .packed import _bounds

_TYPES = (torch.float32, *_ops.HALF)


def _row_ints(name: str, t: torch.Tensor, rows: int, dtype: torch.dtype) -> torch.Tensor:
    if t.dtype != dtype:
        raise TypeError(f"mhc_amd: {name} must be {dtype}, got {t.dtype}")
    if tuple(t.shape) != (rows,):
        raise ValueError(f"mhc_amd: {name} must be [{rows}], got {tuple(t.shape)}")
    return t.contiguous()


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t in order and on 16 bytes, as the kernel reads it."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _checked(probs, tokens, cu_seqlens, parents, draft_probs, uniforms, types, dev):
    """(tokens, parents, uniforms, cu_seqlens) of a call, checked and in order."""
    if probs.dim() != 2 or probs.shape[1] < 1:
        raise ValueError(f"mhc_amd: probs must be [rows, V], got {tuple(probs.shape)}")
    T = probs.shape[0]
    for name, t in (("probs", probs), ("draft_probs", draft_probs)):
        if t is not None and t.dtype not in types:
            raise TypeError(f"mhc_amd: {name} must be fp32, bf16 or fp16, got {t.dtype}")
    if draft_probs is not None:
        if draft_probs.shape != probs.shape:
            raise ValueError(f"mhc_amd: draft_probs {tuple(draft_probs.shape)} and probs {tuple(probs.shape)} differ")
        if uniforms is None:
            raise ValueError("mhc_amd: draft_probs need uniforms")
    tokens = _row_ints("tokens", tokens, T, torch.int64)
    if parents is not None:
        parents = _row_ints("parents", parents, T, torch.int32)
    if uniforms is not None:
        if not uniforms.is_floating_point() or tuple(uniforms.shape) != (T,):
            raise ValueError(f"mhc_amd: uniforms must be [{T}] floating point, got {tuple(uniforms.shape)} {uniforms.dtype}")
        uniforms = uniforms.detach().to(torch.float32).contiguous()
    return tokens, parents, uniforms, _bounds("cu_seqlens", cu_seqlens, None, dev)


def verify_drafts(probs: torch.Tensor, tokens: torch.Tensor, cu_seqlens: torch.Tensor,
                  parents: Optional[torch.Tensor] = None, draft_probs: Optional[torch.Tensor] = None,
                  uniforms: Optional[torch.Tensor] = None):
    """(kept [n] int32, path [rows] int32, next [n] int64) of n packed sequences' drafts.

    Sequence i has the rows cu_seqlens[i] to cu_seqlens[i + 1] (int32, beginning with row 0): its
    last token first, then its drafted ones, a tree.  tokens [rows] int64.
    parents [rows] int32: the place in its sequence of the token that a row follows, before its
    own (the first row's does not count, any other without such a parent is never accepted); None:
    each follows the one before it.
    probs [rows, V] fp32, bf16 or fp16: the target's probabilities after each row's token (greedy:
    logits will do).  draft_probs [rows, V]: those a row's children were drawn from, independently;
    None: the drafts were certain (siblings then differ, as a draft's most probable tokens do).
    uniforms [rows] in [0, 1): random numbers, one a drafted row and, in the first row, one for the
    next token; None: greedy.

    Sampled, kept rows and next token together are distributed as the target's own samples: at a
    node, with target p and draft q, a = 0 and c = 1, its children in turn (token x, number u) are
    accepted if u q(x) c < max(p(x) - a q(x), 0), else a += c and c = sum max(p - a q, 0); where none
    is left, next is the first token whose cumulated max(p - a q, 0) exceeds the first row's number
    times the total.  Certain drafts: accepted if u c < p(x), else c -= p(x), and x is out.  Greedy:
    accepted if x is the first of the most probable tokens.  In 64 bits; probabilities that are not
    positive finite numbers count as 0; where nothing is left next comes from p itself, and is -1
    where p has nothing either.

    kept: accepted rows of each sequence with the first one (0 without rows); path: their places
    in the sequence, in order, then -1.  Rows behind the last sequence keep -1.  Not differentiable.
    """
    dev = H.require_device(probs, tokens, parents, draft_probs, uniforms)
    tokens, parents, uniforms, cu = _checked(probs, tokens, cu_seqlens, parents, draft_probs, uniforms, _TYPES, dev)
    T, V = probs.shape
    probs, n = probs.detach(), cu.numel() - 1
    if draft_probs is not None:
        draft_probs = draft_probs.detach()
        if draft_probs.dtype != probs.dtype:
            probs, draft_probs = probs.float(), draft_probs.float()
        draft_probs = _aligned(draft_probs)
    probs = _aligned(probs)
    kept = torch.empty(n, dtype=torch.int32, device=dev)
    path = torch.empty(T, dtype=torch.int32, device=dev) if n else torch.full((T,), -1, dtype=torch.int32, device=dev)
    following = torch.empty(n, dtype=torch.int64, device=dev)
    with _ops.launch_device(probs):
        H.check(H.load().mhc_verify_drafts(
            probs.data_ptr(), H.ptr(draft_probs), H.dtype_tag(probs), tokens.data_ptr(), H.ptr(parents), H.ptr(uniforms),
            cu.data_ptr(), kept.data_ptr(), path.data_ptr(), following.data_ptr(), T, V, n, H.stream(dev)),
            "mhc_verify_drafts")
    return kept, path, following


def plain_verify(probs, tokens, cu_seqlens, parents=None, draft_probs=None, uniforms=None):
    """verify_drafts on the host, a sequence at a time, for tensors that are on no GPU (probabilities of
    64 bits too)."""
    tokens, parents, uniforms, cu = _checked(probs, tokens, cu_seqlens, parents, draft_probs, uniforms,
                                             (*_TYPES, torch.float64), probs.device)
    T, V = probs.shape
    ends = [0, *(min(max(e, 0), T) for e in cu.tolist()[1:])]
    tokens = tokens.tolist()
    up = parents.tolist() if parents is not None else None
    u = uniforms.double().tolist() if uniforms is not None else None
    p_all, q_all = (None if t is None else torch.where((t > 0) & torch.isfinite(t), t, 0).double() for t in (probs, draft_probs))
    path, kept, following = torch.full((T,), -1, dtype=torch.int32), [], []
    for a, b in zip(ends, ends[1:]):
        if b <= a:
            kept.append(0)
            following.append(-1)
            continue
        node, count, j = 0, 1, 0
        path[a] = 0

        def enter():
            best = -1
            if u is None:
                raw = probs[a + node].double()
                there = raw[~raw.isnan()]
                best = int((raw == there.max()).nonzero()[0]) if len(there) else -1
            return best, p_all[a + node].clone(), None if q_all is None else q_all[a + node], 0.0, 1.0
        best, p, q, ratio, norm = enter()
        for j in range(1, b - a):
            parent = j - 1 if up is None else up[a + j]
            if parent != node:
                continue
            x = tokens[a + j]
            inside = 0 <= x < V
            if u is None:
                good = inside and x == best
            else:
                px, qx = float(p[x]) if inside else 0.0, 1.0 if q is None else float(q[x]) if inside else 0.0
                good = u[a + j] * qx * norm < max(px - ratio * (0.0 if q is None else qx), 0.0)
            if good:
                node = j
                path[a + count] = j
                count += 1
                best, p, q, ratio, norm = enter()
            elif q is not None:
                ratio += norm
                norm = float((p - ratio * q).clamp_min(0).sum())
            elif u is not None and inside:
                norm = max(norm - px, 0.0)
                p[x] = 0.0
        if u is not None:
            w = p if q is None else (p - ratio * q).clamp_min(0)
            if not float(w.sum()) > 0:
                w = p_all[a + node]
            run = w.cumsum(0)
            past = ((run > u[a] * run[-1]) & (w > 0)).nonzero()
            some = (w > 0).nonzero()
            best = int(past[0]) if len(past) else int(some[-1]) if len(some) else -1
        kept.append(count)
        following.append(best)
    return torch.tensor(kept, dtype=torch.int32), path, torch.tensor(following, dtype=torch.int64)


def verify(probs, tokens, cu_seqlens, parents=None, draft_probs=None, uniforms=None):
    """verify_drafts; on the host (a synchronisation) where there is no GPU or a type that the kernel does not take."""
    if probs.is_cuda and all(t is None or t.dtype in _TYPES for t in (probs, draft_probs)):
        return verify_drafts(probs, tokens, cu_seqlens, parents, draft_probs, uniforms)
    args = (None if t is None else t.detach().cpu() for t in (probs, tokens, cu_seqlens, parents, draft_probs, uniforms))
    return tuple(t.to(probs.device) for t in plain_verify(*args))
