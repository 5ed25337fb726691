"""Packed sequences: several of different lengths one after another in one tensor, without
padding, as a batch of prompts, of training documents, or of next tokens over caches that
have grown to different lengths.

No reference counterpart: the reference pads (model/model_minimind.py:161-256).
"""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _hip as H
from . import _ops

HEAD_DIMS = _ops.ATTN_HEAD_DIMS


def _bounds(name: str, t, n: Optional[int], dev: torch.device) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.dim() != 1:
        raise TypeError(f"mhc_amd: {name} must be a one-dimensional int32 tensor")
    if t.device != dev:
        raise RuntimeError(f"mhc_amd: {name} is on {t.device}, the tensors on {dev}")
    if t.numel() != n if n is not None else t.numel() < 1:
        raise ValueError(f"mhc_amd: {name} has {t.numel()} entries, expected "
                         f"{'at least 1' if n is None else n}")
    return t if t.is_contiguous() else t.contiguous()


def _strided(t: torch.Tensor):
    """(t, its row and head strides); a copy in order where the kernels cannot take t's."""
    row, head = (t.stride(i) if t.shape[i] > 1 else 0 for i in (0, 1))
    if t.stride(2) != 1 or row % 8 or head % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        row, head = t.shape[1] * t.shape[2], t.shape[2]
    return t, row, head


def _dims(q, k, v):
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 3:
            raise ValueError(f"mhc_amd: {name} must be [rows, heads, head_dim], got {tuple(t.shape)}")
    (Tq, heads, hd), (Tk, kv, _) = q.shape, k.shape
    if k.shape != v.shape or k.shape[2] != hd:
        raise ValueError(f"mhc_amd: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} "
                         "do not belong together")
    if hd not in HEAD_DIMS:
        raise ValueError(f"mhc_amd: head_dim must be one of {HEAD_DIMS}, got {hd}")
    if kv < 1 or heads < 1 or heads % kv:
        raise ValueError(f"mhc_amd: {heads} query heads are no multiple of {kv} key heads")
    if q.dtype not in _ops.HALF or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"mhc_amd: q, k and v must share bf16 or fp16, got {q.dtype}, {k.dtype}, {v.dtype}")
    return Tq, heads, hd, Tk, kv


def _forward(q, k, v, cu_q, cu_k, used, scale, graph):
    (q, *qs), (k, *ks), (v, *vs) = _strided(q), _strided(k), _strided(v)
    Tq, heads, hd = q.shape
    Tk, kv, B = k.shape[0], k.shape[1], cu_q.numel() - 1
    dev, lib = q.device, H.load()
    out = torch.empty((Tq, heads, hd), dtype=q.dtype, device=dev)
    rest = torch.empty_like(out) if graph else None
    lse = torch.empty((heads, Tq), dtype=torch.float32, device=dev) if graph else None
    with _ops.launch_device(q):
        nbytes = lib.mhc_packed_attn_workspace_bytes(B, Tq, Tk, heads, kv, hd)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes > 0 else None
        H.check(lib.mhc_packed_attn_fwd(
            q.data_ptr(), *qs, k.data_ptr(), *ks, v.data_ptr(), *vs, cu_q.data_ptr(), cu_k.data_ptr(),
            H.ptr(used), out.data_ptr(), H.ptr(rest), H.ptr(lse), H.ptr(ws), max(nbytes, 0), B, Tq, Tk,
            heads, kv, hd, H.dtype_tag(q), scale, H.stream(dev)), "mhc_packed_attn_fwd")
    return out, rest, lse


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, used, scale):
        out, rest, lse = _forward(q, k, v, cu_q, cu_k, used, scale, True)
        ctx.save_for_backward(q, k, v, cu_q, cu_k, used, out, rest, lse)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        q, k, v, cu_q, cu_k, used, out, rest, lse = ctx.saved_tensors
        (q, *qs), (k, *ks), (v, *vs) = _strided(q), _strided(k), _strided(v)
        g = g.to(out.dtype).contiguous()
        if g.data_ptr() % 16:  # a caller's view; the kernels load 16 bytes
            g = g.clone()
        Tq, heads, hd = q.shape
        Tk, kv = k.shape[:2]
        dev, new = q.device, torch.empty
        g_q = new((Tq, heads, hd), dtype=q.dtype, device=dev)
        g_k, g_v = (new((Tk, kv, hd), dtype=q.dtype, device=dev) for _ in range(2))
        delta = new((heads, Tq), dtype=torch.float32, device=dev)
        with _ops.launch_device(q):
            H.check(H.load().mhc_packed_attn_bwd(
                q.data_ptr(), *qs, k.data_ptr(), *ks, v.data_ptr(), *vs, cu_q.data_ptr(),
                cu_k.data_ptr(), H.ptr(used), out.data_ptr(), rest.data_ptr(), lse.data_ptr(), g.data_ptr(),
                delta.data_ptr(), g_q.data_ptr(), g_k.data_ptr(), g_v.data_ptr(), cu_q.numel() - 1,
                Tq, Tk, heads, kv, hd, H.dtype_tag(q), ctx.scale, H.stream(dev)), "mhc_packed_attn_bwd")
        return g_q, g_k, g_v, None, None, None, None


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     cu_seqlens_k: Optional[torch.Tensor] = None,
                     key_lengths: Optional[torch.Tensor] = None,
                     scale: Optional[float] = None) -> torch.Tensor:
    """Causal attention of each packed sequence over its own keys: [rows, heads, head_dim].

    q [rows, heads, head_dim], k and v [key rows, kv heads, head_dim]: bf16 or fp16,
    head_dim 64, 96 or 128, heads a multiple of the kv heads (query head h reads kv head
    h // (heads / kv heads)); any strides, though only those with contiguous heads on
    16-byte boundaries are read in place.  Under autocast they are cast to its type.
    cu_seqlens [n + 1] int32, on the same GPU: sequence i has the rows cu_seqlens[i] to
    cu_seqlens[i + 1] of q, beginning with row 0.
    cu_seqlens_k [n + 1]: the same for the rows of k and v (default: cu_seqlens).  A sequence
    with more keys than queries continues after a past: its last query sits at its last
    key.  One with more queries than keys leaves the first queries without a key.
    key_lengths [n] int32: only so many of the sequence's key rows are in use, as in a cache
    of slots that fill up; the rows behind them are not read.
    scale: a positive factor of the scores (default head_dim ** -0.5).

    Rows that see no key, and rows behind the last sequence, are 0, and so are the gradients
    of keys that no query sees.  The bounds stay on the device (no synchronisation; a
    captured graph takes other lengths on its next replay): they are clamped to the tensors,
    and bounds that decrease give unspecified rows.  Differentiable once; the gradients are
    the same bits on every run.
    """
    if torch.is_autocast_enabled("cuda"):
        low = torch.get_autocast_dtype("cuda")
        q, k, v = q.to(low), k.to(low), v.to(low)
    dev = H.require_device(q, k, v)
    Tq, heads, hd, Tk, kv = _dims(q, k, v)
    cu_q = _bounds("cu_seqlens", cu_seqlens, None, dev)
    if cu_seqlens_k is None:
        if Tk != Tq:
            raise ValueError(f"mhc_amd: {Tq} query rows and {Tk} key rows need a cu_seqlens_k")
        cu_k = cu_q
    else:
        cu_k = _bounds("cu_seqlens_k", cu_seqlens_k, cu_q.numel(), dev)
    used = None if key_lengths is None else _bounds("key_lengths", key_lengths, cu_q.numel() - 1, dev)
    scale = 1.0 / math.sqrt(hd) if scale is None else float(scale)
    if not (0.0 < scale < 3e38):
        raise ValueError(f"mhc_amd: scale must be positive, got {scale}")
    if _ops.wants_graph(q, k, v):
        return _PackedAttention.apply(q, k, v, cu_q, cu_k, used, scale)
    return _forward(q, k, v, cu_q, cu_k, used, scale, False)[0]
