"""Rotary positions of queries and keys on HIP kernels: pairs in halves or interleaved, the
whole head or its first part, any table of angles.

The reference turns whole heads in halves with chains of torch ops
(model/model_minimind.py:132-160).
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _hip as H
from . import _ops


def _tables(cos: torch.Tensor, sin: torch.Tensor, head_dim: int):
    """(cos, sin, row stride) of tables [positions, rotary_dim / 2]."""
    shape = cos.shape
    if len(shape) != 2 or shape != sin.shape or cos.dtype != sin.dtype:
        raise ValueError(f"mhc_amd: cos {tuple(shape)} and sin {tuple(sin.shape)} must be alike, "
                         "[positions, rotary_dim / 2]")
    if 2 * shape[1] > head_dim:
        raise ValueError(f"mhc_amd: tables of {shape[1]} angles for heads of {head_dim}")
    H.dtype_tag(cos)
    stride = cos.stride()
    if stride != sin.stride() or shape[1] > 1 and stride[1] != 1:
        cos, sin = cos.contiguous(), sin.contiguous()
        stride = cos.stride()
    return cos, sin, stride[0] if shape[0] > 1 else shape[1]


def _rows(t: torch.Tensor, rows: int):
    """t [..., heads, head_dim] as (t [rows, heads, head_dim], row stride, head stride)."""
    if t.dim() != 3:
        try:
            t = t.view(rows, t.shape[-2], t.shape[-1])
        except RuntimeError:  # rows that no one stride joins
            t = t.reshape(rows, t.shape[-2], t.shape[-1])
    row, head, one = t.stride()
    if one != 1 and t.shape[2] > 1:
        t = t.contiguous()
        row, head, one = t.stride()
    return t, row, head


def _turn(q, k, cos, sin, stride, positions, flags):
    rows, shape, dev = positions.numel(), q.shape, q.device
    q3, *qs = _rows(q, rows)
    out_q, out_k, k3, ks, kv = torch.empty(shape, dtype=q.dtype, device=dev), None, None, (0, 0), 0
    if k is not None:
        k3, *ks = _rows(k, rows)
        out_k, kv = torch.empty(k.shape, dtype=q.dtype, device=dev), k.shape[-2]
    with _ops.launch_device(q):
        H.check(H.load().mhc_rotary(
            q3.data_ptr(), *qs, H.ptr(k3), *ks, cos.data_ptr(), sin.data_ptr(), stride, cos.shape[0],
            H.dtype_tag(cos), positions.data_ptr(), positions.element_size(), out_q.data_ptr(), H.ptr(out_k),
            rows, shape[-2], kv, shape[-1], 2 * cos.shape[1], flags, H.dtype_tag(q), H.stream(dev)),
            "mhc_rotary")
    return out_q, out_k


class _Rotary(torch.autograd.Function):
    """A linear map: its backward pass is the transposed one, itself a _Rotary."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, stride, positions, flags):
        ctx.save_for_backward(cos, sin, positions)
        ctx.stride, ctx.flags = stride, flags
        ctx.set_materialize_grads(False)
        return _turn(q, k, cos, sin, stride, positions, flags)

    @staticmethod
    def backward(ctx, gq, gk):
        cos, sin, positions = ctx.saved_tensors
        back = (cos, sin, ctx.stride, positions, ctx.flags ^ 2)
        if gq is None:
            if gk is not None:
                gk = _apply(gk, None, *back)[0]
        else:
            gq, gk = _apply(gq, gk, *back)
        return gq, gk, None, None, None, None, None


def _apply(q, k, *args):
    if _ops.wants_graph(q, q if k is None else k):
        return _Rotary.apply(q, k, *args)
    return _turn(q, k, *args)


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], cos: torch.Tensor, sin: torch.Tensor,
           positions: torch.Tensor, interleaved: bool = False):
    """(q, k) turned by their rows' positions, in their type: contiguous tensors of their shapes.

    q [..., heads, head_dim], k [..., kv heads, head_dim] (or None): fp32, bf16 or fp16, any
    head_dim, any strides (those with a head's elements in order are read in place).
    cos, sin [positions, rotary_dim / 2] fp32, bf16 or fp16: the angles, with whatever scaling
    they are to have.  The first rotary_dim elements of a head are pairs, in halves (d, d +
    rotary_dim / 2) or interleaved (2 d, 2 d + 1): (a, b) becomes (a c - b s, b c + a s); the others
    stay.  positions [...] int32 or int64: each row's row of the tables; the pairs of a row whose
    position lies outside them are NaN.

    Differentiable in q and k, as often as wanted; the tables are constants.
    """
    dev = H.require_device(q, k, cos, sin, positions)
    H.dtype_tag(q)
    if q.dim() < 2 or k is not None and (k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]):
        raise ValueError(f"mhc_amd: q {tuple(q.shape)} and k {None if k is None else tuple(k.shape)} do not belong together")
    if k is not None and k.dtype != q.dtype:
        raise TypeError(f"mhc_amd: q and k must share a type, got {q.dtype} and {k.dtype}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"mhc_amd: positions must be int32 or int64, got {positions.dtype}")
    if positions.shape != q.shape[:-2]:
        raise ValueError(f"mhc_amd: positions {tuple(positions.shape)} do not belong to q {tuple(q.shape)}")
    if torch.is_grad_enabled() and (cos.requires_grad or sin.requires_grad):
        raise RuntimeError("mhc_amd: the tables of rotary are constants; detach them")
    tables = _tables(cos, sin, q.shape[-1])
    positions = positions if positions.is_contiguous() else positions.contiguous()
    return _apply(q, k, *tables, positions, 1 if interleaved else 0)


def plain_rotary(q, k, cos, sin, positions, interleaved: bool = False):
    """rotary on torch ops, for what the kernel does not take (the CPU, traced calls)."""
    rd, table = 2 * cos.shape[1], cos.shape[0]
    at = positions.clamp(0, max(table - 1, 0))
    lost = ((positions < 0) | (positions >= table))[..., None, None]
    c, s = (t[at].unsqueeze(-2).to(torch.promote_types(t.dtype, torch.float32)) for t in (cos, sin))

    def turn(x):
        y = x[..., :rd]
        a, b = (y[..., 0::2], y[..., 1::2]) if interleaved else y.chunk(2, -1)
        a, b = a * c - b * s, b * c + a * s
        y = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
        return torch.cat([y.masked_fill(lost, float("nan")).to(x.dtype), x[..., rd:]], -1)
    return turn(q), None if k is None else turn(k)
