"""A cache of pages for packed sequences, and what reads and writes it: new tokens normed,
rotated and stored on the way, attention of single tokens, chunks of prompts or drafted trees,
and the accepted branch of a tree moved into place.

No reference counterpart: the reference grows dense caches by copies
(model/model_minimind.py:196-200).
"""
from __future__ import annotations

import functools
import math
from typing import Optional

import torch

from . import _hip as H
from . import _ops
from .packed import HEAD_DIMS, PackedBatch, _bounds
from .rotary import _rows, _tables, plain_rotary


def _no_graph(what: str, *ts) -> None:
    if _ops.wants_graph(*(t for t in ts if t is not None)):
        raise RuntimeError(f"mhc_amd: {what} is for inference; call under torch.no_grad()")


def _pages(k_pages: torch.Tensor, v_pages: torch.Tensor, hd: int):
    """(pages, page, kv heads, strides of page, row and head) of the cache's two tensors."""
    shape, strides = k_pages.shape, k_pages.stride()
    if len(shape) != 4 or shape != v_pages.shape or k_pages.dtype != v_pages.dtype or strides != v_pages.stride():
        raise ValueError(f"mhc_amd: k_pages {tuple(shape)} {k_pages.dtype} (strides {strides}) and v_pages "
                         f"{tuple(v_pages.shape)} {v_pages.dtype} ({v_pages.stride()}) must be alike, "
                         "[pages, page, kv heads, head_dim]")
    if k_pages.dtype not in _ops.HALF:
        raise TypeError(f"mhc_amd: pages hold bf16 or fp16, not {k_pages.dtype}")
    n, page, kv, dim = shape
    if page < 16 or page & (page - 1):
        raise ValueError(f"mhc_amd: a page must have a power of two of at least 16 rows, got {page}")
    if dim != hd:
        raise ValueError(f"mhc_amd: heads of {hd} and pages of {dim}")
    p, t, h, one = strides
    if one != 1 or (p | t | h) % 8 or t >= 1 << 23 or (k_pages.data_ptr() | v_pages.data_ptr()) % 16:
        raise ValueError(f"mhc_amd: pages must have heads in order on 16 bytes (strides {strides})")
    return n, page, kv, p, t, h


def _written(*ts: torch.Tensor) -> None:
    """Tells autograd that a kernel has written these tensors in place."""
    for t in ts:
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _table(page_table: torch.Tensor, n: int, dev: torch.device) -> torch.Tensor:
    if page_table.dtype != torch.int32 or page_table.dim() != 2:
        raise TypeError("mhc_amd: page_table must be a two-dimensional int32 tensor")
    if page_table.get_device() != dev.index:
        raise RuntimeError(f"mhc_amd: page_table is on {page_table.device}, the tensors on {dev}")
    if page_table.shape[0] != n:
        raise ValueError(f"mhc_amd: a page_table of {page_table.shape[0]} sequences for {n}")
    return page_table if page_table.is_contiguous() else page_table.contiguous()


def paged_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 page_table: torch.Tensor, lengths: torch.Tensor, cu_seqlens: torch.Tensor, cos: torch.Tensor,
                 sin: torch.Tensor, depths: Optional[torch.Tensor] = None, q_gain: Optional[torch.Tensor] = None,
                 k_gain: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False) -> torch.Tensor:
    """Stores the new tokens' keys and values, and returns their queries rotated: [rows, heads,
    head_dim].

    q [rows, heads, head_dim], k and v [rows, kv heads, head_dim]: the projections, in the pages'
    type, any strides (those with a head's elements in order are read in place).
    k_pages, v_pages [pages, page, kv heads, head_dim] bf16 or fp16, written in place: the same strides,
    of whole 16 bytes, a page a power of two of at least 16 rows.  page_table [n, width] int32: key x
    of sequence i lies in page page_table[i, x // page], row x % page.
    cu_seqlens [n + 1] int32: sequence i has the new rows cu_seqlens[i] to cu_seqlens[i + 1],
    beginning with row 0; lengths [n] int32: the keys it has before them.  Row j of them becomes key
    lengths[i] + j, at position lengths[i] + depths[row] (int32 [rows]; None: lengths[i] + j).
    q_gain, k_gain [head_dim]: with one, that tensor's heads get an RMSNorm (eps) before the
    rotation.  cos, sin, interleaved: as in rotary; a position outside the tables makes NaN of a
    row's pairs, in q and in the stored key.

    Rows of no sequence come out 0 and store nothing; nor do rows past width pages, or whose page
    number is none of the pages.  Nothing else in the pages changes.  Two sequences must not share
    the pages of their new rows.  All of it is read on the device: a captured graph takes other
    lengths and pages on its replays.
    """
    dev = H.require_device(q, k, v, k_pages, v_pages, cos, sin, depths, q_gain, k_gain)
    _no_graph("paged_append", q, k, v, k_pages, v_pages, q_gain, k_gain, cos, sin)
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError(f"mhc_amd: q and k must be [rows, heads, head_dim], got {tuple(q.shape)} and {tuple(k.shape)}")
    T, heads, hd = q.shape
    pages, page, kv, *strides = _pages(k_pages, v_pages, hd)
    if k.shape != v.shape or tuple(k.shape) != (T, kv, hd) or heads < 1:
        raise ValueError(f"mhc_amd: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} and pages "
                         f"{tuple(k_pages.shape)} do not belong together")
    if q.dtype != k_pages.dtype or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"mhc_amd: q, k, v and the pages must share a type, got {q.dtype}, {k.dtype}, {v.dtype}, "
                        f"{k_pages.dtype}")
    cu = _bounds("cu_seqlens", cu_seqlens, None, dev)
    n = cu.numel() - 1
    lens = _bounds("lengths", lengths, n, dev)
    deep = None if depths is None else _bounds("depths", depths, T, dev)
    table = _table(page_table, n, dev)
    gains, tag = (None, None), 0
    if q_gain is not None or k_gain is not None:
        gains = [None if g is None else g.contiguous() for g in (q_gain, k_gain)]
        given = [g for g in gains if g is not None]
        for g in given:
            if tuple(g.shape) != (hd,):
                raise ValueError(f"mhc_amd: a gain must be [{hd}], got {tuple(g.shape)}")
        if len({g.dtype for g in given}) > 1:
            gains = [g.float() for g in gains]
            given = gains
        tag = H.dtype_tag(given[0])
    cos, sin, stride = _tables(cos, sin, hd)
    (q, *qs), (k, *ks), (v, *vs) = _rows(q, T), _rows(k, T), _rows(v, T)
    out = torch.empty((T, heads, hd), dtype=q.dtype, device=dev)
    with _ops.launch_device(q):
        H.check(H.load().mhc_paged_append(
            q.data_ptr(), *qs, k.data_ptr(), *ks, v.data_ptr(), *vs, H.ptr(gains[0]), H.ptr(gains[1]), tag, float(eps),
            cos.data_ptr(), sin.data_ptr(), stride, cos.shape[0], H.dtype_tag(cos), cu.data_ptr(), lens.data_ptr(),
            H.ptr(deep), table.data_ptr(), out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), *strides, T, n, heads, kv, hd, 2 * cos.shape[1], table.shape[1], pages, page,
            1 if interleaved else 0, H.dtype_tag(q), H.stream(dev)), "mhc_paged_append")
    _written(k_pages, v_pages)
    return out


@functools.lru_cache(maxsize=4096)
def _workspace(*sizes) -> int:
    """Bytes, which the sizes alone decide: asked of the library once for each."""
    return max(H.load().mhc_paged_attn_workspace_bytes(*sizes), 0)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    lengths: torch.Tensor, cu_seqlens: torch.Tensor, tree: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None) -> torch.Tensor:
    """Attention of the new rows of packed sequences over their keys in pages: [rows, heads, head_dim].

    q [rows, heads, head_dim] in the pages' type, head_dim 64, 96 or 128, heads a multiple of the kv
    heads (query head h reads kv head h // (heads / kv heads)).  k_pages, v_pages, page_table,
    lengths, cu_seqlens: as in paged_append, which has stored the new rows' keys behind the first
    lengths[i].  A row sees those first keys and, of its sequence's new rows, the ones up to itself;
    with tree [rows, words] int64 instead those whose bit is set: new row j of the sequence is bit
    j % 64 of word j // 64 (a drafted token sees itself and the tokens that lead to it: DraftTree).
    scale: a positive factor of the scores (default head_dim ** -0.5).

    Rows that see no key, and rows behind the last sequence, are 0.  Keys of a page number that is
    none of the pages are not there.  The same bits on every run.  For inference.  Not-finite keys
    or values of a token may turn rows of its own sequence that do not see it into NaN, as a dense
    product under a mask does.
    """
    dev = H.require_device(q, k_pages, v_pages, tree)
    _no_graph("paged_attention", q, k_pages, v_pages)
    if q.dim() != 3:
        raise ValueError(f"mhc_amd: q must be [rows, heads, head_dim], got {tuple(q.shape)}")
    T, heads, hd = q.shape
    pages, page, kv, *strides = _pages(k_pages, v_pages, hd)
    if hd not in HEAD_DIMS:
        raise ValueError(f"mhc_amd: head_dim must be one of {HEAD_DIMS}, got {hd}")
    if kv < 1 or heads < 1 or heads % kv:
        raise ValueError(f"mhc_amd: {heads} query heads are no multiple of {kv} key heads")
    if q.dtype != k_pages.dtype:
        raise TypeError(f"mhc_amd: q and the pages must share a type, got {q.dtype} and {k_pages.dtype}")
    cu = _bounds("cu_seqlens", cu_seqlens, None, dev)
    n = cu.numel() - 1
    lens, table = _bounds("lengths", lengths, n, dev), _table(page_table, n, dev)
    words = 0
    if tree is not None:
        if tree.dtype != torch.int64 or tree.dim() != 2 or tree.shape[0] != T or tree.shape[1] < 1:
            raise ValueError(f"mhc_amd: tree must be int64 [{T}, words], got {tree.dtype} {tuple(tree.shape)}")
        tree, words = tree.contiguous(), tree.shape[1]
    scale = 1.0 / math.sqrt(hd) if scale is None else float(scale)
    if not (0.0 < scale < 3e38):
        raise ValueError(f"mhc_amd: scale must be positive, got {scale}")
    row, head, one = q.stride()
    row, head = row if T > 1 else 0, head if heads > 1 else 0
    if one != 1 or (row | head) % 8 or row >= 1 << 23 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
        row, head = heads * hd, hd
    out = torch.empty((T, heads, hd), dtype=q.dtype, device=dev)
    with _ops.launch_device(q):
        nbytes = _workspace(n, T, heads, kv, hd)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes > 0 else None
        H.check(H.load().mhc_paged_attn_fwd(
            q.data_ptr(), row, head, k_pages.data_ptr(), v_pages.data_ptr(), *strides,
            table.data_ptr(), lens.data_ptr(), cu.data_ptr(), H.ptr(tree), words, out.data_ptr(), H.ptr(ws), nbytes,
            n, T, heads, kv, hd, table.shape[1], pages, page, H.dtype_tag(q), scale, H.stream(dev)), "mhc_paged_attn_fwd")
    return out


def paged_keep(planes: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, cu_seqlens: torch.Tensor,
               kept: torch.Tensor, path: torch.Tensor) -> torch.Tensor:
    """Moves the accepted rows of each sequence's drafts together, and returns its new length: [n] int32.

    planes [planes, pages, page, kv heads, head_dim] of any type, in order, written in place: keys
    and values of every layer.  page_table, lengths, cu_seqlens: as in paged_append.  kept [n] and
    path [rows] int32, as verify_drafts gives them: key lengths[i] + path[cu_seqlens[i] + j] moves to
    lengths[i] + j for j < kept[i]; the new length is lengths[i] + kept[i].  Entries of a path below
    their own place, or that are no row of the sequence, move nothing.
    """
    dev = H.require_device(planes)
    if planes.dim() != 5 or not planes.is_contiguous():
        raise ValueError(f"mhc_amd: planes must be [planes, pages, page, kv heads, head_dim] in order, got "
                         f"{tuple(planes.shape)}")
    P, pages, page, kv, hd = planes.shape
    row = kv * hd * planes.element_size()
    if page < 16 or page & (page - 1):
        raise ValueError(f"mhc_amd: a page must have a power of two of at least 16 rows, got {page}")
    if row < 16 or row % 16 or planes.data_ptr() % 16:
        raise ValueError(f"mhc_amd: rows of {row} bytes are no multiple of 16, or not on 16 bytes")
    cu = _bounds("cu_seqlens", cu_seqlens, None, dev)
    n = cu.numel() - 1
    lens, table, kept = _bounds("lengths", lengths, n, dev), _table(page_table, n, dev), _bounds("kept", kept, n, dev)
    if path.dtype != torch.int32 or path.dim() != 1 or path.device != dev:
        raise TypeError("mhc_amd: path must be a one-dimensional int32 tensor on the pages' GPU")
    path, new = path.contiguous(), torch.empty(n, dtype=torch.int32, device=dev)
    with _ops.launch_device(planes):
        H.check(H.load().mhc_paged_keep(
            planes.data_ptr(), table.data_ptr(), lens.data_ptr(), cu.data_ptr(), kept.data_ptr(), path.data_ptr(),
            new.data_ptr(), path.numel(), n, P, pages * page * row, row, table.shape[1], pages, page, H.stream(dev)),
            "mhc_paged_keep")
    _written(planes)
    return new
