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
def _workspace(device: int, *sizes) -> int:
    """Bytes, which the sizes and the current device's compute units decide: asked of the library once for each."""
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
        nbytes = _workspace(dev.index, n, T, heads, kv, hd)
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


def _capturing(t: torch.Tensor) -> bool:
    return t.is_cuda and torch.cuda.is_current_stream_capturing()


class DraftTree:
    """Drafted tokens of a PackedBatch: each sequence's first row is its last token, the others a tree
    behind it, parents before children.  A model call with drafts=DraftTree(...) over a PagedCache
    stores them without moving the sequences on; PagedCache.keep then keeps a branch.

    parents [rows] int32: the place in its sequence of the row that a row follows (the first row's
    does not count; a row without a parent before it sees only itself and the past).  None: chains,
    each row following the one before it.
    mask [rows, words] int64 (None for chains): the rows that each row sees, as paged_attention takes
    them; depths [rows] int32: their distance from the first row.  Both are formed here, on the
    device, so other trees need another DraftTree (in a captured graph: formed inside it)."""

    def __init__(self, batch: PackedBatch, parents: Optional[torch.Tensor] = None):
        self.batch, self.parents, self.mask, self.depths = batch, parents, None, None
        if parents is None:
            return
        rows, dev = batch.rows, batch.cu_seqlens.device
        if parents.dtype != torch.int32 or tuple(parents.shape) != (rows,) or parents.device != dev:
            raise ValueError(f"mhc_amd: parents must be int32 [{rows}] on {dev}, got {parents.dtype} "
                             f"{tuple(parents.shape)} on {parents.device}")
        most = rows if batch.longest is None else batch.longest
        with torch.inference_mode(False):  # ordinary tensors, as the batch's
            r, place = torch.arange(rows, device=dev), batch.positions
            first = r - place
            up = parents.long()
            good = (up >= 0) & (up < place) & (batch.sequence < len(batch))
            jump = torch.cat([torch.where(good, first + up, rows), r.new_full((1,), rows)])  # the last: none
            mask = torch.zeros(rows + 1, max((most + 63) // 64, 1), dtype=torch.int64, device=dev)
            inside = place < 64 * mask.shape[1]
            word = torch.where(inside, place // 64, 0)
            mask[r, word] = torch.where(inside, torch.ones_like(r) << (place % 64), 0)
            depth = torch.cat([good.int(), r.new_zeros(1, dtype=torch.int32)])
            step = 1
            while step < most:  # each round doubles the ancestors that a row has joined with
                mask |= mask[jump]
                depth += depth[jump]
                jump = jump[jump]
                step *= 2
            self.mask, self.depths = mask[:rows].contiguous(), depth[:rows].contiguous()


class PagedCache:
    """Keys and values of n sequences in pages that are handed out as the sequences grow: pass it as
    past_key_values with a PackedBatch of n sequences.

    capacity: the most keys a sequence may have; page: rows of a page, a power of two of at least
    16; pages: how many there are for all sequences together (default: enough for every one to reach
    its capacity).  The kernels read and write the pages in place; a sequence's pages stand in
    page_table [n, width] (int32, -1: none), its keys in lengths [n] (int32), both on the device.

    A call's new rows need pages before it: a call with a batch made from_lengths hands them out by
    itself, as does reserve(), and raises where none are left.  The host counts what the sequences may
    have at most; after keep(), which only the device knows the result of, it counts all of a tree's
    rows, until it looks at the lengths: where its count leaves no room, or in settle(), which takes back
    the pages that are not needed.  A call that is captured into a graph hands out none: reserve() what its
    replays will need before.  Replays move the lengths on where the host does not see it: from a cache's
    first captured call on, reserve() and calls that hand out pages look at the lengths first (a
    synchronisation).  Rows that have no page are dropped, and their sequence's outputs mean nothing from
    then on: wherever the host looks, a length behind the sequence's pages raises (free() it, or set its
    length back)."""

    def __init__(self, config, sequences: int, capacity: int, page: int = 64, pages: Optional[int] = None,
                 dtype=torch.bfloat16, device="cuda"):
        if sequences < 1 or capacity < 1:
            raise ValueError(f"mhc_amd: a cache of {sequences} sequences of {capacity} keys")
        if page < 16 or page & (page - 1):
            raise ValueError(f"mhc_amd: a page must have a power of two of at least 16 rows, got {page}")
        width = (capacity + page - 1) // page
        pages = sequences * width if pages is None else pages
        if pages < 1:
            raise ValueError(f"mhc_amd: a cache of {pages} pages")
        with torch.inference_mode(False):  # ordinary tensors: a cache outlives the mode it is made in
            self.planes = torch.zeros(2 * config.num_hidden_layers, pages, page, config.num_key_value_heads,
                                      config.head_dim, dtype=dtype, device=device)
            self.page_table = torch.full((sequences, width), -1, dtype=torch.int32, device=device)
            self.lengths = torch.zeros(sequences, dtype=torch.int32, device=device)
        self.layers = [(self.planes[2 * i], self.planes[2 * i + 1]) for i in range(config.num_hidden_layers)]
        self.sequences, self.capacity, self.page = sequences, capacity, page
        self.replays = False  # whether a call was captured, whose replays the host does not count
        self._empty()

    def clear(self) -> None:
        """Empties every sequence and takes all pages back."""
        self._outside_a_capture()
        self._empty()
        self.lengths.zero_()
        self.page_table.fill_(-1)

    def _empty(self) -> None:
        self.most = [0] * self.sequences  # keys that each sequence has at most
        self.held = [0] * self.sequences  # keys that reserve() was asked for pages for
        self.drafted = [0] * self.sequences  # rows behind those that keep() may still move
        self.owned = [[] for _ in range(self.sequences)]
        self.free_pages = list(range(self.planes.shape[1]))[::-1]

    def free(self, sequence: int) -> None:
        """Empties a sequence and takes its pages back."""
        self._outside_a_capture()
        self.free_pages += self.owned[sequence][::-1]
        self.owned[sequence], self.most[sequence] = [], 0
        self.held[sequence] = self.drafted[sequence] = 0
        self.lengths[sequence] = 0
        self.page_table[sequence] = -1

    def _outside_a_capture(self) -> None:
        if _capturing(self.lengths):
            raise RuntimeError("mhc_amd: pages are handed out and taken back outside of a captured call")

    def _rows(self, rows) -> list:
        rows = [int(rows)] * self.sequences if not hasattr(rows, "__len__") else [int(n) for n in rows]
        if len(rows) != self.sequences:
            raise ValueError(f"mhc_amd: rows of {len(rows)} sequences for a cache of {self.sequences}")
        return rows

    def reserve(self, rows) -> None:
        """Pages for so many more rows of each sequence (a number, or one for each): all of them or, with
        an error, none.  Where the host's count leaves no room for them it looks at the lengths (a
        synchronisation) and takes back pages behind them, but none that were reserved."""
        self._outside_a_capture()
        rows = self._rows(rows)
        self._provide(rows)
        self.held = [max(h, m + n) if n else h for h, m, n in zip(self.held, self.most, rows)]

    def _need(self, rows):
        """Pages that so many more rows of each sequence take, or the error where there is no room."""
        need = []
        for i, n in enumerate(rows):
            if n and self.most[i] + n > self.capacity:
                return ValueError(f"mhc_amd: {self.most[i]} + {n} keys may not fit a sequence's {self.capacity}")
            need.append(max(0, -(-(self.most[i] + n) // self.page) - len(self.owned[i])) if n else 0)
        if sum(need) > len(self.free_pages):
            return RuntimeError(f"mhc_amd: {sum(need)} pages needed, {len(self.free_pages)} left")
        return need

    def _provide(self, rows: list) -> None:
        asked = [i for i, n in enumerate(rows) if n]
        if self.replays:
            self._look(asked)
        need = self._need(rows)
        if isinstance(need, Exception):
            if not self.replays:
                self._look(asked)
            self._take_back()
            need = self._need(rows)
        if isinstance(need, Exception):
            raise need
        if not any(need):
            return
        seqs, slots, numbers = [], [], []
        for i, n in enumerate(need):
            for _ in range(n):
                seqs.append(i)
                slots.append(len(self.owned[i]))
                numbers.append(self.free_pages.pop())
                self.owned[i].append(numbers[-1])
        at = torch.tensor([seqs, slots], device=self.page_table.device)
        self.page_table[at[0], at[1]] = torch.tensor(numbers, dtype=torch.int32, device=self.page_table.device)

    def _look(self, sequences) -> None:
        """The host's count from the lengths themselves (a synchronisation); raises where one of these
        sequences has lost rows."""
        have = self.lengths.tolist()
        self.most = [min(max(n, 0), self.capacity) for n in have]
        for i in sequences:
            if have[i] > len(self.owned[i]) * self.page:
                raise RuntimeError(f"mhc_amd: sequence {i} has {have[i]} keys and pages for {len(self.owned[i]) * self.page}: "
                                   "rows were dropped (free() it, or set its length back)")

    def settle(self, spare=None) -> None:
        """Looks at the lengths (a synchronisation) and takes back the pages behind them, but for those of so
        many spare rows of each sequence (a number, or one for each).  None: what is reserved stays in a cache
        with captured calls, whose replays count on it, and goes in any other.  Pages of drafts that keep()
        may still move stay.  Raises where a sequence's length is behind its pages (one without any page is
        not in use)."""
        self._outside_a_capture()
        spare = None if spare is None else self._rows(spare)
        self._look([i for i, pages in enumerate(self.owned) if pages])
        if spare is not None:
            self.held = [m + n for m, n in zip(self.most, spare)]
        elif not self.replays:
            self.held = [0] * self.sequences
        self._take_back()

    def _take_back(self) -> None:
        """Takes back the pages that nobody counts on."""
        seqs, slots = [], []
        for i, n in enumerate(self.most):
            keep = -(-max(n + self.drafted[i], self.held[i]) // self.page)
            slots += range(keep, len(self.owned[i]))
            seqs += [i] * (len(self.owned[i]) - keep)
            self.free_pages += self.owned[i][keep:][::-1]
            del self.owned[i][keep:]
        if seqs:
            self.page_table[seqs, slots] = -1

    def grown(self, batch: PackedBatch) -> torch.Tensor:
        """The lengths with the batch's rows, as far as there is room."""
        return (self.lengths + batch.cu_seqlens.diff()).clamp_max_(self.page_table.shape[1] * self.page)

    def keep(self, batch: PackedBatch, kept: torch.Tensor, path: torch.Tensor) -> None:
        """Keeps the accepted rows of a call with drafts (verify_drafts' kept and path): moves their keys
        and values together in every layer, and the lengths on."""
        if len(batch) != self.sequences:
            raise ValueError(f"mhc_amd: a batch of {len(batch)} sequences on a cache of {self.sequences}")
        if self.planes.is_cuda:
            new = paged_keep(self.planes, self.page_table, self.lengths, batch.cu_seqlens, kept, path)
        else:
            new = self._plain_keep(batch, kept, path)
        self.lengths.copy_(new)
        self._count(batch)

    def _count(self, batch: PackedBatch) -> None:
        """The rows of a call, as far as the host knows them (a captured call has stored none yet, and
        any number once it is replayed)."""
        if _capturing(self.lengths):
            self.replays = True
            return
        new = [batch.rows] * self.sequences if batch.lengths is None else batch.lengths
        self.drafted = [0 if n else d for n, d in zip(new, self.drafted)]
        self.most = [min(a + b, self.capacity) for a, b in zip(self.most, new)]

    def rows_of(self, sequence: torch.Tensor, key: torch.Tensor) -> torch.Tensor:
        """Rows of a plane, its pages one after another, of keys of sequences; -1 where there is none."""
        width, pages = self.page_table.shape[1], self.planes.shape[1]
        inside = (sequence < self.sequences) & (key >= 0) & (key < width * self.page)
        number = self.page_table[sequence.clamp_max(self.sequences - 1), (key // self.page).clamp(0, width - 1)]
        inside &= (number >= 0) & (number < pages)
        return torch.where(inside, number.long() * self.page + key % self.page, -1)

    def _plain_keep(self, batch, kept, path):
        seq, place = batch.sequence, batch.positions
        count = batch.cu_seqlens.diff()
        kept = torch.minimum(kept, count).clamp_min(0)
        at = seq.clamp_max(self.sequences - 1)
        go = (seq < self.sequences) & (place < kept[at]) & (path > place) & (path < count[at])
        src = self.rows_of(at, (self.lengths[at] + path).long())
        dst = self.rows_of(at, (self.lengths[at] + place).long())
        go &= (src >= 0) & (dst >= 0)
        flat = self.planes.flatten(1, 2)
        flat[:, dst[go]] = flat[:, src[go]]
        return (self.lengths + kept).clamp_max(self.page_table.shape[1] * self.page)


class PagedCall:
    """One model call on a PackedBatch over a PagedCache: where its rows stand.  A call that is refused
    has handed out no pages; table: the positions that the model has, if it is to be refused for those."""

    def __init__(self, batch: PackedBatch, cache: PagedCache, drafts: Optional[DraftTree] = None,
                 table: Optional[int] = None):
        if len(batch) != cache.sequences:
            raise ValueError(f"mhc_amd: a batch of {len(batch)} sequences on a cache of {cache.sequences}")
        if drafts is not None and drafts.batch is not batch:
            raise ValueError("mhc_amd: drafts of another batch")
        self.batch, self.cache, self.drafts = batch, cache, drafts
        # positions that the host knows the sequences reach, and a bound on those they may reach
        self.reach, self.most = max(batch.lengths or [0]), cache.capacity
        if table is not None and self.reach > table:
            raise ValueError(f"a packed sequence reaches {self.reach} positions, max_position_embeddings is {table}")
        if batch.lengths is not None and not _capturing(cache.lengths):
            cache._provide(batch.lengths)
        self.depths = None if drafts is None else drafts.depths
        deep = batch.positions if self.depths is None else self.depths.long()
        self.past = cache.lengths[batch.sequence.clamp_max(cache.sequences - 1)]
        self.positions = self.past + deep

    def within(self, table: int) -> None:
        """Rows past a table of so many positions take its last one (their outputs mean nothing; as NaN
        they would reach the other rows of their sequences)."""
        self.depths = (self.positions.clamp(0, table - 1) - self.past).int()

    def done(self) -> None:
        """The call has stored its rows: without drafts they stay."""
        if self.drafts is None:
            self.cache.lengths.copy_(self.cache.grown(self.batch))
            self.cache._count(self.batch)
        elif _capturing(self.cache.lengths):
            self.cache.replays = True
        elif self.batch.lengths is not None:
            self.cache.drafted = [n or d for n, d in zip(self.batch.lengths, self.cache.drafted)]

    def attention(self, m, q, k, v, tables, layer: int) -> torch.Tensor:
        """q [1, rows, heads, head_dim], k, v [1, rows, kv heads, head_dim], the projections of the
        attention layer m: [1, rows, heads * head_dim]; tables: cos and sin, [positions, rotary_dim / 2]."""
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
            raise RuntimeError("mhc_amd: a cache is for inference; call under torch.no_grad()")
        q, k, v, dtype = q[0], k[0], v[0], q.dtype
        cache, cu, tree = self.cache, self.batch.cu_seqlens, self.drafts
        kp, vp = cache.layers[layer]
        if self._fused(m, q, kp):
            q, k, v = (t if t.dtype == kp.dtype else t.to(kp.dtype) for t in (q, k, v))
            q = paged_append(q, k, v, kp, vp, cache.page_table, cache.lengths, cu, *tables,
                             depths=self.depths, q_gain=m.q_norm.weight,
                             k_gain=m.k_norm.weight, eps=m.q_norm.eps, interleaved=m.rope_interleaved)
            out = paged_attention(q, kp, vp, cache.page_table, cache.lengths, cu, tree=None if tree is None else tree.mask)
        else:
            at = self.positions if self.depths is None else self.past + self.depths
            q, k = plain_rotary(m.q_norm(q), m.k_norm(k), *tables, at, m.rope_interleaved)
            out = self._plain(q.to(kp.dtype), k.to(kp.dtype), v.to(kp.dtype), kp, vp, m.dropout if m.training else 0.0)
        if out.dtype != dtype and not torch.is_autocast_enabled(out.device.type):
            out = out.to(dtype)
        return out.reshape(1, out.shape[0], -1)

    @staticmethod
    def _fused(m, q, pages) -> bool:
        """Whether the kernels take this layer's norms and types, in a call that nothing traces."""
        norms = (m.q_norm, m.k_norm)
        return (q.is_cuda and pages.dtype in _ops.HALF and q.shape[2] in HEAD_DIMS and _ops.eager_call()
                and not (m.training and m.dropout > 0)
                and all(_ops.plain_module(n, torch.nn.RMSNorm) and n.weight is not None and n.eps is not None
                        and n.weight.dtype in (torch.float32, *_ops.HALF) for n in norms)
                and m.q_norm.eps == m.k_norm.eps)

    def _plain(self, q, k, v, kp, vp, dropout):
        """Storing and attention on torch ops, for what the kernels do not take: one attention under a
        mask over all sequences' keys."""
        cache, batch, tree = self.cache, self.batch, self.drafts
        n, room = cache.sequences, cache.page_table.shape[1] * cache.page
        seq, dev = batch.sequence, q.device
        mine = seq.clamp_max(n - 1)
        past = cache.lengths.clamp(0, room).long()
        rows = cache.rows_of(seq, past[mine] + batch.positions)
        there = rows >= 0
        kf, vf = kp.flatten(0, 1), vp.flatten(0, 1)
        kf[rows[there]], vf[rows[there]] = k[there], v[there]
        have = torch.minimum(past + batch.cu_seqlens.diff(), past.new_full((), room))
        owner = torch.arange(n, device=dev).repeat_interleave(room)
        key = torch.arange(room, device=dev).repeat(n)
        at = cache.rows_of(owner, key)
        real = (at >= 0) & (key < have[owner])
        fresh = key - past[owner]  # place among the new rows
        seen = (seq[:, None] == owner) & real
        if tree is None or tree.mask is None:
            seen &= fresh <= batch.positions[:, None]
        else:
            bit = fresh.clamp(0, 64 * tree.mask.shape[1] - 1)
            own = (tree.mask[:, bit // 64] >> (bit % 64)) & 1 == 1
            seen &= (fresh < 0) | own & (fresh < 64 * tree.mask.shape[1])
        rep = q.shape[1] // kp.shape[2]
        kk, vv = (t[at.clamp_min(0)] for t in (kf, vf))
        # keys that are no numbers: a probability of 0 would not keep them from other rows
        bad = real[:, None] & ~(torch.isfinite(kk).all(2) & torch.isfinite(vv).all(2))
        kk, vv = (torch.where((real[:, None] & ~bad)[:, :, None], t, 0).repeat_interleave(rep, 1).transpose(0, 1) for t in (kk, vv))
        some = seen.any(1)
        out = torch.nn.functional.scaled_dot_product_attention(
            q.transpose(0, 1)[None], kk[None], vv[None], attn_mask=seen | ~some[:, None], dropout_p=dropout)
        out = torch.where(some[:, None, None], out[0].transpose(0, 1), 0)
        hit = torch.stack([(seen & b).any(1) for b in bad.unbind(1)], 1)
        return out.masked_fill(hit.repeat_interleave(rep, 1)[:, :, None], math.nan)
