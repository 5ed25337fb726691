"""Packed sequences: several of different lengths one after another in one tensor, without
padding, as a batch of prompts, of training documents, or of next tokens over caches that
have grown to different lengths.

No reference counterpart: the reference pads (model/model_minimind.py:161-256).
"""
from __future__ import annotations

import contextlib
import functools
import math
from typing import Optional

import torch

from . import _hip as H
from . import _ops

HEAD_DIMS = _ops.ATTN_HEAD_DIMS


def _autocast() -> bool:
    return torch.is_autocast_enabled("cuda")


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
    if t.stride(2) != 1 or row % 8 or head % 8 or row >= 1 << 23 or t.data_ptr() % 16:
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


@functools.lru_cache(maxsize=4096)
def _workspace(backward: bool, *sizes) -> int:
    """Bytes, which the sizes alone decide: asked of the library once for each (1.5 us)."""
    lib = H.load()
    ask = lib.mhc_packed_attn_bwd_workspace_bytes if backward else lib.mhc_packed_attn_workspace_bytes
    return max(ask(*sizes), 0)


def _forward(q, k, v, cu_q, cu_k, used, scale, graph):
    (q, *qs), (k, *ks), (v, *vs) = _strided(q), _strided(k), _strided(v)
    Tq, heads, hd = q.shape
    Tk, kv, B = k.shape[0], k.shape[1], cu_q.numel() - 1
    dev, lib = q.device, H.load()
    out = torch.empty((Tq, heads, hd), dtype=q.dtype, device=dev)
    rest = torch.empty_like(out) if graph else None
    lse = torch.empty((heads, Tq), dtype=torch.float32, device=dev) if graph else None
    with _ops.launch_device(q):
        nbytes = _workspace(False, B, Tq, Tk, heads, kv, hd)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes > 0 else None
        H.check(lib.mhc_packed_attn_fwd(
            q.data_ptr(), *qs, k.data_ptr(), *ks, v.data_ptr(), *vs, cu_q.data_ptr(), cu_k.data_ptr(),
            H.ptr(used), out.data_ptr(), H.ptr(rest), H.ptr(lse), H.ptr(ws), nbytes, B, Tq, Tk,
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
    def backward(ctx, g):
        saved = ctx.saved_tensors  # once: checkpointing hands them out a single time
        with torch.no_grad():
            grads = _PackedAttention._backward(ctx.scale, g, *saved)
        return (*_ops.once(grads, *saved[:3], g), None, None, None, None)

    @staticmethod
    def _backward(scale, g, q, k, v, cu_q, cu_k, used, out, rest, lse):
        (q, *qs), (k, *ks), (v, *vs) = _strided(q), _strided(k), _strided(v)
        g = g.to(out.dtype).contiguous()
        if g.data_ptr() % 16:  # a caller's view; the kernels load 16 bytes
            g = g.clone()
        Tq, heads, hd = q.shape
        Tk, kv = k.shape[:2]
        dev, new = q.device, torch.empty
        g_q = new((Tq, heads, hd), dtype=q.dtype, device=dev)
        g_k, g_v = (new((Tk, kv, hd), dtype=q.dtype, device=dev) for _ in range(2))
        B, lib = cu_q.numel() - 1, H.load()
        with _ops.launch_device(q):
            nbytes = _workspace(True, B, Tq, Tk, heads, kv, hd)
            ws = new(nbytes, dtype=torch.uint8, device=dev)
            H.check(lib.mhc_packed_attn_bwd(
                q.data_ptr(), *qs, k.data_ptr(), *ks, v.data_ptr(), *vs, cu_q.data_ptr(),
                cu_k.data_ptr(), H.ptr(used), out.data_ptr(), rest.data_ptr(), lse.data_ptr(), g.data_ptr(),
                g_q.data_ptr(), g_k.data_ptr(), g_v.data_ptr(), ws.data_ptr(), nbytes, B, Tq, Tk,
                heads, kv, hd, H.dtype_tag(q), scale, H.stream(dev)), "mhc_packed_attn_bwd")
        return g_q, g_k, g_v


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
    the same bits on every run.  Not-finite keys or values of a token may turn earlier rows of
    its own sequence into NaN, as a dense product under a mask does.
    """
    if _autocast():
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


class PackedBatch:
    """The sequences of one packed call: their bounds, and each row's place in its own.

    cu_seqlens [n + 1] int32: sequence i has the rows cu_seqlens[i] to cu_seqlens[i + 1] of
    `rows`, beginning with row 0; rows behind the last belong to none (their outputs mean
    nothing).  Everything stays on cu_seqlens' device, without a synchronisation; rows' places
    are formed here, so other bounds need another batch (in a captured graph: formed inside it)."""

    def __init__(self, cu_seqlens: torch.Tensor, rows: int):
        cu = _bounds("cu_seqlens", cu_seqlens, None, cu_seqlens.device)
        self.rows = int(rows)
        self.lengths: Optional[list] = None  # of the sequences, where the host knows
        self.longest: Optional[int] = None
        with torch.inference_mode(False):  # ordinary tensors: a batch outlives the mode it is made in
            # from row 0, within the rows, not decreasing: no place formed of them lies outside a tensor
            r = torch.arange(self.rows, dtype=torch.int32, device=cu.device)
            self.cu_seqlens = torch.cat([r.new_zeros(1), cu[1:].clamp(0, self.rows)]).cummax(0).values
            self.sequence = torch.searchsorted(self.cu_seqlens[1:], r, right=True)  # n behind the last
            self.positions = (r - self.cu_seqlens[self.sequence]).long()

    @classmethod
    def from_lengths(cls, lengths, rows: Optional[int] = None, device="cuda") -> "PackedBatch":
        """Of these lengths; rows: their sum, or more."""
        lengths, ends = [int(n) for n in lengths], [0]
        for n in lengths:
            if n < 0:
                raise ValueError(f"mhc_amd: a sequence of {n} tokens")
            ends.append(ends[-1] + n)
        rows = ends[-1] if rows is None else rows
        if rows < ends[-1]:
            raise ValueError(f"mhc_amd: {ends[-1]} tokens do not fit {rows} rows")
        b = cls(torch.tensor(ends, dtype=torch.int32, device=device), rows)
        b.lengths, b.longest = lengths, max(lengths, default=0)
        return b

    def __len__(self) -> int:
        return self.cu_seqlens.numel() - 1

    def next_labels(self, labels: torch.Tensor, ignore_index: int = -100) -> torch.Tensor:
        """labels [1, rows] moved up by one row within each sequence: what each row is to
        predict, ignore_index in a sequence's last row and behind the last."""
        if tuple(labels.shape) != (1, self.rows):
            raise ValueError(f"mhc_amd: labels {tuple(labels.shape)} are not [1, {self.rows}]")
        n = len(self)
        after = torch.cat([self.sequence[1:], self.sequence.new_full((1,), n)]) if self.rows else self.sequence
        moved = torch.cat([labels[:, 1:], labels[:, :1]], 1)
        return moved.masked_fill((after != self.sequence) | (self.sequence == n), ignore_index)

    def sums(self, t: torch.Tensor) -> torch.Tensor:
        """The sum of t [rows] over each sequence, [n], in 64 bits and in the same order on every
        run.  Each by itself: differences of one running sum would carry a value that is not
        finite into every later sequence."""
        return torch.segment_reduce(t.double(), "sum", offsets=self.cu_seqlens.long(), initial=0.0, unsafe=True)


class PackedCache:
    """Keys and values of n sequences that grow in place, each in a slot of `capacity` rows
    with a length of its own: pass it as past_key_values with a PackedBatch of n sequences.

    A call appends its sequences' tokens and moves `lengths` on (on the device, so a captured
    decode step can be replayed).  Tokens that a slot has no room for are not stored, and
    their sequence's outputs mean nothing from then on; a batch made from_lengths is refused
    before that, as far as the host has seen the slots fill up.  Rows of no sequence change
    nothing.  `lengths` may be set from outside, to free a slot or roll it back.  dtype may differ from the model's: 16-bit slots are read by the kernels, under any
    autocast."""

    def __init__(self, config, sequences: int, capacity: int, dtype=torch.bfloat16, device="cuda"):
        if sequences < 1 or capacity < 1:
            raise ValueError(f"mhc_amd: a cache of {sequences} slots of {capacity} rows")
        shape = (sequences * capacity + 1, config.num_key_value_heads, config.head_dim)  # the last: what is dropped
        with torch.inference_mode(False):  # ordinary tensors: a cache outlives the mode it is made in
            self.layers = [tuple(torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
                           for _ in range(config.num_hidden_layers)]
            self.slots = torch.arange(sequences + 1, dtype=torch.int32, device=device) * capacity
            self.lengths = torch.zeros(sequences, dtype=torch.int32, device=device)
        self.sequences, self.capacity = sequences, capacity
        self._count()

    def clear(self) -> None:
        """Empties every slot."""
        self.lengths.zero_()
        self._count()

    def _count(self, seen: Optional[list] = None) -> None:
        """The slots' lengths as far as the host has seen them, of the tensor as it stands now."""
        self._seen, self._of = seen or [0] * self.sequences, self.lengths._version

    def seen(self) -> list:
        if self._of != self.lengths._version:  # set from outside since
            self._count()
        return self._seen


class PackedCall:
    """One model call on a PackedBatch: positions, and with a cache where rows go.

    A batch whose lengths the host knows is refused where its longest sequence would not fit
    behind the longest slot; with `slots` (as the model calls it) only where a sequence would not
    fit its own."""

    def __init__(self, batch: PackedBatch, cache: Optional[PackedCache] = None, slots: bool = False):
        self.batch, self.cache = batch, cache
        self.positions, self.lengths, self.rows = batch.positions, None, None
        # positions that the host knows the sequences reach, and a bound on those they may reach
        self.reach, self.most = batch.longest or 0, batch.rows if batch.longest is None else batch.longest
        if cache is None:
            return
        n, cap = cache.sequences, cache.capacity
        if len(batch) != n:
            raise ValueError(f"mhc_amd: a batch of {len(batch)} sequences on a cache of {n}")
        if batch.lengths is not None:
            seen = cache.seen()
            have, more = max(seen), batch.longest
            if slots and have + more > cap:
                have, more = max(zip(seen, batch.lengths), key=sum)
            if have + more > cap:
                raise ValueError(f"mhc_amd: {have} + {more} tokens may not fit slots of {cap} rows")
            self.reach = max((a + b for a, b in zip(seen, batch.lengths) if b), default=0)
        self.most = cap
        seq = batch.sequence.clamp_max(n - 1)
        self.positions = cache.lengths[seq] + batch.positions
        room = (batch.sequence < n) & (self.positions < cap)
        self.rows = torch.where(room, seq * cap + self.positions, n * cap)
        self.lengths = (cache.lengths + batch.cu_seqlens.diff()).clamp_max_(cap)

    def done(self) -> None:
        """The call has stored its tokens: the lengths move on (those that the host keeps too, unless
        the call was only captured)."""
        if self.cache is None:
            return
        seen = self.cache.seen()
        self.cache.lengths.copy_(self.lengths)
        if self.batch.lengths is not None and not (
                self.lengths.is_cuda and torch.cuda.is_current_stream_capturing()):
            seen = [a + b for a, b in zip(seen, self.batch.lengths)]
        self.cache._count(seen)

    def attention(self, q, k, v, layer: int, dropout: float = 0.0) -> torch.Tensor:
        """q [1, rows, heads, head_dim], k, v [1, rows, kv heads, head_dim] of the new tokens:
        [1, rows, heads * head_dim], over their sequences' keys so far."""
        q, k, v, cu = q[0], k[0], v[0], self.batch.cu_seqlens
        cu_k, used, dtype = cu, None, q.dtype
        if self.cache is not None:
            if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad):
                raise RuntimeError("mhc_amd: a cache is for inference; call under torch.no_grad()")
            ck, cv = self.cache.layers[layer]
            ck.index_copy_(0, self.rows, k.to(ck.dtype))
            cv.index_copy_(0, self.rows, v.to(cv.dtype))
            q, k, v, cu_k, used = q.to(ck.dtype), ck, cv, self.cache.slots, self.lengths
        half = q.dtype in _ops.HALF or _autocast()
        if q.is_cuda and half and q.shape[2] in HEAD_DIMS and dropout == 0.0 and _ops.eager_call():
            # the cache's 16-bit type goes before an autocast's, which would copy every slot
            slots = self.cache is not None and k.dtype in _ops.HALF
            with torch.autocast("cuda", enabled=False) if slots and _autocast() else contextlib.nullcontext():
                out = packed_attention(q, k, v, cu, cu_seqlens_k=cu_k, key_lengths=used)
        else:
            out = _plain_attention(q, k, v, cu, cu_k, used, dropout)
        if self.cache is not None and not torch.is_autocast_enabled(q.device.type):
            out = out.to(dtype)  # the layer's, whatever the cache keeps; under autocast any type will do
        return out.reshape(1, out.shape[0], -1)


def _plain_attention(q, k, v, cu_q, cu_k, used, dropout):
    """packed_attention on torch ops, for what the kernels do not take (fp32, the CPU, other
    head_dims, dropout): one attention under a mask over all rows."""
    def places(cu, rows):
        r = torch.arange(rows, dtype=torch.int32, device=q.device)
        seq = torch.searchsorted(cu[1:], r, right=True)
        return seq, r - cu[seq]
    (qs, qp), (ks, kp) = places(cu_q, q.shape[0]), places(cu_k, k.shape[0])
    n = cu_q.numel() - 1
    new, have = cu_q.diff(), cu_k.diff() if used is None else used
    shift = torch.cat([have - new, new.new_zeros(1)])  # the last query sits at the last key
    inside = kp < torch.cat([have, new.new_zeros(1)])[ks]
    seen = (qs[:, None] == ks) & inside & (kp <= (qp + shift[qs])[:, None]) & (qs < n)[:, None]
    rep = q.shape[1] // k.shape[1]
    # keys in use that are no numbers: a probability of 0 would not keep them from other rows
    bad = ~(torch.isfinite(k).all(2) & torch.isfinite(v).all(2))
    k, v = (torch.where((inside & (ks < n))[:, None, None] & ~bad[:, :, None], t, 0)
            .repeat_interleave(rep, 1).transpose(0, 1) for t in (k, v))
    some = seen.any(1)
    out = torch.nn.functional.scaled_dot_product_attention(
        q.transpose(0, 1)[None], k[None], v[None], attn_mask=seen | ~some[:, None], dropout_p=dropout)
    out = torch.where(some[:, None, None], out[0].transpose(0, 1), 0)
    # [rows, kv heads]: whether one is among the keys a row sees, from its sequence's first to its own
    upto = torch.cat([bad.new_zeros(1, bad.shape[1], dtype=torch.int32), bad.cumsum(0, dtype=torch.int32)])
    first = cu_k.clamp(0, k.shape[1])[qs]
    count = torch.minimum(qp + shift[qs] + 1, torch.cat([have, new.new_zeros(1)])[qs]).clamp_min(0)
    hit = upto[(first + count).clamp_max(k.shape[1])] > upto[first]
    return out.masked_fill(hit.repeat_interleave(rep, 1)[:, :, None], math.nan)
