"""Operators on a paged K/V cache, on torch tensors: drafted tokens verified
over the cache in one pass, and the cache cut to a budget.

  tree_attention   drafted tokens (a tree, one bit mask a token) attend the
                   cache and one another; one token a sequence is the
                   ordinary decode step
  append           accepted drafts (or a prompt) written behind the cache
  rotate           queries and keys of new tokens, normed and rotated by positions
                   of one or several axes
  read             positions of a packed cache as numbers again
  attention_mass   the attention weight that cached positions received,
                   added to a running sum
  evict            keeps the first, the last and the most attended positions
                   (select, then compact)

A cache holds f32, f16 or bf16 (:class:`PagedCache`), or 4 bits (:class:`PackedCache`, for
tree_attention, append and read).

All run on the tensors' device and torch's current stream, read lengths on the
device and wait for nothing, so they can be captured in a CUDA graph.  They call
the C ABI of include/ocrvl_cuda.h (ocrvl_op_tree_attn and following), whose
comments say what each computes; a wrong argument raises OcrvlError or
ValueError before anything runs.  There is no backward pass: a tensor that
requires a gradient is refused unless gradients are off.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from . import build as _build

_lib.load()
_build.build_torch()
from . import _kvops  # noqa: E402

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}


class PagedCache:
    """A paged cache: ``k`` and ``v`` are [pages, layers, kv heads, page_size,
    head_dim] tensors of the same type and strides (views of one pool, for
    instance) and ``table`` [batch, max_pages] int32 names the pages of each
    sequence in order, an entry outside 0..pages-1 none; its rows may lie apart, but not
    share memory.  Page sizes are powers of two from 16 on, head_dim is 64 or 128."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor):
        if k.dim() != 5 or k.shape != v.shape or k.stride() != v.stride() or k.dtype is not v.dtype:
            raise ValueError("k and v must be [pages, layers, kv heads, page_size, head_dim] of one type and one set of strides")
        if k.dtype not in _TYPES or not k.is_cuda or v.device != k.device:
            raise ValueError("k and v must be float32, float16 or bfloat16 CUDA tensors")
        if k.stride(4) != 1:
            raise ValueError("head_dim must be contiguous")
        if table.dim() != 2 or table.dtype is not torch.int32 or table.device != k.device or table.stride(1) != 1:
            raise ValueError(f"table must be a [batch, max_pages] int32 tensor on {k.device}")
        if table.shape[0] > 1 and table.stride(0) < table.shape[1]:
            raise ValueError("the table's rows must not overlap (an expanded row needs a copy: .contiguous())")
        self.k, self.v, self.table = k, v, table
        self.dtype, self.device = k.dtype, k.device
        pages, layers, heads, page, dim = k.shape
        d = _lib.KVCache(_TYPES[k.dtype], dim, heads, layers, page, pages, table.shape[0], table.shape[1], k.stride(0),
                         k.stride(1), k.stride(2), k.stride(3), table.stride(0) if table.shape[0] > 1 else table.shape[1], k.data_ptr(),
                         v.data_ptr(), table.data_ptr())
        self._set(d)

    def _set(self, d) -> None:
        self.desc = d
        self._ref = (C.addressof(d), self.device.index, self.k, self.v)  # for the native side
        self.head_dim, self.kv_heads, self.layers, self.batch = d.head_dim, d.num_kv_heads, d.num_layers, d.batch
        self.capacity = d.max_pages * d.page_size

    @classmethod
    def of_sequence(cls, seq) -> "PagedCache":
        """The cache of an engine sequence (``Runtime.new_sequence``): f32,
        every layer, one table row.  It stays valid while the sequence lives, its
        table follows the sequence, and positions past it are unmapped (``append`` is for
        caches of the caller's own); order work on it against ``Runtime.stream_handle`` (the engine's calls
        wait for their own work before they return)."""
        self = cls.__new__(cls)
        d = _lib.KVCache()
        _lib.check(seq.rt._L.ocrvl_seq_kv_view(seq._h, C.byref(d)))
        self.k = self.v = self.table = None
        self._seq = seq  # holds the memory
        self.dtype, self.device = torch.float32, torch.device("cuda", seq.rt.device)
        self._set(d)
        return self

    def work_bytes(self, heads: int, max_draft: int = 64) -> int:
        """Bytes of workspace a ``tree_attention`` call with that many query heads takes."""
        n = C.c_int64()
        _lib.check(_lib.load().ocrvl_op_tree_attn_workspace(C.byref(self.desc), heads, max_draft, C.byref(n)))
        return n.value


class PackedCache:
    """A paged cache in 4 bits: ``k`` and ``v`` are [pages, layers, kv heads, page_size, head_dim / 2] uint8 tensors,
    ``k_scale`` and ``v_scale`` [pages, layers, kv heads, page_size, head_dim / 32] bfloat16 ones (each pair of the same
    strides, the last two dimensions contiguous), ``table`` as in :class:`PagedCache`.  32 dims of a position share a
    scale s and are whole numbers of -7 .. 7 times s: see ``ocrvl_packed_cache`` in the header.  ``append`` quantises into
    it, ``tree_attention`` attends it, ``read`` gives it back; :meth:`empty` makes one."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, table: torch.Tensor):
        for name, x, y, dtype in (("k and v", k, v, torch.uint8), ("k_scale and v_scale", k_scale, v_scale, torch.bfloat16)):
            if x.dim() != 5 or x.shape != y.shape or x.stride() != y.stride() or x.dtype is not dtype or y.dtype is not dtype:
                raise ValueError(f"{name} must be five-dimensional {dtype} tensors of one shape and one set of strides")
            if not x.is_cuda or x.device != k.device or y.device != k.device:
                raise ValueError("k, v and their scales must be on one CUDA device")
            if x.stride(4) != 1 or x.stride(3) != x.shape[4]:
                raise ValueError(f"the positions of a page of {name} must be contiguous")
        pages, layers, heads, page, half = k.shape
        if half not in (32, 64) or k_scale.shape != (pages, layers, heads, page, half // 16):
            raise ValueError("k must be [pages, layers, kv heads, page_size, head_dim / 2] with head_dim 64 or 128, its scales one for 32 dims")
        if table.dim() != 2 or table.dtype is not torch.int32 or table.device != k.device or table.stride(1) != 1:
            raise ValueError(f"table must be a [batch, max_pages] int32 tensor on {k.device}")
        if table.shape[0] > 1 and table.stride(0) < table.shape[1]:
            raise ValueError("the table's rows must not overlap (an expanded row needs a copy: .contiguous())")
        self.k, self.v, self.k_scale, self.v_scale, self.table, self.device = k, v, k_scale, v_scale, table, k.device
        self.desc = _lib.PackedCache(2 * half, heads, layers, page, pages, table.shape[0], table.shape[1], 0, *k.stride()[:3],
                                     *k_scale.stride()[:3], table.stride(0) if table.shape[0] > 1 else table.shape[1],
                                     k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), table.data_ptr())
        self._ref = (C.addressof(self.desc), self.device.index, k, v, k_scale, v_scale)  # for the native side
        self.head_dim, self.kv_heads, self.layers, self.batch = 2 * half, heads, layers, table.shape[0]
        self.capacity = table.shape[1] * page

    def work_bytes(self, heads: int, max_draft: int = 64, dtype: Optional[torch.dtype] = None) -> int:
        """Bytes of workspace a ``tree_attention`` call with that many query heads (of ``dtype``, or of any type) takes."""
        if dtype is not None and dtype not in _TYPES:
            raise ValueError("dtype must be float32, float16 or bfloat16")
        n, most = C.c_int64(), 0
        for t in _TYPES.values() if dtype is None else (_TYPES[dtype],):
            _lib.check(_lib.load().ocrvl_op_packed_attn_workspace(C.byref(self.desc), t, heads, max_draft, C.byref(n)))
            most = max(most, n.value)
        return most

    @classmethod
    def empty(cls, pages: int, layers: int, kv_heads: int, head_dim: int, table: torch.Tensor, *, page_size: int = 16) -> "PackedCache":
        """A cache of ``pages`` pages on the table's device (every number in it 0)."""
        if head_dim not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        k, v = torch.full((2, pages, layers, kv_heads, page_size, head_dim // 2), 0x88, dtype=torch.uint8, device=table.device)
        ks, vs = torch.zeros(2, pages, layers, kv_heads, page_size, head_dim // 32, dtype=torch.bfloat16, device=table.device)
        return cls(k, v, ks, vs, table)


class Rotary:
    """Rotary positions: which dims of a head turn by which of a token's positions, and how fast.

    ``pairs`` (default: half of head_dim) pairs of dims turn, by ``theta ** (-p / pairs)`` radians a position or by
    ``freq`` [pairs]; the dims behind them stay.  Pair p is dims p and p + pairs, or 2 p and 2 p + 1 with ``neighbours``.
    Without more a token has one position.  ``sections`` (pairs of each axis, in order: (16, 24, 24) for time, height and width, say)
    or ``axis`` [pairs] (each pair's, in any order) give it several."""

    def __init__(self, head_dim: int, *, theta: float = 10000.0, pairs: Optional[int] = None, freq: Optional[Sequence[float]] = None,
                 sections: Optional[Sequence[int]] = None, axis: Optional[Sequence[int]] = None, neighbours: bool = False):
        pairs = head_dim // 2 if pairs is None else pairs
        if not 8 <= head_dim <= 256 or head_dim % 8:
            raise ValueError("head_dim must be a multiple of 8, at most 256")
        if not 4 <= pairs <= head_dim // 2 or pairs % 4:
            raise ValueError("pairs must be a multiple of 4, at most half of head_dim")
        if sections is not None and axis is not None:
            raise ValueError("sections or axis, not both")
        if sections is not None:
            axis = [a for a, n in enumerate(sections) for _ in range(n)]
        axis = [0] * pairs if axis is None else [int(a) for a in axis]
        axes = len(sections) if sections is not None else max(axis, default=0) + 1
        if len(axis) != pairs or not 1 <= axes <= 8 or min(axis) < 0 or (sections is not None and min(sections) < 0):
            raise ValueError(f"sections (or axis) must say which of at most 8 axes each of the {pairs} pairs has")
        if freq is None and not (theta > 0 and math.isfinite(theta)):
            raise ValueError("theta must be positive")
        freq = [float(theta) ** (-p / pairs) for p in range(pairs)] if freq is None else [float(f) for f in freq]
        if len(freq) != pairs or not all(map(math.isfinite, freq)):
            raise ValueError(f"freq must be {pairs} finite numbers")
        self.desc = _lib.Rotary(head_dim, pairs, axes, int(bool(neighbours)), (C.c_double * 128)(*freq), (C.c_uint8 * 128)(*axis))
        self.head_dim, self.pairs, self.axes = head_dim, pairs, axes
        self._ref = C.addressof(self.desc)


def rotate(q: torch.Tensor, k: Optional[torch.Tensor], pos: torch.Tensor, rotary: Rotary, *, q_weight: Optional[torch.Tensor] = None,
           k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, q_out: Optional[torch.Tensor] = None,
           k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Queries and keys of new tokens, normed and rotated in one pass.

    q [tokens, heads, head_dim], k [tokens, kv heads, head_dim] (or None), each with a stride of its own between tokens:
    views of one projection's output, say.  ``pos`` [tokens, axes] int32 ([tokens] with one axis).  With ``q_weight`` and
    ``k_weight`` [head_dim] (float32 or q's type) each head is first divided by the root of its mean square (plus
    ``eps``) and multiplied by the weights.  ``q_out`` and ``k_out`` may be q and k themselves.  Angles are worked out in
    64 bits.  Returns (q, k) turned."""
    if not isinstance(rotary, Rotary):
        raise ValueError("rotary must be a Rotary")
    return _kvops.rotate(rotary._ref, q, k, pos, q_weight, k_weight, eps, q_out, k_out)


def tree_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: Union[PagedCache, PackedCache], lens: torch.Tensor,
                   indptr: torch.Tensor, mask: torch.Tensor, *, layer: int = 0, max_draft: Optional[int] = None,
                   scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                   lse: Optional[torch.Tensor] = None, work: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of drafted tokens over a cache and over one another.

    q [tokens, heads, head_dim]; k, v [tokens, kv heads, head_dim]: the drafts'
    own keys and values, which are not in the cache yet.  ``indptr`` [batch + 1]
    int32 bounds each sequence's tokens, ``lens`` [batch] int32 are the cached
    lengths.  ``mask`` [tokens] int64: bit j lets the token attend its
    sequence's token j, its own included only if set (-1: all).  ``max_draft``
    bounds the tokens of a sequence (64 at most; the default is the call's tokens, up to
    64; more are not computed and their outputs not written): name the smallest that
    holds, kernels are chosen by it.  ``work``: a uint8 tensor
    of ``cache.work_bytes(heads, max_draft)``, else one is taken from torch's allocator.

    Returns (out, lse): out like q, lse [tokens, heads] f32.  A token that
    attends nothing gets 0 and -inf."""
    return _kvops.tree_attention(cache._ref, q, k, v, lens, indptr, mask, layer, max_draft, scale, out, lse, work)



def attention_mass(q: torch.Tensor, lse: torch.Tensor, cache: PagedCache, lens: torch.Tensor, indptr: torch.Tensor, *,
                   layer: int = 0, max_draft: Optional[int] = None, scale: Optional[float] = None,
                   counted: Optional[torch.Tensor] = None, acc: Optional[torch.Tensor] = None, decay: float = 1.0,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The attention weight that each cached position got from the tokens, per
    kv head, added to ``decay`` times the sums so far.

    q, lens, indptr, max_draft and scale as ``tree_attention`` took them, lse
    as it returned it.  ``counted`` [batch] int64: bit i counts the sequence's
    token i (the accepted ones, say), all without it.  ``acc`` [batch, kv
    heads, width] f32, or None for zeros.  Returns the new sums, [batch, kv heads,
    width] (the cache's capacity without acc), 0 past each length; ``out`` may be
    ``acc`` itself."""
    return _kvops.attention_mass(cache._ref, q, lse, lens, indptr, layer, max_draft, scale, counted, acc, decay, out)



def select(cache: PagedCache, acc: torch.Tensor, lens: torch.Tensor, *, keep: int, sinks: int = 0,
           recent: int = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The positions that a cut to ``keep`` leaves of each layer, sequence and
    kv head: all where the length is at most ``keep``, else the first ``sinks``,
    the last ``recent`` and of the others those with the largest sums, the lower
    position first among equals.  ``acc`` [layers, batch, kv heads, width] f32; of a
    length above the width the first ``width`` positions count.

    Returns (idx, sums, new_lens): idx [layers, batch, kv heads, keep] int32 in
    rising order, -1 past the count, with their sums (0 there), and [batch]
    int32."""
    return _kvops.select(cache._ref, acc, lens, keep, sinks, recent)



def _other(cache: PagedCache, into: Optional[PagedCache]) -> PagedCache:
    if into is None:
        return cache
    if into.device != cache.device:
        raise ValueError(f"into must be on {cache.device}")
    return into


def compact(cache: PagedCache, idx: torch.Tensor, *, into: Optional[PagedCache] = None) -> None:
    """Moves the positions that ``idx`` (from :func:`select`) names to the
    front, in place or into the pages of another cache of the same shape
    (which share nothing with this one's), with room for them.  All these
    positions' pages have to be mapped."""
    _kvops.compact(cache._ref, idx, _other(cache, into)._ref)



def evict(cache: PagedCache, acc: torch.Tensor, lens: torch.Tensor, *, keep: int, sinks: int = 0, recent: int = 0,
          into: Optional[PagedCache] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cuts the cache to ``keep`` positions a sequence (:func:`select` then
    :func:`compact`) and returns what select does.  Keys keep the rotary
    positions they were written with, so tokens after the cut go on counting
    from the old length: the caller keeps that count."""
    return _kvops.evict(cache._ref, acc, lens, keep, sinks, recent, _other(cache, into)._ref)



def append(cache: Union[PagedCache, PackedCache], k: torch.Tensor, v: torch.Tensor, lens: torch.Tensor, indptr: torch.Tensor, *,
           path: Optional[torch.Tensor] = None, n_path: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Writes tokens behind the cache, for all layers at once.

    k, v [layers, tokens, kv heads, head_dim]; ``indptr`` [batch + 1] int32
    bounds each sequence's tokens.  ``path`` [batch, most] int32 with ``n_path``
    [batch] int32 names the tokens of each sequence to write, in order (the
    accepted path through its tree); without them all are written.  A
    :class:`PackedCache` gets them quantised, from any of the three types.  Returns the new lengths."""
    return _kvops.append(cache._ref, k, v, lens, indptr, path, n_path)


def read(cache: PackedCache, lens: torch.Tensor, indptr: torch.Tensor, tokens: int, *, dtype: torch.dtype = torch.bfloat16,
         k: Optional[torch.Tensor] = None, v: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Reads positions of a packed cache back, all layers at once: what ``append`` with the same ``lens`` and ``indptr`` wrote.

    ``indptr`` [batch + 1] int32 says how many positions of each sequence, from ``lens`` [batch] int32 on, and where they go;
    ``tokens`` is the length of that flat axis (indptr's last value, which is on the device).  Returns k and v
    [layers, tokens, kv heads, head_dim] of ``dtype`` (or the tensors given, which share no memory), 0 where a position has no page; tokens behind
    indptr's last are not written."""
    return _kvops.read(cache._ref, lens, indptr, tokens, dtype, k, v)
