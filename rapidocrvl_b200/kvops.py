"""Operators on a paged K/V cache, on torch tensors: drafted tokens verified
over the cache in one pass, and the cache cut to a budget.

  tree_attention   drafted tokens (a tree, one bit mask a token) attend the
                   cache and one another; one token a sequence is the
                   ordinary decode step
  append           accepted drafts (or a prompt) written behind the cache
  attention_mass   the attention weight that cached positions received,
                   added to a running sum
  evict            keeps the first, the last and the most attended positions
                   (select, then compact)

All run on the tensors' device and torch's current stream, read lengths on the
device and wait for nothing, so they can be captured in a CUDA graph.  They call
the C ABI of include/ocrvl_cuda.h (ocrvl_op_tree_attn and following), whose
comments say what each computes; a wrong argument raises OcrvlError or
ValueError before anything runs.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Tuple

import torch

from . import _lib

MAX_DRAFT = 64
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}


def _stream(device: torch.device) -> int:
    if torch.cuda.current_device() != device.index:
        raise ValueError(f"the tensors are on {device}, the current device is cuda:{torch.cuda.current_device()}")
    return torch.cuda.current_stream(device).cuda_stream


def _ints(t, name: str, device, dtype=torch.int32, size: Optional[int] = None) -> int:
    if t.dtype is not dtype or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor on {device}")
    if size is not None and t.numel() != size:
        raise ValueError(f"{name} must hold {size} values, got {t.numel()}")
    return t.data_ptr()


def _tokens(t, name: str, cache: "PagedCache", heads: Optional[int] = None) -> int:
    """The stride between the tokens of [tokens, heads, head_dim] of the cache's type."""
    if t.dim() != 3 or t.dtype is not cache.dtype or t.device != cache.device:
        raise ValueError(f"{name} must be a [tokens, heads, head_dim] {cache.dtype} tensor on {cache.device}")
    n, h, d = t.shape
    s = t.stride()
    if d != cache.head_dim or (heads is not None and h != heads) or s[2] != 1 or (h > 1 and s[1] != d):
        raise ValueError(f"{name}: [tokens, {heads or 'heads'}, {cache.head_dim}] with the heads of a token contiguous "
                         f"is needed, got {tuple(t.shape)} with strides {s}")
    return s[0] if n > 1 else h * d


class PagedCache:
    """A paged cache: ``k`` and ``v`` are [pages, layers, kv heads, page_size,
    head_dim] tensors of the same type and strides (views of one pool, for
    instance) and ``table`` [batch, max_pages] int32 names the pages of each
    sequence in order, an entry outside 0..pages-1 none.  Page sizes are powers
    of two from 16 on, head_dim is 64 or 128."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor):
        if k.dim() != 5 or k.shape != v.shape or k.stride() != v.stride() or k.dtype is not v.dtype:
            raise ValueError("k and v must be [pages, layers, kv heads, page_size, head_dim] of one type and one set of strides")
        if k.dtype not in _TYPES or not k.is_cuda or v.device != k.device:
            raise ValueError("k and v must be float32, float16 or bfloat16 CUDA tensors")
        if k.stride(4) != 1:
            raise ValueError("head_dim must be contiguous")
        if table.dim() != 2 or table.dtype is not torch.int32 or table.device != k.device or table.stride(1) != 1:
            raise ValueError(f"table must be a [batch, max_pages] int32 tensor on {k.device}")
        self.k, self.v, self.table = k, v, table
        self.dtype, self.device = k.dtype, k.device
        pages, layers, heads, page, dim = k.shape
        d = _lib.KVCache(_TYPES[k.dtype], dim, heads, layers, page, pages, table.shape[0], table.shape[1], k.stride(0),
                         k.stride(1), k.stride(2), k.stride(3), max(table.stride(0), table.shape[1]), k.data_ptr(),
                         v.data_ptr(), table.data_ptr())
        self._set(d)

    def _set(self, d) -> None:
        self.desc, self._ref = d, C.byref(d)
        self.head_dim, self.kv_heads, self.layers, self.batch = d.head_dim, d.num_kv_heads, d.num_layers, d.batch
        self.capacity = d.max_pages * d.page_size
        self._work_bytes = None

    @classmethod
    def of_sequence(cls, seq) -> "PagedCache":
        """The cache of an engine sequence (``Runtime.new_sequence``): f32,
        every layer, one table row.  It stays valid while the sequence lives;
        order work on it against ``Runtime.stream_handle`` (the engine's calls
        wait for their own work before they return)."""
        self = cls.__new__(cls)
        d = _lib.KVCache()
        _lib.check(seq.rt._L.ocrvl_seq_kv_view(seq._h, C.byref(d)))
        self.k = self.v = self.table = None
        self._seq = seq  # holds the memory
        self.dtype, self.device = torch.float32, torch.device("cuda", seq.rt.device)
        self._set(d)
        return self

    def work_bytes(self) -> int:
        """Bytes of workspace a ``tree_attention`` call takes."""
        if self._work_bytes is None:
            n = C.c_int64()
            _lib.check(_lib.load().ocrvl_op_tree_attn_workspace(self._ref, self.kv_heads, 1, C.byref(n)))
            self._work_bytes = n.value
        return self._work_bytes


def tree_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: PagedCache, lens: torch.Tensor,
                   indptr: torch.Tensor, mask: torch.Tensor, *, layer: int = 0, max_draft: Optional[int] = None,
                   scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                   lse: Optional[torch.Tensor] = None, work: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of drafted tokens over a cache and over one another.

    q [tokens, heads, head_dim]; k, v [tokens, kv heads, head_dim]: the drafts'
    own keys and values, which are not in the cache yet.  ``indptr`` [batch + 1]
    int32 bounds each sequence's tokens, ``lens`` [batch] int32 are the cached
    lengths.  ``mask`` [tokens] int64: bit j lets the token attend its
    sequence's token j, its own included only if set (-1: all).  ``max_draft``
    bounds the tokens of a sequence (64 at most, which is the default; more
    are not computed and their outputs not written).  ``work``: a uint8 tensor
    of ``cache.work_bytes()``, else one is taken from torch's allocator.

    Returns (out, lse): out like q, lse [tokens, heads] f32.  A token that
    attends nothing gets 0 and -inf."""
    n, heads = q.shape[0], q.shape[1]
    q_stride, kv_stride = _tokens(q, "q", cache), _tokens(k, "k", cache, cache.kv_heads)
    if _tokens(v, "v", cache, cache.kv_heads) != kv_stride or k.shape[0] != n or v.shape[0] != n:
        raise ValueError("k and v must have q's tokens and the same stride")
    if out is None:
        out = torch.empty((n, heads, cache.head_dim), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape:
        raise ValueError("out must have q's shape")
    if lse is None:
        lse = torch.empty((n, heads), dtype=torch.float32, device=q.device)
    if work is None:
        work = torch.empty(cache.work_bytes(), dtype=torch.uint8, device=q.device)
    dev = cache.device
    _lib.check(_lib.load().ocrvl_op_tree_attn(
        cache._ref, layer, heads, n, min(MAX_DRAFT, max(1, n)) if max_draft is None else max_draft,
        _ints(lens, "lens", dev, size=cache.batch), _ints(indptr, "indptr", dev, size=cache.batch + 1),
        _ints(mask, "mask", dev, torch.int64, n), q.data_ptr(), q_stride, k.data_ptr(), v.data_ptr(), kv_stride,
        1.0 / math.sqrt(cache.head_dim) if scale is None else scale, out.data_ptr(), _tokens(out, "out", cache, heads),
        _ints(lse, "lse", dev, torch.float32, n * heads), work.data_ptr(), work.numel(), _stream(dev)))
    return out, lse


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
    n, heads = q.shape[0], q.shape[1]
    q_stride = _tokens(q, "q", cache)
    dev, L = cache.device, _lib.load()
    if out is None:
        width = cache.capacity if acc is None else acc.shape[-1]
        out = torch.empty((cache.batch, cache.kv_heads, width), dtype=torch.float32, device=dev)
    _lib.check(L.ocrvl_op_attn_mass(
        cache._ref, layer, heads, n, min(MAX_DRAFT, max(1, n)) if max_draft is None else max_draft,
        _ints(lens, "lens", dev, size=cache.batch), _ints(indptr, "indptr", dev, size=cache.batch + 1),
        None if counted is None else _ints(counted, "counted", dev, torch.int64, cache.batch), q.data_ptr(), q_stride,
        _ints(lse, "lse", dev, torch.float32, n * heads), 1.0 / math.sqrt(cache.head_dim) if scale is None else scale, decay,
        None if acc is None else acc.data_ptr(), 0 if acc is None else acc.shape[-1],
        0 if acc is None else _rows(acc, "acc", cache, (cache.batch, cache.kv_heads)),
        out.data_ptr(), out.shape[-1], _rows(out, "out", cache, (cache.batch, cache.kv_heads)), _stream(dev)))
    return out


def _rows(t, name: str, cache: PagedCache, lead: tuple) -> int:
    """The stride between the rows of an f32 tensor [*lead, width]."""
    if t.dtype is not torch.float32 or t.device != cache.device or tuple(t.shape[:-1]) != lead or t.stride(-1) != 1:
        raise ValueError(f"{name} must be a [{', '.join(map(str, lead))}, width] float32 tensor on {cache.device}")
    size, row = 1, None
    for dim in range(len(lead) - 1, -1, -1):
        if lead[dim] > 1:
            if row is None:
                row = t.stride(dim) // size if t.stride(dim) % size == 0 else -1
            elif t.stride(dim) != row * size:
                raise ValueError(f"{name}: the rows must be one stride apart, got strides {t.stride()}")
        size *= lead[dim]
    return t.shape[-1] if row is None else row


def select(cache: PagedCache, acc: torch.Tensor, lens: torch.Tensor, *, keep: int, sinks: int = 0,
           recent: int = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The positions that a cut to ``keep`` leaves of each layer, sequence and
    kv head: all where the length is at most ``keep``, else the first ``sinks``,
    the last ``recent`` and of the others those with the largest sums, the lower
    position first among equals.  ``acc`` [layers, batch, kv heads, width] f32.

    Returns (idx, sums, new_lens): idx [layers, batch, kv heads, keep] int32 in
    rising order, -1 past the count, with their sums (0 there), and [batch]
    int32."""
    dev = cache.device
    lead = (cache.layers, cache.batch, cache.kv_heads)
    stride = _rows(acc, "acc", cache, lead)
    idx = torch.empty((*lead, max(keep, 0)), dtype=torch.int32, device=dev)
    sums = torch.empty((*lead, max(keep, 0)), dtype=torch.float32, device=dev)
    new_lens = torch.empty(cache.batch, dtype=torch.int32, device=dev)
    _lib.check(_lib.load().ocrvl_op_kv_select(*lead, acc.data_ptr(), acc.shape[-1], stride,
                                              _ints(lens, "lens", dev, size=cache.batch), keep, sinks, recent,
                                              idx.data_ptr(), sums.data_ptr(), new_lens.data_ptr(), _stream(dev)))
    return idx, sums, new_lens


def compact(cache: PagedCache, idx: torch.Tensor, *, into: Optional[PagedCache] = None) -> None:
    """Moves the positions that ``idx`` (from :func:`select`) names to the
    front, in place or into the pages of another cache of the same shape
    (which share nothing with this one's)."""
    to = cache if into is None else into
    lead = (cache.layers, cache.batch, cache.kv_heads)
    if idx.dim() != 4 or tuple(idx.shape[:3]) != lead:
        raise ValueError(f"idx must be [{', '.join(map(str, lead))}, keep]")
    _lib.check(_lib.load().ocrvl_op_kv_compact(cache._ref, to._ref, _ints(idx, "idx", cache.device), idx.shape[3],
                                               _stream(cache.device)))


def evict(cache: PagedCache, acc: torch.Tensor, lens: torch.Tensor, *, keep: int, sinks: int = 0, recent: int = 0,
          into: Optional[PagedCache] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cuts the cache to ``keep`` positions a sequence (:func:`select` then
    :func:`compact`) and returns what select does.  Keys keep the rotary
    positions they were written with, so tokens after the cut go on counting
    from the old length: the caller keeps that count."""
    idx, sums, new_lens = select(cache, acc, lens, keep=keep, sinks=sinks, recent=recent)
    compact(cache, idx, into=into)
    return idx, sums, new_lens


def append(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, lens: torch.Tensor, indptr: torch.Tensor, *,
           path: Optional[torch.Tensor] = None, n_path: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Writes tokens behind the cache, for all layers at once.

    k, v [layers, tokens, kv heads, head_dim]; ``indptr`` [batch + 1] int32
    bounds each sequence's tokens.  ``path`` [batch, most] int32 with ``n_path``
    [batch] int32 names the tokens of each sequence to write, in order (the
    accepted path through its tree); without them all are written.  Returns
    the new lengths."""
    dev = cache.device
    if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.shape[0] != cache.layers:
        raise ValueError(f"k and v must be [{cache.layers}, tokens, {cache.kv_heads}, {cache.head_dim}] of the same strides")
    stride = _tokens(k[0], "k", cache, cache.kv_heads)
    if v.dtype is not k.dtype or v.device != k.device:
        raise ValueError("k and v must be of one type on one device")
    if (path is None) != (n_path is None) or (path is not None and (path.dim() != 2 or path.shape[0] != cache.batch)):
        raise ValueError(f"path must be [{cache.batch}, most], with n_path")
    new_lens = torch.empty(cache.batch, dtype=torch.int32, device=dev)
    _lib.check(_lib.load().ocrvl_op_kv_append(
        cache._ref, k.shape[1], _ints(lens, "lens", dev, size=cache.batch), _ints(indptr, "indptr", dev, size=cache.batch + 1),
        None if path is None else _ints(path, "path", dev), None if path is None else _ints(n_path, "n_path", dev, size=cache.batch),
        0 if path is None else path.shape[1], k.data_ptr(), v.data_ptr(), stride, k.stride(0) if k.shape[0] > 1 else 0,
        new_lens.data_ptr(), _stream(dev)))
    return new_lens
