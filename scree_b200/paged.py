"""A paged K/V cache and attention over it (no reference counterpart; the
reference lists KV-cache support as planned, docs/kernels.md:178).

  cache = paged_cache(layers, pages, page_size, kv_heads, head_dim, slots, max_pages, dtype)
  cache = paged_reserve(cache, slots, counts)      room for new tokens
  paged_write(cache, layer, slots, k, v)           their K / V, layer by layer
  out   = paged_attention(q, cache, layer, slots, mask=None)
  cache = paged_accept(cache, slots, drafted, path)  keep one path of a drafted tree
  cache = paged_fork(cache, parents, children)     share a prefix, copy what is not full
  cache = paged_free(cache, slots)
  cache = paged_compact(cache)                     used pages to the front of the pools
  mask  = tree_mask(parents)                       who sees whom in drafted trees

A ``PagedCache`` is immutable like ``Array``: every call returns a new one with
new bookkeeping tensors; the K / V pools are shared and updated in place.
Slots, counts and paths are int32 CUDA tensors and nothing here reads them on
the host.  What a call cannot do (a slot out of range or named twice, too few
free pages, a draft on shared pages) leaves the bookkeeping as it was and sets
the device status word, which ``scree_b200._lib.raise_device_status()`` turns
into ``ScreeError``.  All calls on one cache must be ordered on the GPU (one
stream, or streams that wait for one another).
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass, field
from typing import Any

import torch

from . import _lib
from ._core import Array, _require_cuda

__all__ = ["PagedCache", "paged_cache", "paged_reserve", "paged_write", "paged_accept", "paged_fork",
           "paged_free", "paged_compact", "paged_attention", "tree_mask"]


@dataclass(frozen=True)
class PagedCache:
    """K / V pools (layers, pages, kv_heads, page_size, head_dim) and their bookkeeping:
    ``table`` (slots, max_pages) page ids, -1 beyond a slot's pages; ``lengths`` (slots,)
    tokens of each slot, 0 if free; ``refs`` (pages,) slots that hold each page; all int32."""

    k: Any
    v: Any
    table: Any
    lengths: Any
    refs: Any
    _work: Any = field(default=None, repr=False, compare=False)  # plan workspace, shared by derived caches
    _pools: Any = field(default=None, repr=False, compare=False)

    def __post_init__(self) -> None:
        if self._pools is not None:
            return  # derived from a checked cache
        for name in ("k", "v", "table", "lengths", "refs"):
            _require_cuda(getattr(self, name), "PagedCache")
        if self.k.ndim != 5 or self.k.shape != self.v.shape or self.k.dtype != self.v.dtype:
            raise ValueError("k and v must be (layers, pages, kv_heads, page_size, head_dim) of one shape and dtype")
        if not (self.k.is_contiguous() and self.v.is_contiguous()):
            raise ValueError("k and v must be contiguous")
        if self.table.ndim != 2 or self.lengths.shape != self.table.shape[:1] or self.refs.shape != self.k.shape[1:2]:
            raise ValueError("table must be (slots, max_pages), lengths (slots,), refs (pages,)")
        for t in (self.table, self.lengths, self.refs):
            if t.dtype != torch.int32 or not t.is_contiguous():
                raise ValueError("table, lengths and refs must be contiguous int32")
        if len({t.device for t in (self.k, self.v, self.table, self.lengths, self.refs)}) != 1:
            raise ValueError("all tensors of a cache must be on one device")
        L, P, H, _, D = self.k.shape
        size = _lib.load().scree_paged_workspace_size(self.table.shape[0], P)
        object.__setattr__(self, "_work", torch.empty(size, dtype=torch.uint8, device=self.k.device))
        object.__setattr__(self, "_pools", _lib.PagedPools(self.k.data_ptr(), self.v.data_ptr(), L, H,
                                                           D * self.k.element_size()))

    @property
    def page_size(self) -> int:
        return int(self.k.shape[3])

    @property
    def slots(self) -> int:
        return int(self.table.shape[0])


def paged_cache(layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, slots: int,
                max_pages: int, dtype=torch.bfloat16, device="cuda") -> PagedCache:
    """An empty cache; a slot can hold up to max_pages * page_size tokens."""
    shape = (layers, pages, kv_heads, page_size, head_dim)
    i32 = dict(dtype=torch.int32, device=device)
    return PagedCache(k=torch.zeros(shape, dtype=dtype, device=device), v=torch.zeros(shape, dtype=dtype, device=device),
                      table=torch.full((slots, max_pages), -1, **i32), lengths=torch.zeros(slots, **i32),
                      refs=torch.zeros(pages, **i32))


def _ints(t, n, what, cache):
    """An int32 CUDA vector (of n entries, if n is given) next to the cache."""
    if not (isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.device == cache.k.device):
        raise TypeError(f"{what} must be an int32 tensor on the cache's device")
    if t.ndim != 1 or (n is not None and t.shape[0] != n):
        raise ValueError(f"{what} must be 1-D" + (f" with {n} entries" if n is not None else ""))
    return t.contiguous()


def _book_call(cache: PagedCache, name: str, *args) -> PagedCache:
    table, lengths, refs = torch.empty_like(cache.table), torch.empty_like(cache.lengths), torch.empty_like(cache.refs)
    S, M = cache.table.shape
    book = _lib.PagedBook(cache.table.data_ptr(), cache.lengths.data_ptr(), cache.refs.data_ptr(), table.data_ptr(),
                          lengths.data_ptr(), refs.data_ptr(), S, M, cache.refs.shape[0], cache.k.shape[3])
    rc = getattr(_lib.load(), name)(ctypes.byref(book), *args, cache._work.data_ptr(), cache._work.numel(),
                                    _lib.stream_ptr(cache.k.device))
    if rc:
        _lib.check(rc, name)
    return PagedCache(k=cache.k, v=cache.v, table=table, lengths=lengths, refs=refs, _work=cache._work,
                      _pools=cache._pools)


def paged_reserve(cache: PagedCache, slots, counts) -> PagedCache:
    """Grows slot slots[i] by counts[i] tokens, from the lowest free pages."""
    slots = _ints(slots, None, "slots", cache)
    counts = _ints(counts, slots.shape[0], "counts", cache)
    return _book_call(cache, "scree_paged_reserve", slots.data_ptr(), counts.data_ptr(), slots.shape[0])


def paged_accept(cache: PagedCache, slots, drafted, path) -> PagedCache:
    """Of the last drafted[i] tokens of slot slots[i], keeps those whose indices into the
    draft row i of ``path`` (n, depth) lists, ascending and ended by -1; their rows move to
    the front of the draft in every layer, the others are dropped and their pages freed."""
    slots = _ints(slots, None, "slots", cache)
    drafted = _ints(drafted, slots.shape[0], "drafted", cache)
    if not (isinstance(path, torch.Tensor) and path.dtype == torch.int32 and path.device == cache.k.device):
        raise TypeError("path must be an int32 tensor on the cache's device")
    if path.ndim != 2 or path.shape[0] != slots.shape[0]:
        raise ValueError("path must be (slots, depth)")
    path = path.contiguous()
    return _book_call(cache, "scree_paged_accept", ctypes.byref(cache._pools), slots.data_ptr(), drafted.data_ptr(),
                      path.data_ptr(), path.shape[1], slots.shape[0])


def paged_fork(cache: PagedCache, parents, children) -> PagedCache:
    """The empty slots children[i] become copies of parents[i] (which may repeat, and may not
    be children): full pages are shared, a part-filled page is copied."""
    parents = _ints(parents, None, "parents", cache)
    children = _ints(children, parents.shape[0], "children", cache)
    return _book_call(cache, "scree_paged_fork", ctypes.byref(cache._pools), parents.data_ptr(), children.data_ptr(),
                      parents.shape[0])


def paged_free(cache: PagedCache, slots) -> PagedCache:
    """Empties the slots; pages that no other slot holds become free."""
    slots = _ints(slots, None, "slots", cache)
    return _book_call(cache, "scree_paged_free", slots.data_ptr(), slots.shape[0])


def paged_compact(cache: PagedCache) -> PagedCache:
    """Moves used pages so that they are the first of the pools; of the pages above their
    count, the k-th used one goes to the k-th hole below it."""
    return _book_call(cache, "scree_paged_compact", ctypes.byref(cache._pools))


def _offsets(arr: Array):
    offs = arr.offsets
    if not (isinstance(offs, torch.Tensor) and offs.device == arr.values.device
            and offs.dtype in (torch.int32, torch.int64)):
        offs = torch.as_tensor(arr.host_offsets(), dtype=torch.int64, device=arr.values.device)
    return offs.contiguous()


def paged_write(cache: PagedCache, layer: int, slots, k: Array, v: Array) -> None:
    """Writes the rows of sequence b of k / v (T, kv_heads, head_dim) as the K / V of the last
    tokens of slot slots[b] in one layer."""
    slots = _ints(slots, k.batch_size, "slots", cache)
    kt, vt = k.values, v.values
    L, P, H, page, D = cache.k.shape
    if tuple(kt.shape[1:]) != (H, D) or kt.shape != vt.shape:
        raise ValueError(f"k and v must be (tokens, {H}, {D})")
    if kt.dtype != cache.k.dtype or vt.dtype != cache.k.dtype:
        raise ValueError("k and v must have the cache's dtype")
    if kt.device != cache.k.device or vt.device != cache.k.device:
        raise TypeError("k and v must be on the cache's device")
    if kt.stride(2) != 1:
        kt = kt.contiguous()
    if vt.stride(2) != 1:
        vt = vt.contiguous()
    offs = _offsets(k)
    es = kt.element_size()
    S, M = cache.table.shape
    rc = _lib.load().scree_paged_write(
        ctypes.byref(cache._pools), cache.table.data_ptr(), cache.lengths.data_ptr(), S, M, P, page, int(layer),
        slots.data_ptr(), kt.data_ptr(), kt.stride(0) * es, kt.stride(1) * es, vt.data_ptr(), vt.stride(0) * es,
        vt.stride(1) * es, offs.data_ptr(), 1 if offs.dtype == torch.int64 else 0, k.batch_size, kt.shape[0],
        _lib.stream_ptr(kt.device))
    if rc:
        _lib.check(rc, "paged_write")


def tree_mask(parents: Array, max_nodes: int = None):
    """Visibility of drafted trees for ``paged_attention``: ``parents`` holds each node's
    parent, an index within its sequence smaller than the node's own, or a negative number for
    a root.  Returns (T, ceil(max_nodes / 64)) int64 bit rows (bit j of node i: j is i or an
    ancestor of i); ``max_nodes`` bounds the nodes of a sequence (default: read from the
    offsets, which costs a host read if the Array does not hold them)."""
    _require_cuda(parents.values, "tree_mask")
    if parents.values.dtype != torch.int32 or parents.values.ndim != 1:
        raise TypeError("parents must hold 1-D int32 values")
    if max_nodes is None:
        host = parents.host_offsets()
        max_nodes = max(b - a for a, b in zip(host, host[1:]))
    vals, offs = parents.values.contiguous(), _offsets(parents)
    words = max(1, -(-int(max_nodes) // 64))
    mask = torch.empty((vals.shape[0], words), dtype=torch.int64, device=vals.device)
    rc = _lib.load().scree_tree_mask(vals.data_ptr(), offs.data_ptr(), 1 if offs.dtype == torch.int64 else 0,
                                     parents.batch_size, vals.shape[0], words, mask.data_ptr(),
                                     _lib.stream_ptr(vals.device))
    _lib.check(rc, "tree_mask")
    return mask


def paged_attention(q: Array, cache: PagedCache, layer: int, slots, mask=None, return_lse: bool = False):
    """Attention of each sequence's new tokens over its slot, scale 1/sqrt(head_dim).

    ``q`` (T, heads, head_dim) fp16 / bf16: the queries of sequence b are the last tokens of slot
    slots[b], whose K / V ``paged_write`` has written.  They see every earlier token, and of
    their own number those that their row of ``mask`` names (``tree_mask``, or any (T, words)
    int64 bits), or the earlier ones and themselves if mask is None.  A query that sees nothing
    gets 0 and LSE -inf.  heads is a multiple of the cache's kv_heads; head_dim 32, 64 or 128;
    page_size a multiple of 16; at most 4096 sequences.  Returns an Array on q's offsets (and
    the LSE (T, heads) fp32 when ``return_lse``)."""
    qt = q.values
    _require_cuda(qt, "paged_attention")
    slots = _ints(slots, q.batch_size, "slots", cache)
    assert qt.dtype in (torch.float16, torch.bfloat16), "fp16 or bf16 only"
    L, P, Hkv, page, D = cache.k.shape
    assert qt.dtype == cache.k.dtype and qt.device == cache.k.device, "q must have the cache's dtype and device"
    assert qt.ndim == 3 and qt.shape[2] == D and qt.shape[1] % Hkv == 0, \
        "q must be (tokens, heads, head_dim) with heads a multiple of the cache's kv_heads"
    T, H, _ = qt.shape
    words = 0
    if mask is not None:
        if not (isinstance(mask, torch.Tensor) and mask.dtype == torch.int64 and mask.device == qt.device):
            raise TypeError("mask must be an int64 tensor on q's device")
        if mask.ndim != 2 or mask.shape[0] != T or mask.shape[1] < 1:
            raise ValueError("mask must be (tokens, words)")
        mask = mask.contiguous()
        words = mask.shape[1]
    if qt.stride(2) != 1 or qt.stride(0) % 8 or qt.stride(1) % 8 or qt.data_ptr() % 16:
        qt = qt.clone(memory_format=torch.contiguous_format)  # contiguous() would keep a misaligned base
    out = torch.empty((T, H, D), dtype=qt.dtype, device=qt.device)
    lse = torch.empty((T, H), dtype=torch.float32, device=qt.device) if return_lse else None
    if T:
        lib = _lib.load()
        offs = _offsets(q)
        S, M = cache.table.shape
        B = q.batch_size
        ws = torch.empty(lib.scree_attn_fwd_paged_workspace_size(B, T, H, Hkv, D), dtype=torch.uint8, device=qt.device)
        rc = lib.scree_attn_fwd_paged(
            qt.data_ptr(), qt.stride(0), qt.stride(1), ctypes.byref(cache._pools), int(layer), cache.table.data_ptr(),
            cache.lengths.data_ptr(), S, M, P, page, slots.data_ptr(), offs.data_ptr(),
            1 if offs.dtype == torch.int64 else 0, B, T, H, D, _lib.dtype_code(qt.dtype), 1.0 / math.sqrt(D),
            mask.data_ptr() if mask is not None else None, words, out.data_ptr(), out.stride(0), out.stride(1),
            lse.data_ptr() if return_lse else None, ws.data_ptr(), ws.numel(), _lib.stream_ptr(qt.device))
        if rc:
            _lib.check(rc, "paged_attention")
    res = q._with_values(out)
    return (res, lse) if return_lse else res

