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
free pages, a draft on shared pages) leaves the bookkeeping as it was, or the
rows unwritten, and sets the device status word, which
``scree_b200._lib.raise_device_status()`` turns into ``ScreeError``.  All calls
on one cache must be ordered on the GPU (one stream, or streams that wait for
one another).
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
    _pools: Any = field(default=None, repr=False, compare=False)

    def __post_init__(self) -> None:
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
        L, P, H, page, D = self.k.shape
        S, M = self.table.shape
        pools = _lib.PagedPools(self.k.data_ptr(), self.v.data_ptr(), L, H, D * self.k.element_size())
        # What every call of this cache and those derived from it passes on.
        pools.sizes = (S, M, P, page, H, D)
        pools.dtype, pools.device = self.k.dtype, self.k.device
        pools.ref, pools.work_bytes = ctypes.byref(pools), _lib.load().scree_paged_workspace_size(S, P)
        pools.work_at = -(-4 * (S * M + S + P) // 16) * 16  # bytes, in a call's allocation
        pools.ints = (pools.work_at + pools.work_bytes) // 4
        object.__setattr__(self, "_pools", pools)

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


def _ints(t, n, what, device):
    """An int32 CUDA vector (of n entries, if n is given) next to the cache."""
    if not (isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.device == device):
        raise TypeError(f"{what} must be an int32 tensor on the cache's device")
    if t.ndim != 1 or (n is not None and t.shape[0] != n):
        raise ValueError(f"{what} must be 1-D" + (f" with {n} entries" if n is not None else ""))
    return t if t.is_contiguous() else t.contiguous()


def _book_call(cache: PagedCache, fn, name: str, *args) -> PagedCache:
    pools = cache._pools
    S, M, P, page, _, _ = pools.sizes
    # One allocation: the new bookkeeping, and behind it the plan's workspace.  That is the call's
    # own, of the stream it runs on: another call, on another stream or thread, cannot come between
    # the plan and its apply.
    buf = cache.refs.new_empty(pools.ints)
    table = buf.as_strided((S, M), (M, 1), 0)
    lengths = buf.as_strided((S,), (1,), S * M)
    refs = buf.as_strided((P,), (1,), S * M + S)
    at = buf.data_ptr()
    book = _lib.PagedBook(cache.table.data_ptr(), cache.lengths.data_ptr(), cache.refs.data_ptr(), at, at + 4 * S * M,
                          at + 4 * (S * M + S), S, M, P, page)
    rc = fn(ctypes.byref(book), *args, at + pools.work_at, pools.work_bytes, _lib.stream_ptr(pools.device))
    if rc:
        _lib.check(rc, name)
    out = object.__new__(PagedCache)  # nothing to check: the same pools and shapes
    out.__dict__.update(cache.__dict__, table=table, lengths=lengths, refs=refs)
    return out


def paged_reserve(cache: PagedCache, slots, counts) -> PagedCache:
    """Grows slot slots[i] by counts[i] tokens, from the lowest free pages."""
    dev = cache._pools.device
    slots = _ints(slots, None, "slots", dev)
    n = slots.shape[0]
    counts = _ints(counts, n, "counts", dev)
    return _book_call(cache, _lib.load().scree_paged_reserve, "paged_reserve", slots.data_ptr(), counts.data_ptr(), n)


def paged_accept(cache: PagedCache, slots, drafted, path) -> PagedCache:
    """Of the last drafted[i] tokens of slot slots[i], keeps those whose indices into the
    draft row i of ``path`` (n, depth) lists, ascending and ended by -1; their rows move to
    the front of the draft in every layer, the others are dropped and their pages freed."""
    dev = cache._pools.device
    slots = _ints(slots, None, "slots", dev)
    n = slots.shape[0]
    drafted = _ints(drafted, n, "drafted", dev)
    if not (isinstance(path, torch.Tensor) and path.dtype == torch.int32 and path.device == dev):
        raise TypeError("path must be an int32 tensor on the cache's device")
    if path.ndim != 2 or path.shape[0] != n:
        raise ValueError("path must be (slots, depth)")
    path = path.contiguous()
    return _book_call(cache, _lib.load().scree_paged_accept, "paged_accept", cache._pools.ref, slots.data_ptr(),
                      drafted.data_ptr(), path.data_ptr(), path.shape[1], n)


def paged_fork(cache: PagedCache, parents, children) -> PagedCache:
    """The empty slots children[i] become copies of parents[i] (which may repeat, and may not
    be children): full pages are shared, a part-filled page is copied."""
    dev = cache._pools.device
    parents = _ints(parents, None, "parents", dev)
    n = parents.shape[0]
    children = _ints(children, n, "children", dev)
    return _book_call(cache, _lib.load().scree_paged_fork, "paged_fork", cache._pools.ref, parents.data_ptr(),
                      children.data_ptr(), n)


def paged_free(cache: PagedCache, slots) -> PagedCache:
    """Empties the slots; pages that no other slot holds become free."""
    slots = _ints(slots, None, "slots", cache._pools.device)
    return _book_call(cache, _lib.load().scree_paged_free, "paged_free", slots.data_ptr(), slots.shape[0])


def paged_compact(cache: PagedCache) -> PagedCache:
    """Moves used pages so that they are the first of the pools; of the pages above their
    count, the k-th used one goes to the k-th hole below it."""
    return _book_call(cache, _lib.load().scree_paged_compact, "paged_compact", cache._pools.ref)


def _offsets(arr: Array, device):
    """Offsets on the device, whether they are int64, sequences."""
    offs = arr.offsets
    if not (isinstance(offs, torch.Tensor) and offs.device == device and offs.dtype in (torch.int32, torch.int64)):
        offs = torch.as_tensor(arr.host_offsets(), dtype=torch.int64, device=device)
    if not offs.is_contiguous():
        offs = offs.contiguous()
    return offs, 1 if offs.dtype == torch.int64 else 0, offs.shape[0] - 1


def paged_write(cache: PagedCache, layer: int, slots, k: Array, v: Array) -> None:
    """Writes the rows of sequence b of k / v (T, kv_heads, head_dim) as the K / V of the last
    tokens of slot slots[b] in one layer.  Not written, with the status word set: the rows of
    sequences that name one slot, or have more tokens than it holds, rows on a page that other
    slots hold, and all rows if k and v have different offsets."""
    if k.ragged_dim != 0 or v.ragged_dim != 0:
        raise NotImplementedError("paged_write supports ragged_dim=0 only in v0.1")
    kt, vt, pools = k.values, v.values, cache._pools
    S, M, P, page, H, D = pools.sizes
    dev = pools.device
    if kt.ndim != 3 or kt.shape[1] != H or kt.shape[2] != D or kt.shape != vt.shape:
        raise ValueError(f"k and v must be (tokens, {H}, {D})")
    if kt.dtype != pools.dtype or vt.dtype != pools.dtype:
        raise ValueError("k and v must have the cache's dtype")
    if kt.device != dev or vt.device != dev:
        raise TypeError("k and v must be on the cache's device")
    offs, is64, B = _offsets(k, dev)
    slots = _ints(slots, B, "slots", dev)
    v_offs = None
    if v.offsets is not k.offsets:  # compared on the device, so that nothing is read from it
        v_offs, v_is64, v_batch = _offsets(v, dev)
        if v_batch != B:
            raise ValueError(f"k and v must have identical offsets ({B} and {v_batch} sequences)")
        if v_is64 != is64:
            v_offs = v_offs.to(offs.dtype)
    (kr, kh, kd), (vr, vh, vd) = kt.stride(), vt.stride()
    if kd != 1 or vd != 1:
        kt, vt = kt.contiguous(), vt.contiguous()
        (kr, kh, _), (vr, vh, _) = kt.stride(), vt.stride()
    es = kt.element_size()
    rc = _lib.load().scree_paged_write_ex(
        pools.ref, cache.table.data_ptr(), cache.lengths.data_ptr(), cache.refs.data_ptr(), S, M, P, page, layer,
        slots.data_ptr(), kt.data_ptr(), kr * es, kh * es, vt.data_ptr(), vr * es, vh * es, offs.data_ptr(),
        None if v_offs is None else v_offs.data_ptr(), is64, B, kt.shape[0], _lib.stream_ptr(dev))
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
    vals = parents.values.contiguous()
    offs, is64, B = _offsets(parents, vals.device)
    words = max(1, -(-int(max_nodes) // 64))
    mask = torch.empty((vals.shape[0], words), dtype=torch.int64, device=vals.device)
    rc = _lib.load().scree_tree_mask(vals.data_ptr(), offs.data_ptr(), is64, B, vals.shape[0], words,
                                     mask.data_ptr(), _lib.stream_ptr(vals.device))
    _lib.check(rc, "tree_mask")
    return mask


def paged_attention(q: Array, cache: PagedCache, layer: int, slots, mask=None, return_lse: bool = False):
    """Attention of each sequence's new tokens over its slot, scale 1/sqrt(head_dim).

    ``q`` (T, heads, head_dim) fp16 / bf16: the queries of sequence b are the last tokens of slot
    slots[b], whose K / V ``paged_write`` has written.  They see every earlier token, and of
    their own number those that their row of ``mask`` names (``tree_mask``, or any (T, words)
    int64 bits), or the earlier ones and themselves if mask is None.  A query that sees nothing
    gets 0 and LSE -inf.  heads is a multiple of the cache's kv_heads; head_dim 32, 64 or 128;
    page_size a multiple of 16; at most 4096 sequences.  The probabilities are rounded to q's
    dtype for their product with V; sums are fp32.  Infinities and NaN in the K / V of new tokens
    reach the queries that see them and no others; earlier tokens' are taken to be finite.
    Forward only (inference), like ``varlen_attention_kv``: the result has no gradient.  Returns
    an Array on q's offsets (and the LSE (T, heads) fp32 when ``return_lse``)."""
    qt, pools = q.values, cache._pools
    _require_cuda(qt, "paged_attention")
    if q.ragged_dim != 0:
        raise NotImplementedError("paged_attention supports ragged_dim=0 only in v0.1")
    S, M, P, page, Hkv, D = pools.sizes
    dev, dtype = qt.device, qt.dtype
    assert dtype in (torch.float16, torch.bfloat16), "fp16 or bf16 only"
    assert dtype == pools.dtype and dev == pools.device, "q must have the cache's dtype and device"
    assert qt.ndim == 3 and qt.shape[2] == D and qt.shape[1] % Hkv == 0, \
        "q must be (tokens, heads, head_dim) with heads a multiple of the cache's kv_heads"
    T, H, _ = qt.shape
    offs, is64, B = _offsets(q, dev)
    slots = _ints(slots, B, "slots", dev)
    mask_ptr, words = None, 0
    if mask is not None:
        if not (isinstance(mask, torch.Tensor) and mask.dtype == torch.int64 and mask.device == dev):
            raise TypeError("mask must be an int64 tensor on q's device")
        if mask.ndim != 2 or mask.shape[0] != T or mask.shape[1] < 1:
            raise ValueError("mask must be (tokens, words)")
        mask = mask.contiguous()
        mask_ptr, words = mask.data_ptr(), mask.shape[1]
    sr, sh, sd = qt.stride()
    if sd != 1 or sr % 8 or sh % 8 or sr * sh == 0 or qt.data_ptr() % 16:
        qt = qt.clone(memory_format=torch.contiguous_format)  # contiguous() would keep a misaligned base
        sr, sh, _ = qt.stride()
    out = torch.empty_like(qt, memory_format=torch.contiguous_format)  # (1.3 us, empty 1.6)
    lse = torch.empty((T, H), dtype=torch.float32, device=dev) if return_lse else None
    if T:
        lib = _lib.load()
        size = lib.scree_attn_fwd_paged_workspace_size(B, T, H, Hkv, D)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        rc = lib.scree_attn_fwd_paged(
            qt.data_ptr(), sr, sh, pools.ref, layer, cache.table.data_ptr(), cache.lengths.data_ptr(), S, M, P, page,
            slots.data_ptr(), offs.data_ptr(), is64, B, T, H, D, _lib.BF16 if dtype == torch.bfloat16 else _lib.F16,
            1.0 / math.sqrt(D), mask_ptr, words, out.data_ptr(), H * D, D, lse.data_ptr() if return_lse else None,
            ws.data_ptr(), size, _lib.stream_ptr(dev))
        if rc:
            _lib.check(rc, "paged_attention")
    res = q._with_values(out)
    return (res, lse) if return_lse else res
