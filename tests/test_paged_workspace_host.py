"""A cache's calls share no workspace: what one has planned and not yet applied is not
another's to overwrite, on whatever stream or thread that one runs.  No GPU: the library call
is a stand-in that starts a second call in the middle of the first."""

import ctypes

import torch

from scree_b200 import _lib, paged


def _cache(monkeypatch):
    monkeypatch.setattr(paged, "_require_cuda", lambda *a: None)
    monkeypatch.setattr(_lib, "stream_ptr", lambda device=None: 0)
    kv = torch.zeros((1, 6, 1, 4, 8))
    i32 = dict(dtype=torch.int32)
    return paged.PagedCache(k=kv, v=kv.clone(), table=torch.full((3, 2), -1, **i32), lengths=torch.zeros(3, **i32),
                            refs=torch.zeros(6, **i32))


def test_calls_in_flight_have_workspaces_of_their_own(monkeypatch):
    cache = _cache(monkeypatch)
    need = _lib.load().scree_paged_workspace_size(3, 6)
    spans = []

    def call(book, workspace, size, stream):
        assert size >= need and workspace % 16 == 0
        spans.append((workspace, workspace + size))
        if len(spans) < 3:
            paged._book_call(cache, call, "inner")
        return 0

    out = paged._book_call(cache, call, "outer")
    assert len(spans) == 3
    for i, a in enumerate(spans):
        for b in spans[:i]:
            assert a[1] <= b[0] or b[1] <= a[0]
    for t, like in ((out.table, cache.table), (out.lengths, cache.lengths), (out.refs, cache.refs)):
        assert t.shape == like.shape and t.dtype == like.dtype and t.is_contiguous()
        end = t.data_ptr() + 4 * t.numel()
        assert end <= spans[0][0] or spans[0][1] <= t.data_ptr()
        assert all(end <= o.data_ptr() or o.data_ptr() + 4 * o.numel() <= t.data_ptr()
                   for o in (out.table, out.lengths, out.refs) if o is not t)
    # A derived cache keeps nothing of its call but the new bookkeeping.
    fresh = {k for k, v in out.__dict__.items() if v is not cache.__dict__.get(k)}
    assert fresh == {"table", "lengths", "refs"}


def test_a_cache_holds_no_memory_but_its_tensors(monkeypatch):
    cache = _cache(monkeypatch)
    held = [k for k, v in cache.__dict__.items() if isinstance(v, torch.Tensor)]
    assert sorted(held) == ["k", "lengths", "refs", "table", "v"]
    assert isinstance(cache._pools, ctypes.Structure)


def test_a_step_without_sequences_is_taken_by_every_entry_point():
    """No entries, no tokens: as reserve, accept, fork and free take n = 0 (they need a GPU)."""
    lib = _lib.load()
    pools = ctypes.byref(_lib.PagedPools(16, 16, 1, 2, 128))
    write = [pools, 16, 16, 4, 4, 16, 16, 0, 16, 16, 256, 128, 16, 256, 128, 16, 0, 0, 0, None]
    assert lib.scree_paged_write(*write) == _lib.SCREE_OK
    assert lib.scree_paged_write_ex(*write[:3], 16, *write[3:16], None, *write[16:]) == _lib.SCREE_OK
    assert lib.scree_tree_mask(16, 16, 0, 0, 0, 1, 16, None) == _lib.SCREE_OK
    attention = [16, 256, 64, pools, 0, 16, 16, 4, 4, 16, 16, 16, 16, 0, 0, 0, 4, 64, _lib.BF16, 0.125, None, 0, 16, 256,
                 64, None, 16, 1 << 30, None]
    assert lib.scree_attn_fwd_paged(*attention) == _lib.SCREE_OK
    # Tokens of no sequence are not.
    for args, fn in ((write[:18] + [3] + write[19:], lib.scree_paged_write), ([16, 16, 0, 0, 3, 1, 16, None], lib.scree_tree_mask),
                     (attention[:15] + [3] + attention[16:], lib.scree_attn_fwd_paged)):
        assert fn(*args) == _lib.SCREE_ERR_INVALID
