"""Argument checks of the paged-cache and score entry points that need no GPU: bad sizes
and null pointers are refused before any CUDA call."""

import ctypes

import pytest
import torch

from scree_b200 import _lib


def _book(S=4, M=4, P=16, page=16, ptr=16, out=None):
    return ctypes.byref(_lib.PagedBook(ptr, ptr, ptr, out or 32, out or 32, out or 32, S, M, P, page))


def _pools(L=1, H=2, row_bytes=128, ptr=16):
    return ctypes.byref(_lib.PagedPools(ptr, ptr, L, H, row_bytes))


def _ws(S=4, P=16):
    return 16, _lib.load().scree_paged_workspace_size(S, P)


def test_workspace_sizes():
    lib = _lib.load()
    assert lib.scree_paged_workspace_size(0, 5) == 0 and lib.scree_paged_workspace_size(4, 16) == 4 * (16 + 16 + 48)
    few = lib.scree_attn_fwd_paged_workspace_size(4, 4, 8, 2, 128)
    many = lib.scree_attn_fwd_paged_workspace_size(4, 400, 8, 2, 128)
    assert 0 < few < many  # one tile of 16 rows a worker, pairs of 128
    assert lib.scree_attn_fwd_paged_workspace_size(4, 4, 8, 3, 128) == 0


@pytest.mark.parametrize("book", [dict(S=0), dict(S=65537), dict(M=0), dict(P=0), dict(page=0), dict(ptr=None),
                                  dict(out=16)])
def test_bookkeeping_is_checked(book):
    lib = _lib.load()
    assert lib.scree_paged_reserve(_book(**book), 16, 16, 1, *_ws(), None) == _lib.SCREE_ERR_INVALID
    assert lib.scree_paged_free(_book(**book), 16, 1, *_ws(), None) == _lib.SCREE_ERR_INVALID
    assert "paged_free" in _lib.last_error()


def test_entries_workspaces_and_pools_are_checked():
    lib = _lib.load()
    bad = _lib.SCREE_ERR_INVALID
    assert lib.scree_paged_reserve(_book(), 16, 16, 5, *_ws(), None) == bad  # 5 entries, 4 slots
    assert "5 entries for 4 slots" in _lib.last_error()
    assert lib.scree_paged_reserve(_book(), None, 16, 1, *_ws(), None) == bad
    assert lib.scree_paged_reserve(_book(), 16, 16, 1, 16, 8, None) == bad
    assert "workspace" in _lib.last_error()
    assert lib.scree_paged_reserve(None, 16, 16, 1, *_ws(), None) == bad
    assert lib.scree_paged_compact(_book(), None, *_ws(), None) == bad
    assert lib.scree_paged_compact(_book(), _pools(row_bytes=0), *_ws(), None) == bad
    assert lib.scree_paged_accept(_book(), _pools(), 16, 16, 16, -1, 1, *_ws(), None) == bad
    write = [_pools(), 16, 16, 4, 4, 16, 16, 0, 16, 16, 256, 128, 16, 256, 128, 16, 0, 1, 3, None]
    for at, value in ((0, None), (0, _pools(H=0)), (3, 0), (7, 1), (7, -1), (9, None), (17, 0)):
        args = list(write)
        args[at] = value
        assert lib.scree_paged_write(*args) == bad, at
    assert lib.scree_tree_mask(None, 16, 0, 1, 3, 1, 16, None) == bad
    assert lib.scree_tree_mask(16, 16, 0, 1, 3, 0, 16, None) == bad


def test_attention_arguments_are_checked():
    lib = _lib.load()
    base = [16, 256, 64, _pools(), 0, 16, 16, 4, 4, 16, 16, 16, 16, 0, 2, 3, 4, 64, _lib.BF16, 0.125, None, 0, 16, 256,
            64, None, 16, 1 << 30, None]
    cases = [(3, None, _lib.SCREE_ERR_INVALID), (16, 3, _lib.SCREE_ERR_INVALID), (14, 4097, _lib.SCREE_ERR_INVALID),
             (17, 96, _lib.SCREE_ERR_UNSUPPORTED), (18, _lib.F32, _lib.SCREE_ERR_UNSUPPORTED),
             (17, 128, _lib.SCREE_ERR_INVALID), (10, 24, _lib.SCREE_ERR_INVALID), (4, 1, _lib.SCREE_ERR_INVALID),
             (0, None, _lib.SCREE_ERR_INVALID), (0, 24, _lib.SCREE_ERR_INVALID), (1, 252, _lib.SCREE_ERR_INVALID),
             (22, 24, _lib.SCREE_ERR_INVALID), (26, 8, _lib.SCREE_ERR_INVALID)]
    for at, value, want in cases:
        args = list(base)
        args[at] = value
        assert lib.scree_attn_fwd_paged(*args) == want, (at, value, _lib.last_error())
    mask = list(base)
    mask[20] = 16  # a mask of no words
    assert lib.scree_attn_fwd_paged(*mask) == _lib.SCREE_ERR_INVALID
    none = list(base)
    none[15] = 0  # no tokens: nothing to do
    assert lib.scree_attn_fwd_paged(*none) == _lib.SCREE_OK


def test_score_arguments_are_checked():
    lib = _lib.load()
    base = [16, 100, 16, 1, 4, 100, 5, _lib.BF16, 16, 16, 16, 16, 16, None]
    for at, value in ((0, None), (0, 17), (1, 99), (2, None), (4, -1), (5, 0), (6, 33), (6, -1), (7, 7), (8, None),
                      (10, 20), (11, None)):
        args = list(base)
        args[at] = value
        assert lib.scree_token_logprobs_fwd(*args) == _lib.SCREE_ERR_INVALID, (at, value)
    args = list(base)
    args[4] = 0
    assert lib.scree_token_logprobs_fwd(*args) == _lib.SCREE_OK
    back = [16, 100, 16, 1, 16, 16, None, 16, None, 16, 4, 100, 5, _lib.BF16, 16, None]
    assert lib.scree_token_logprobs_bwd(*back) == _lib.SCREE_ERR_INVALID  # alternatives' gradient without their ids


def test_python_entry_points_want_cuda_tensors():
    import scree_b200 as scree
    from scree_b200 import paged
    from scree_b200.kernels import varlen_token_logprobs

    cpu = torch.zeros((1, 2, 1, 16, 8))
    i32 = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(TypeError, match="CUDA"):
        paged.PagedCache(k=cpu, v=cpu, table=torch.zeros((2, 1), dtype=torch.int32), lengths=i32, refs=i32)
    arr = scree.Array(torch.zeros((3, 7)), torch.tensor([0, 3]))
    with pytest.raises(TypeError, match="CUDA"):
        varlen_token_logprobs(arr, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(TypeError, match="CUDA"):
        paged.tree_mask(scree.Array(torch.zeros(3, dtype=torch.int32), torch.tensor([0, 3])))
    again = arr._with_values(torch.ones((3, 2)))
    assert again.offsets is arr.offsets and again.batch_size == 1 and again.feature_shape == (2,)
    with pytest.raises(AssertionError):
        arr._with_values(torch.ones((2, 2)))
