"""Edges of the paged cache and of attention over it on the GPU: what the calls refuse, and
results that depend on where the work is cut.  The model, the reference and the bounds are
those of test_gpu_paged.py."""

import numpy as np
import pytest
import torch
from test_gpu_paged import _causal, _compare, _i32, _make, _reference, _status

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16)])
def test_masked_tiles_of_long_and_short_pieces(cuda, D, dtype):
    """Pieces of one, two and several key tiles, one or two tiles of rows, in turn in every
    CTA: the V rows past each end (NaN here) are cleared in the place that holds them."""
    import scree_b200 as scree
    from scree_b200 import paged

    rng = np.random.default_rng(D)
    kinds = [(20, 21), (97, 33), (300, 40), (611, 17), (40, 100), (0, 25), (230, 64), (129, 70)]
    ctx, news = zip(*(kinds[i] for i in rng.integers(0, len(kinds), 120)))
    lens = [a + b for a, b in zip(ctx, news)]
    H, Hkv = 4, 2
    cache, slots, hs = _make(cuda, lens, 16, Hkv, D, dtype, seed=D)
    q = torch.randn((sum(news), H, D), generator=torch.Generator().manual_seed(1)).to(dtype).to(cuda)
    offs = _i32(np.concatenate([[0], np.cumsum(news)]).tolist(), cuda)
    run = lambda: paged.paged_attention(scree.Array(q, offs), cache, 0, slots, return_lse=True)  # noqa: E731
    out, lse = run()
    _compare(out.values, lse, _reference(q, cache, 0, hs, lens, news, _causal(news)))
    for _ in range(20):
        again, lse2 = run()
        assert torch.equal(again.values, out.values) and torch.equal(lse2, lse)
    assert _status() == 0


def _far_apart(cuda, news, D, dtype, low, seed=2):
    """Sequences without context whose tokens before `low` (of the long ones) have scores of
    about -96 and infinities in V, the others +96: 2^-277 apart, below the smallest float."""
    cache, slots, hs = _make(cuda, news, 16, 1, D, dtype, seed=seed)
    for s, n in zip(hs, news):
        if n <= low:
            continue
        pos = torch.arange(n, device=cuda)
        ids = cache.table[int(s)].long()[pos // 16]
        b = (96.0 / D**0.5) * torch.where(pos < low, -1.0, 1.0)
        cache.k[0, ids, 0, pos % 16] = b[:, None].to(dtype).expand(n, D)
        cache.v[0, ids[3], 0, 3, :2] = float("inf")
        cache.v[0, ids[low - 1], 0, (low - 1) % 16, 2] = float("-inf")
    q = torch.ones((sum(news), 1, D), dtype=dtype, device=cuda)
    return cache, slots, hs, q


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,news,low", [
    (64, [40, 1, 1, 1], 32), (128, [20, 1], 16), (64, [40] * 200 + [1] * 330, 32),  # single rows: cut at each group; runs
    (128, [300], 128), (64, [300], 128), (128, [300] * 40, 128)])                    # tiles of 128: cut at each tile; runs
def test_visible_infinities_do_not_depend_on_the_cut(cuda, D, news, low, dtype):
    """An infinity of a drafted token's V reaches the rows that see it, however small its weight."""
    import scree_b200 as scree
    from scree_b200 import paged

    cache, slots, hs, q = _far_apart(cuda, news, D, dtype, low)
    offs = _i32(np.concatenate([[0], np.cumsum(news)]).tolist(), cuda)
    out, lse = paged.paged_attention(scree.Array(q, offs), cache, 0, slots, return_lse=True)
    ref = _reference(q, cache, 0, hs, news, news, _causal(news))
    assert np.isposinf(ref[0][low:news[0], 0, :2]).all() and np.isneginf(ref[0][low:news[0], 0, 2]).all()
    _compare(out.values, lse, ref)
    got = out.values.float().cpu().numpy()
    assert np.array_equal(np.isposinf(got), np.isposinf(ref[0])) and np.array_equal(np.isneginf(got), np.isneginf(ref[0]))
    assert _status() == 0


# --------------------------------------------------------------------------- writes


def _rows_cache(cuda, S, n=2, layers=1):
    """S slots of n tokens each; every pool element 7."""
    from scree_b200 import paged

    cache = paged.paged_cache(layers, S + 4, 4, 1, 8, S, 3, dtype=torch.float16, device=cuda)
    cache = paged.paged_reserve(cache, torch.arange(S, dtype=torch.int32, device=cuda),
                                torch.full((S,), n, dtype=torch.int32, device=cuda))
    cache.k.fill_(7)
    cache.v.fill_(7)
    return cache


def _held(cache, slot, n):
    return cache.k[0, cache.table[slot, 0].item(), 0, :n], cache.v[0, cache.table[slot, 0].item(), 0, :n]


@pytest.mark.parametrize("B", [3, 40, 300, 1024, 1500, 9000])
def test_write_refuses_a_slot_named_twice(cuda, B):
    """By any two entries that have tokens, wherever they stand; their rows stay as they were."""
    import scree_b200 as scree
    from scree_b200 import _lib, paged

    cache = _rows_cache(cuda, B)
    slots = np.random.default_rng(B).permutation(B)
    for a, b in ((0, B - 1), (B // 2, 0), (B - 1, B - 2)):
        cache.k.fill_(7)  # (entries that name a slot of their own are written)
        cache.v.fill_(7)
        news = np.ones(B, np.int64)
        news[b] = 2
        offs = _i32(np.concatenate([[0], np.cumsum(news)]).tolist(), cuda)
        named = slots.copy()
        named[a] = named[b]
        rows = torch.ones((int(news.sum()), 1, 8), dtype=torch.float16, device=cuda)
        paged.paged_write(cache, 0, _i32(named.tolist(), cuda), scree.Array(rows, offs), scree.Array(rows, offs))
        st = _lib.device_status()
        assert st >> 16 == _lib.DEVERR_BAD_INPUT and st & 0xFFFF == 60
        for pool in _held(cache, int(named[b]), 2):
            assert (pool == 7).all()
    assert _status() == 0


@pytest.mark.parametrize("B", [3, 300, 1500])
def test_write_takes_entries_without_tokens_whatever_they_name(cuda, B):
    """The places of a batch that are not in use may all name one slot."""
    import scree_b200 as scree
    from scree_b200 import paged

    cache = _rows_cache(cuda, B)
    news = np.zeros(B, np.int64)
    news[[0, B // 2]] = 1
    slots = np.full(B, 1)
    slots[0] = 2
    offs = torch.tensor(np.concatenate([[0], np.cumsum(news)]), device=cuda)
    rows = torch.arange(2 * 8, device=cuda).view(2, 1, 8).to(torch.float16)
    paged.paged_write(cache, 0, _i32(slots.tolist(), cuda), scree.Array(rows, offs), scree.Array(-rows, offs))
    for slot, t in ((2, 0), (1, 1)):
        k, v = _held(cache, slot, 2)
        assert torch.equal(k[1], rows[t, 0]) and torch.equal(v[1], -rows[t, 0]) and (k[0] == 7).all()
    assert (cache.k == 7).sum() == cache.k.numel() - 16 + 1 and _status() == 0  # (one new element is a 7)


@pytest.mark.parametrize("page,n", [(4, 8), (4, 10), (16, 16)])
def test_write_refuses_pages_that_other_slots_hold(cuda, page, n):
    """After a fork the shared pages are no slot's own: written over, the sibling's K / V would go."""
    import scree_b200 as scree
    from scree_b200 import _lib, paged

    cache = paged.paged_cache(2, 12, page, 2, 16, 4, 4, dtype=torch.bfloat16, device=cuda)
    one = _i32([1], cuda)
    cache = paged.paged_reserve(cache, one, _i32([n], cuda))
    gen = torch.Generator().manual_seed(n)
    rows = lambda m: scree.Array(torch.randn((m, 2, 16), generator=gen).to(torch.bfloat16).to(cuda), _i32([0, m], cuda))  # noqa: E731
    k, v = rows(n), rows(n)
    paged.paged_write(cache, 1, one, k, v)
    cache = paged.paged_fork(cache, one, _i32([3], cuda))
    assert _status() == 0
    before = cache.k.clone(), cache.v.clone()
    full = n // page * page
    for slot in (1, 3):
        k2, v2 = rows(n), rows(n)
        paged.paged_write(cache, 1, _i32([slot], cuda), k2, v2)
        st = _lib.device_status()
        assert st >> 16 == _lib.DEVERR_BAD_INPUT and st & 0xFFFF == 62
        ids = cache.table[1, :full // page].long()
        assert torch.equal(cache.k[:, ids], before[0][:, ids]) and torch.equal(cache.v[:, ids], before[1][:, ids])
    # What is behind them is a slot's own, and so are all pages once the sibling is gone.
    grown = paged.paged_reserve(cache, one, _i32([page], cuda))
    k3, v3 = rows(page), rows(page)
    paged.paged_write(grown, 1, one, k3, v3)
    at = [(grown.table[1, i // page].item(), i % page) for i in range(n, n + page)]
    assert _status() == 0 and all(torch.equal(grown.k[1, p, :, r], k3.values[i]) for i, (p, r) in enumerate(at))
    alone = paged.paged_free(grown, _i32([3], cuda))
    k4, v4 = rows(n + page), rows(n + page)
    paged.paged_write(alone, 0, one, k4, v4)
    at = [(alone.table[1, i // page].item(), i % page) for i in range(n + page)]
    assert _status() == 0 and all(torch.equal(alone.v[0, p, :, r], v4.values[i]) for i, (p, r) in enumerate(at))


def test_write_compares_the_offsets_of_k_and_v(cuda):
    """v's rows of a sequence are those of its own offsets: other ones than k's are refused."""
    import scree_b200 as scree
    from scree_b200 import _lib, paged

    cache = _rows_cache(cuda, 4, n=3)
    slots = _i32([2, 0, 3], cuda)
    rows = torch.arange(6 * 8, device=cuda).view(6, 1, 8).to(torch.float16)
    k = scree.Array(rows, _i32([0, 2, 3, 6], cuda))
    for offs in ([0, 1, 3, 6], [0, 2, 4, 6], [0, 2, 2, 6]):
        cache.k.fill_(7)
        cache.v.fill_(7)
        paged.paged_write(cache, 0, slots, k, scree.Array(rows, _i32(offs, cuda)))
        st = _lib.device_status()
        assert st >> 16 == _lib.DEVERR_BAD_INPUT and st & 0xFFFF == 60
        assert (cache.k == 7).all() and (cache.v == 7).all()
    with pytest.raises(ValueError, match="identical offsets"):
        paged.paged_write(cache, 0, slots, k, scree.Array(rows, _i32([0, 2, 6], cuda)))
    for same in (k.offsets.clone(), k.offsets.long(), k.offsets.cpu()):  # equal ones of another tensor
        cache.v.fill_(7)
        paged.paged_write(cache, 0, slots, k, scree.Array(rows, same))
        assert torch.equal(_held(cache, 3, 3)[1], rows[3:, 0]) and torch.equal(_held(cache, 0, 3)[1][2], rows[2, 0])
    assert _status() == 0


def test_arrays_must_be_ragged_in_their_tokens(cuda):
    """Offsets that count heads are not offsets of tokens, even where the numbers would do."""
    import scree_b200 as scree
    from scree_b200 import paged

    cache = paged.paged_cache(1, 4, 16, 2, 64, 1, 2, device=cuda)
    cache = paged.paged_reserve(cache, _i32([0], cuda), _i32([2], cuda))
    t = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device=cuda)
    offs = _i32([0, 2], cuda)
    heads, tokens = scree.Array(t, offs, ragged_dim=1), scree.Array(t, offs)
    for k, v in ((heads, tokens), (tokens, heads)):
        with pytest.raises(NotImplementedError, match="ragged_dim"):
            paged.paged_write(cache, 0, _i32([0], cuda), k, v)
    with pytest.raises(NotImplementedError, match="ragged_dim"):
        paged.paged_attention(heads, cache, 0, _i32([0], cuda))
    assert paged.paged_attention(tokens, cache, 0, _i32([0], cuda)).ragged_dim == 0 and _status() == 0


def test_offsets_below_zero_are_refused(cuda):
    """Offsets between the first and the last may be anything: nothing is read in front of the parents."""
    import scree_b200 as scree
    from scree_b200 import _lib, paged

    offs = _i32([0, -5, 3], cuda)

    def site():
        st = _lib.device_status()
        assert st >> 16 == _lib.DEVERR_BAD_INPUT
        return st & 0xFFFF

    mask = paged.tree_mask(scree.Array(_i32([2, 2, 2], cuda), offs), max_nodes=8)
    assert site() == 60 and (mask == 0).all()
    cache = _rows_cache(cuda, 2, n=10)
    rows = scree.Array(torch.ones((3, 1, 8), dtype=torch.float16, device=cuda), offs)
    paged.paged_write(cache, 0, _i32([0, 1], cuda), rows, rows)
    assert site() == 60 and (cache.k == 7).all()
    assert _status() == 0
