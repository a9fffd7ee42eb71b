"""The paged K/V cache on the GPU: its bookkeeping and row moves against a plain
Python model (exact), and attention over it against a float64 evaluation of the
definition.

Attention bounds.  P is rounded to the 16-bit type (relative u16, and an absolute
2^-25 where fp16 is subnormal; the row sum is at least 1 in P's scale), O once more
(u16), and scores and exponentials are fp32 with an error far below 2^-13:
  |O - ref| <= (u16 + 2^-13) sum_j p_j |v_j| + 2^-25 sum_j |v_j| + u16 |O|
The LSE's error is that of a score: D u32 sum |q k| scale < 1e-4 for N(0, 1) inputs.
"""

import math
import random

import numpy as np
import pytest
import torch

from gpu_helpers import to64

pytestmark = pytest.mark.gpu

U16 = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def _status():
    from scree_b200 import _lib

    return _lib.device_status()


def _i32(x, cuda):
    return torch.tensor(x, dtype=torch.int32, device=cuda)


# --------------------------------------------------------------------------- bookkeeping


class Model:
    """The cache's rules on Python lists; rows are (slot writes) tagged by number."""

    def __init__(self, P, page, S, M):
        self.P, self.page, self.S, self.M = P, page, S, M
        self.table = [[] for _ in range(S)]
        self.len = [0] * S
        self.refs = [0] * P
        self.rows = {}  # (page, row) -> tag

    def take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def reserve(self, slots, counts):
        for s, c in zip(slots, counts):
            self.len[s] += c
            while len(self.table[s]) * self.page < self.len[s]:
                self.table[s].append(self.take())

    def at(self, s, pos):
        return self.table[s][pos // self.page], pos % self.page

    def write(self, s, tags):
        for i, t in enumerate(tags):
            self.rows[self.at(s, self.len[s] - len(tags) + i)] = t

    def drop(self, s, pages):
        for p in pages:
            self.refs[p] -= 1

    def accept(self, s, drafted, path):
        base = self.len[s] - drafted
        got = [self.rows[self.at(s, base + i)] for i in path]
        for d, t in enumerate(got):
            self.rows[self.at(s, base + d)] = t
        self.len[s] = base + len(path)
        keep = -(-self.len[s] // self.page)
        self.drop(s, self.table[s][keep:])
        del self.table[s][keep:]

    def fork(self, parents, children):
        shared = list(zip(parents, children))
        for p, c in shared:
            full, part = divmod(self.len[p], self.page)
            self.table[c] = self.table[p][:full]
            self.len[c] = self.len[p]
        fresh = {}
        free = [x for x in range(self.P) if self.refs[x] == 0]
        for p, c in shared:
            full, part = divmod(self.len[p], self.page)
            for x in self.table[p][:full]:
                self.refs[x] += 1
            if part:
                new = free.pop(0)
                fresh[c] = new
                self.refs[new] = 1
                for r in range(part):
                    self.rows[(new, r)] = self.rows[(self.table[p][full], r)]
                self.table[c].append(new)

    def free(self, slots):
        for s in slots:
            self.drop(s, self.table[s])
            self.table[s], self.len[s] = [], 0

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        holes = [p for p in range(used) if self.refs[p] == 0]
        move = dict(zip([p for p in range(used, self.P) if self.refs[p] > 0], holes))
        for a, b in move.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
            for r in range(self.page):
                if (a, r) in self.rows:
                    self.rows[(b, r)] = self.rows[(a, r)]
        self.table = [[move.get(p, p) for p in t] for t in self.table]

    def check(self, cache, new_rows):
        assert cache.lengths.tolist() == self.len
        assert cache.refs.tolist() == self.refs
        assert cache.table.tolist() == [t + [-1] * (self.M - len(t)) for t in self.table]
        pages, rows, tags = [], [], []
        for s in range(self.S):
            for pos in range(self.len[s]):
                p, r = self.at(s, pos)
                pages.append(p)
                rows.append(r)
                tags.append(self.rows[(p, r)])
        if not pages:
            return
        for layer in range(cache.k.shape[0]):
            for pool, src in ((cache.k, 0), (cache.v, 1)):
                got = pool[layer][pages, :, rows]
                want = torch.stack([new_rows[t][layer][src] for t in tags])
                assert torch.equal(got, want)


@pytest.mark.parametrize("seed,page,heads,dim,layers,dtype", [
    (0, 16, 2, 64, 2, torch.bfloat16), (1, 16, 3, 5, 1, torch.float16), (2, 4, 1, 1, 3, torch.float32),
    (3, 1, 2, 32, 1, torch.bfloat16), (4, 48, 4, 128, 2, torch.float16), (5, 7, 1, 3, 2, torch.int8)])
def test_random_operations_match_the_model(cuda, seed, page, heads, dim, layers, dtype):
    import scree_b200 as scree
    from scree_b200 import paged

    rng = random.Random(seed)
    S, M = 9, 12
    P = 60 if page > 1 else 90
    cache = paged.paged_cache(layers, P, page, heads, dim, S, M, dtype=dtype, device=cuda)
    model = Model(P, page, S, M)
    g = torch.Generator().manual_seed(seed)
    new_rows = []
    for step in range(60):
        live = [s for s in range(S) if model.len[s] > 0]
        empty = [s for s in range(S) if model.len[s] == 0]
        op = rng.choice(["append", "append", "draft", "draft", "fork", "free", "compact"])
        free_pages = sum(r == 0 for r in model.refs)
        if op in ("append", "draft"):
            slots = rng.sample(range(S), rng.randint(1, 4))
            counts = [rng.choice([0, 1, page, rng.randint(1, 2 * page + 3)]) for _ in slots]
            counts = [min(c, M * page - model.len[s]) for s, c in zip(slots, counts)]
            need = sum(-(-(model.len[s] + c) // page) - len(model.table[s]) for s, c in zip(slots, counts))
            if need > free_pages or sum(counts) == 0:
                continue
            cache = paged.paged_reserve(cache, _i32(slots, cuda), _i32(counts, cuda))
            model.reserve(slots, counts)
            T = sum(counts)
            kv = [[torch.randint(-99, 99, (T, heads, dim), generator=g).to(dtype).to(cuda) for _ in range(2)]
                  for _ in range(layers)]
            offs = _i32(np.concatenate([[0], np.cumsum(counts)]).tolist(), cuda)
            for layer, (k, v) in enumerate(kv):
                paged.paged_write(cache, layer, _i32(slots, cuda), scree.Array(k, offs), scree.Array(v, offs))
            at = 0
            for s, c in zip(slots, counts):
                tags = []
                for i in range(c):
                    tags.append(len(new_rows))
                    new_rows.append([(k[at + i], v[at + i]) for k, v in kv])
                model.write(s, tags)
                at += c
            if op == "draft":
                depth = rng.randint(1, 6)
                path = [sorted(rng.sample(range(c), rng.randint(0, min(c, depth)))) for c in counts]
                pad = [p + [-1] * (depth - len(p)) for p in path]
                cache = paged.paged_accept(cache, _i32(slots, cuda), _i32(counts, cuda), _i32(pad, cuda))
                for s, c, p in zip(slots, counts, path):
                    model.accept(s, c, p)
        elif op == "fork" and live and empty:
            children = rng.sample(empty, rng.randint(1, min(3, len(empty))))
            parents = [rng.choice(live) for _ in children]
            if len(children) > free_pages:
                continue
            cache = paged.paged_fork(cache, _i32(parents, cuda), _i32(children, cuda))
            model.fork(parents, children)
        elif op == "free":
            slots = rng.sample(range(S), rng.randint(0, 3))
            cache = paged.paged_free(cache, _i32(slots, cuda))
            model.free(slots)
        elif op == "compact":
            cache = paged.paged_compact(cache)
            model.compact()
        model.check(cache, new_rows)
    assert len(new_rows) > 20 and _status() == 0


def test_allocation_over_many_pages_and_slots(cuda):
    """More pages than one pass of the scan holds, and more entries than its threads."""
    from scree_b200 import paged

    S, P, page = 3000, 40001, 2
    g = np.random.default_rng(0)
    refs = (g.random(P) < 0.8).astype(np.int32) * 3
    cache = paged.PagedCache(k=torch.zeros((1, P, 1, page, 1), device=cuda), v=torch.zeros((1, P, 1, page, 1), device=cuda),
                             table=torch.full((S, 6), -1, dtype=torch.int32, device=cuda),
                             lengths=torch.zeros(S, dtype=torch.int32, device=cuda), refs=_i32(refs.tolist(), cuda))
    slots = g.permutation(S)[:2500]
    counts = g.integers(0, 7, 2500)
    out = paged.paged_reserve(cache, _i32(slots.tolist(), cuda), _i32(counts.tolist(), cuda))
    free = np.flatnonzero(refs == 0)
    table, at = np.full((S, 6), -1), 0
    for s, c in zip(slots, counts):
        n = -(-c // page)
        table[s, :n] = free[at:at + n]
        at += n
    assert np.array_equal(out.table.cpu().numpy(), table)
    refs[free[:at]] = 1
    assert np.array_equal(out.refs.cpu().numpy(), refs)
    back = paged.paged_free(out, _i32(slots.tolist(), cuda))
    assert torch.equal(back.refs, cache.refs) and torch.equal(back.table, cache.table)
    packed = paged.paged_compact(out).refs.cpu().numpy()
    used = (refs > 0).sum()
    assert (packed[:used] > 0).all() and (packed[used:] == 0).all() and sorted(packed[packed > 0]) == sorted(refs[refs > 0])
    assert _status() == 0


def test_rejected_calls_change_nothing(cuda):
    import scree_b200 as scree
    from scree_b200 import _lib, paged

    def site():
        st = _lib.device_status()
        assert st >> 16 in (0, _lib.DEVERR_BAD_INPUT)
        return st & 0xFFFF

    I = lambda *x: _i32(list(x), cuda)  # noqa: E731
    cache = paged.paged_cache(1, 6, 4, 1, 8, 4, 3, dtype=torch.float16, device=cuda)
    cache = paged.paged_reserve(cache, I(0, 1), I(6, 4))
    cache = paged.paged_fork(cache, I(0), I(2))  # page 0 of slot 0 shared; 2 pages left
    assert site() == 0
    cases = [
        (60, lambda: paged.paged_reserve(cache, I(0, 0), I(1, 1))),       # a slot twice
        (60, lambda: paged.paged_reserve(cache, I(4), I(1))),             # no such slot
        (60, lambda: paged.paged_reserve(cache, I(-1), I(1))),
        (60, lambda: paged.paged_reserve(cache, I(0), I(-1))),
        (60, lambda: paged.paged_reserve(cache, I(0), I(7))),             # its table row is too short
        (61, lambda: paged.paged_reserve(cache, I(1, 3), I(8, 8))),       # 4 pages wanted, 2 free
        (60, lambda: paged.paged_fork(cache, I(0), I(1))),                # child in use
        (60, lambda: paged.paged_fork(cache, I(3), I(3))),                # child its own parent
        (60, lambda: paged.paged_fork(cache, I(0, 0), I(3, 3))),
        (60, lambda: paged.paged_fork(cache, I(9), I(3))),
        (60, lambda: paged.paged_free(cache, I(0, 5))),
        (60, lambda: paged.paged_free(cache, I(1, 1))),
        (60, lambda: paged.paged_accept(cache, I(1), I(5), I(0).view(1, 1))),  # more drafted than held
        (60, lambda: paged.paged_accept(cache, I(1), I(3), I(1, 1).view(1, 2))),  # not ascending
        (60, lambda: paged.paged_accept(cache, I(1), I(3), I(0, 3).view(1, 2))),  # not in the draft
        (62, lambda: paged.paged_accept(cache, I(0), I(4), I(0).view(1, 1))),  # on a shared page
    ]
    k0 = cache.k.clone()
    for want, call in cases:
        out = call()
        torch.cuda.synchronize()
        for a, b in ((out.table, cache.table), (out.lengths, cache.lengths), (out.refs, cache.refs), (out.k, k0)):
            assert torch.equal(a, b)
        assert site() == want
    # While the status word holds an error, nothing is done.
    paged.paged_reserve(cache, I(9), I(1))
    out = paged.paged_reserve(cache, I(1), I(1))
    assert torch.equal(out.lengths, cache.lengths) and torch.equal(out.refs, cache.refs)
    assert site() == 60
    # A write of more rows than the slot holds.
    rows = torch.ones((5, 1, 8), dtype=torch.float16, device=cuda)
    paged.paged_write(cache, 0, I(1), scree.Array(rows, I(0, 5)), scree.Array(rows, I(0, 5)))
    assert site() == 60
    with pytest.raises(TypeError, match="int32"):
        paged.paged_free(cache, I(0).long())
    with pytest.raises(ValueError, match="1-D"):
        paged.paged_reserve(cache, I(0, 1), I(1))
    with pytest.raises(ValueError, match="entries for 4 slots"):
        paged.paged_free(cache, I(0, 1, 2, 3, 3))
    with pytest.raises(ValueError, match="path"):
        paged.paged_accept(cache, I(0), I(1), I(0))
    with pytest.raises(ValueError, match="layer 1 of 1"):
        paged.paged_write(cache, 1, I(1), scree.Array(rows[:1], I(0, 1)), scree.Array(rows[:1], I(0, 1)))
    with pytest.raises(ValueError, match="k and v must be"):
        paged.paged_write(cache, 0, I(1), scree.Array(rows[:1, :, :4], I(0, 1)), scree.Array(rows[:1, :, :4], I(0, 1)))
    with pytest.raises(ValueError, match="contiguous int32"):
        paged.PagedCache(k=cache.k, v=cache.v, table=cache.table.long(), lengths=cache.lengths, refs=cache.refs)
    assert _status() == 0


def test_write_from_strided_views(cuda):
    """K / V as views of a fused (T, 3, H, D) projection, and of a buffer at an odd offset."""
    import scree_b200 as scree
    from scree_b200 import paged

    for dim, shift in ((64, 0), (64, 1), (5, 0)):
        cache = paged.paged_cache(2, 8, 16, 3, dim, 2, 4, dtype=torch.bfloat16, device=cuda)
        slots, counts = _i32([1, 0], cuda), _i32([20, 3], cuda)
        cache = paged.paged_reserve(cache, slots, counts)
        buf = torch.randn((23 * 3 * 3 * dim + 1,), device=cuda).to(torch.bfloat16)
        qkv = buf[shift:shift + 23 * 9 * dim].view(23, 3, 3, dim)
        offs = torch.tensor([0, 20, 23], dtype=torch.int64, device=cuda)
        paged.paged_write(cache, 1, slots, scree.Array(qkv[:, 1], offs), scree.Array(qkv[:, 2], offs))
        for pool, i in ((cache.k, 1), (cache.v, 2)):
            got1 = pool[1, cache.table[1, :2].long()].transpose(1, 2).reshape(32, 3, dim)[:20]
            assert torch.equal(got1, qkv[:20, i])
            assert torch.equal(pool[1, cache.table[0, 0].item()].transpose(0, 1)[:3], qkv[20:, i])
            assert (pool[0] == 0).all()
    assert _status() == 0


# --------------------------------------------------------------------------- tree masks


@pytest.mark.parametrize("sizes", [[1], [5, 0, 64, 1], [65, 200, 3], [33] * 40])
def test_tree_mask(cuda, sizes):
    import scree_b200 as scree
    from scree_b200 import paged

    rng = random.Random(len(sizes))
    parents = [rng.choice([-1, rng.randint(0, i - 1)]) if i else -1 for n in sizes for i in range(n)]
    offs = np.concatenate([[0], np.cumsum(sizes)])
    got = paged.tree_mask(scree.Array(_i32(parents, cuda), _i32(offs.tolist(), cuda))).cpu().numpy().view(np.uint64)
    assert got.shape[1] == max(1, -(-max(sizes) // 64))
    for b, n in enumerate(sizes):
        for i in range(n):
            seen, j = set(), i
            while j >= 0:
                seen.add(j)
                j = parents[offs[b] + j]
            row = got[offs[b] + i]
            assert {j for j in range(64 * len(row)) if int(row[j // 64]) >> (j % 64) & 1} == seen
    assert _status() == 0


def test_tree_mask_refuses_bad_trees(cuda):
    import scree_b200 as scree
    from scree_b200 import paged

    offs = _i32([0, 3], cuda)
    paged.tree_mask(scree.Array(_i32([-1, 1, 0], cuda), offs))  # its own parent
    assert _status() & 0xFFFF == 60
    paged.tree_mask(scree.Array(_i32([-1] * 70, cuda), _i32([0, 70], cuda)), max_nodes=64)
    assert _status() & 0xFFFF == 60
    with pytest.raises(TypeError, match="int32"):
        paged.tree_mask(scree.Array(torch.zeros(3, dtype=torch.int64, device=cuda), offs))


# --------------------------------------------------------------------------- attention


def _make(cuda, lens, page, hkv, D, dtype, seed, layers=1, spare=3, extra_slots=2):
    """A cache with the sequences in shuffled slots and pages; everything that no sequence
    holds (free pages, rows past a sequence's end) is NaN."""
    from scree_b200 import paged

    g = np.random.default_rng(seed)
    used = [-(-n // page) for n in lens]
    P, S = sum(used) + spare, len(lens) + extra_slots
    perm = g.permutation(P)
    slots = g.permutation(S)[:len(lens)]
    table = np.full((S, max(used + [1]) + 1), -1, np.int32)
    lengths, refs = np.zeros(S, np.int32), np.zeros(P, np.int32)
    gen = torch.Generator().manual_seed(seed)
    k = torch.full((layers, P, hkv, page, D), float("nan"), dtype=dtype)
    v = k.clone()
    at = 0
    for s, n, u in zip(slots, lens, used):
        ids = perm[at:at + u]
        at += u
        table[s, :u], lengths[s], refs[ids] = ids, n, 1
        for pool in (k, v):
            rows = torch.full((layers, u * page, hkv, D), float("nan"))
            rows[:, :n] = torch.randn((layers, n, hkv, D), generator=gen)
            pool[:, ids] = rows.view(layers, u, page, hkv, D).transpose(2, 3).to(dtype)
    t = lambda x: _i32(x.tolist(), cuda)  # noqa: E731
    cache = paged.PagedCache(k=k.to(cuda), v=v.to(cuda), table=t(table), lengths=t(lengths), refs=t(refs))
    return cache, t(slots), slots


def _rows(cache, pool, layer, slot, n):
    page = cache.k.shape[3]
    ids = cache.table[slot, :-(-n // page)].long()
    return to64(pool[layer, ids].transpose(1, 2).reshape(-1, *[pool.shape[2], pool.shape[4]])[:n])


def _reference(q, cache, layer, slots, lens, news, see):
    """see(b, i) -> booleans over the new tokens.  Returns O, LSE and the bound on |O - ref|."""
    qn = to64(q)
    T, H, D = qn.shape
    G = H // cache.k.shape[2]
    u = U16[q.dtype]
    out, lse, tol = np.zeros_like(qn), np.full((T, H), -np.inf), np.zeros_like(qn)
    at = 0
    for b, (L, n) in enumerate(zip(lens, news)):
        if n == 0:
            continue
        K, V = _rows(cache, cache.k, layer, slots[b], L), _rows(cache, cache.v, layer, slots[b], L)
        for i in range(n):
            vis = np.ones(L, bool)
            vis[L - n:] = see(b, i)
            for h in range(H):
                if not vis.any():
                    continue
                s = K[vis, h // G] @ qn[at + i, h] / math.sqrt(D)
                m = s.max()
                e = np.exp(s - m)
                Vv = V[vis, h // G]
                with np.errstate(invalid="ignore"):
                    out[at + i, h] = (e / e.sum()) @ Vv
                    tol[at + i, h] = (u + 2.0**-13) * (e / e.sum()) @ np.abs(Vv) + 2.0**-25 * np.abs(Vv).sum(0)
                lse[at + i, h] = m + np.log(e.sum())
        at += n
    return out, lse, tol + u * np.abs(out)


def _compare(got, lse, ref):
    out, rl, tol = ref
    g = to64(got)
    same = (g == out) | (np.isnan(g) & np.isnan(out))
    with np.errstate(invalid="ignore"):
        assert (same | (np.abs(g - out) <= tol)).all(), np.nanmax(np.where(same, 0, np.abs(g - out) - tol))
    gl = to64(lse)
    fin = np.isfinite(rl)
    assert np.array_equal(gl[~fin], rl[~fin]) and (np.abs(gl[fin] - rl[fin]) <= 1e-4).all()


def _causal(news):
    return lambda b, i: np.arange(news[b]) <= i


def _tree(news, rng):
    par = [[-1 if i == 0 else rng.randint(max(0, i - 6), i - 1) for i in range(n)] for n in news]

    def see(b, i):
        v = np.zeros(news[b], bool)
        while i >= 0:
            v[i] = True
            i = par[b][i]
        return v

    return [p for row in par for p in row], see


# (context, new) per sequence
SHAPES = {
    "one_token": [(0, 1), (1, 1), (15, 1), (16, 1), (700, 1)],
    "one_sequence": [(1234, 1)],
    "two_tokens": [(31, 2), (0, 2), (95, 2)],
    "empty_between": [(40, 0), (33, 3), (0, 0), (5, 1)],
    "chunk": [(0, 37), (100, 21), (7, 64)],
    "wide": [(50, 130), (300, 65), (0, 1)],
    "many": [(i * 7 % 90, 1 + i % 3) for i in range(70)],
    "one_tile_of_rows": [(500, 20), (129, 31), (0, 20), (1000, 17)],
    "uneven": [(400, 90), (3, 1), (250, 40), (0, 1), (777, 33)],
}


@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("D,H,Hkv,page,dtype", [
    (128, 8, 2, 16, torch.bfloat16), (64, 3, 3, 64, torch.float16), (32, 14, 2, 48, torch.bfloat16),
    (128, 3, 1, 128, torch.float16), (64, 20, 1, 16, torch.bfloat16), (128, 4, 4, 32, torch.bfloat16),
    (32, 130, 1, 16, torch.float16)])
@pytest.mark.parametrize("tree", [False, True])
def test_attention(cuda, shape, D, H, Hkv, page, dtype, tree):
    import scree_b200 as scree
    from scree_b200 import paged

    ctx, news = zip(*SHAPES[shape])
    lens = [a + b for a, b in zip(ctx, news)]
    cache, slots, hs = _make(cuda, lens, page, Hkv, D, dtype, seed=D + H)
    g = torch.Generator().manual_seed(7)
    T = sum(news)
    q = torch.randn((T, H, D), generator=g).to(dtype).to(cuda)
    offs = _i32(np.concatenate([[0], np.cumsum(news)]).tolist(), cuda)
    mask, see = None, _causal(news)
    if tree:
        parents, see = _tree(news, random.Random(1))
        mask = paged.tree_mask(scree.Array(_i32(parents, cuda), offs))
    out, lse = paged.paged_attention(scree.Array(q, offs), cache, 0, slots, mask=mask, return_lse=True)
    again = paged.paged_attention(scree.Array(q, offs.long()), cache, 0, slots, mask=mask)
    _compare(out.values, lse, _reference(q, cache, 0, hs, lens, news, see))
    assert torch.equal(out.values, again.values)
    assert _status() == 0


def test_attention_long_context_split_over_the_gpu(cuda):
    import scree_b200 as scree
    from scree_b200 import paged

    lens, news = [40003, 17, 9000], [1, 1, 1]
    cache, slots, hs = _make(cuda, lens, 32, 2, 64, torch.bfloat16, seed=3, layers=2)
    q = torch.randn((3, 8, 64), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(cuda)
    offs = _i32([0, 1, 2, 3], cuda)
    out, lse = paged.paged_attention(scree.Array(q, offs), cache, 1, slots, return_lse=True)
    _compare(out.values, lse, _reference(q, cache, 1, hs, lens, news, _causal(news)))
    assert _status() == 0


@pytest.mark.parametrize("D,H,Hkv", [(128, 4, 2), (64, 40, 1), (128, 2, 2), (32, 6, 3)])
@pytest.mark.parametrize("before", [21, 380])
def test_rows_that_see_nothing_and_masked_specials(cuda, D, H, Hkv, before):
    """Masks that leave rows empty; infinities and NaN in K and V of drafted tokens reach
    exactly the rows that see them."""
    import scree_b200 as scree
    from scree_b200 import paged

    news, ctx = [5, 20, 3], [0, before, 0]
    lens = [a + b for a, b in zip(ctx, news)]
    cache, slots, hs = _make(cuda, lens, 16, Hkv, D, torch.float16, seed=11)
    rng = np.random.default_rng(0)
    vis = [rng.random((n, n)) < 0.5 for n in news]
    vis[0][2] = False                      # no context and no visible node
    vis[2][:] = False
    vis[2][1, 0] = True
    for a, bad in ((1, 4), (1, 9), (0, 3)):  # nodes seen by few
        vis[a][:, bad] = False
        vis[a][bad, bad] = True
    vis[1][6, 9] = True

    def put(pool, b, node, value, cols):
        pos = ctx[b] + node
        pool[0, cache.table[int(hs[b]), pos // 16].item(), :, pos % 16, cols] = value

    put(cache.v, 1, 4, float("nan"), slice(3, 9))
    put(cache.v, 1, 9, float("inf"), slice(0, 2))
    put(cache.v, 0, 3, float("-inf"), slice(D - 1, D))
    bits = np.zeros((sum(news), 1), np.int64)
    at = 0
    for b, n in enumerate(news):
        for i in range(n):
            bits[at + i, 0] = int(sum(1 << j for j in range(n) if vis[b][i, j]))
        at += n
    q = torch.randn((sum(news), H, D), generator=torch.Generator().manual_seed(2)).to(torch.float16).to(cuda)
    offs = _i32(np.concatenate([[0], np.cumsum(news)]).tolist(), cuda)
    run = lambda: paged.paged_attention(scree.Array(q, offs), cache, 0, slots,  # noqa: E731
                                        mask=torch.tensor(bits, device=cuda), return_lse=True)
    see = lambda b, i: vis[b][i]  # noqa: E731
    out, lse = run()
    ref = _reference(q, cache, 0, hs, lens, news, see)
    _compare(out.values, lse, ref)
    assert (out.values[2] == 0).all() and torch.isneginf(lse[2]).all()
    nan_rows = np.isnan(to64(out.values)).any((1, 2))
    assert nan_rows[5 + 4] and not nan_rows[[5 + i for i in range(20) if i != 4]].any()
    # K of a node that only it sees: NaN scores elsewhere stay out.
    put(cache.v, 1, 4, 1.0, slice(0, D))
    put(cache.v, 1, 9, 1.0, slice(0, D))
    put(cache.v, 0, 3, 1.0, slice(0, D))
    put(cache.k, 1, 4, float("nan"), slice(0, D))
    out, lse = run()
    rows = np.isnan(to64(out.values)).any((1, 2))
    assert rows.nonzero()[0].tolist() == [5 + 4] and torch.isnan(lse[5 + 4]).all()
    assert _status() == 0


def test_attention_on_views_and_another_stream(cuda):
    import scree_b200 as scree
    from scree_b200 import paged

    lens, news = [300, 41], [2, 1]
    cache, slots, hs = _make(cuda, lens, 16, 2, 64, torch.bfloat16, seed=5)
    qkv = torch.randn((3, 3, 4, 64), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda)
    offs = _i32([0, 2, 3], cuda)
    want = paged.paged_attention(scree.Array(qkv[:, 0].contiguous(), offs), cache, 0, slots)
    odd = torch.empty(3 * 4 * 64 + 1, dtype=torch.bfloat16, device=cuda)[1:].view(3, 4, 64).copy_(qkv[:, 0])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a = paged.paged_attention(scree.Array(qkv[:, 0], offs), cache, 0, slots)
        b = paged.paged_attention(scree.Array(odd, offs), cache, 0, slots)
    side.synchronize()
    assert torch.equal(a.values, want.values) and torch.equal(b.values, want.values)
    assert a.offsets is offs and _status() == 0


def test_offsets_past_32_bits(cuda):
    """Pools of more than 2^32 elements; the sequence lives in their last pages."""
    import scree_b200 as scree
    from scree_b200 import paged

    P, page, H, D = 2**21 + 64, 16, 1, 128
    if torch.cuda.mem_get_info()[0] < 40 * 2**30:
        pytest.skip("needs 40 GB")
    k = torch.empty((1, P, H, page, D), dtype=torch.bfloat16, device=cuda)
    v = torch.empty_like(k)
    refs = torch.ones(P, dtype=torch.int32, device=cuda)
    refs[-9:] = 0
    cache = paged.PagedCache(k=k, v=v, table=torch.full((2, 8), -1, dtype=torch.int32, device=cuda),
                             lengths=torch.zeros(2, dtype=torch.int32, device=cuda), refs=refs)
    slots, n = _i32([1], cuda), 100
    cache = paged.paged_reserve(cache, slots, _i32([n], cuda))
    assert cache.table[1, 0].item() == P - 9
    kv = torch.randn((n, 2, H, D), generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(cuda)
    offs = _i32([0, n], cuda)
    paged.paged_write(cache, 0, slots, scree.Array(kv[:, 0], offs), scree.Array(kv[:, 1], offs))
    cache = paged.paged_fork(cache, slots, _i32([0], cuda))
    q = torch.randn((1, 2, D), generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).to(cuda)
    for s in (0, 1):
        out, lse = paged.paged_attention(scree.Array(q, _i32([0, 1], cuda)), cache, 0, _i32([s], cuda), return_lse=True)
        _compare(out.values, lse, _reference(q, cache, 0, [s], [n], [1], _causal([1])))
    assert _status() == 0


def test_prompt_in_chunks_equals_the_prompt_at_once(cuda):
    """Causal attention of a long prompt, cached in chunks, against varlen self-attention."""
    import scree_b200 as scree
    from scree_b200 import paged
    from scree_b200.kernels.native import varlen_attention_triton

    n, H, Hkv, D = 1500, 4, 2, 64
    q, k, v = (torch.randn((n, h, D), generator=torch.Generator().manual_seed(h + i)).to(torch.bfloat16).to(cuda)
               for i, h in enumerate((H, Hkv, Hkv)))
    cache = paged.paged_cache(1, 100, 16, Hkv, D, 2, 100, device=cuda)
    slots, got, at = _i32([1], cuda), [], 0
    for size in (700, 1, 300, 499):
        cache = paged.paged_reserve(cache, slots, _i32([size], cuda))
        a = lambda t: scree.Array(t[at:at + size], _i32([0, size], cuda))  # noqa: B023, E731
        paged.paged_write(cache, 0, slots, a(k), a(v))
        got.append(paged.paged_attention(a(q), cache, 0, slots).values)
        at += size
    want = varlen_attention_triton(q, k, v, _i32([0, n], cuda), causal=True)
    # each within half an ulp of its own P and O roundings of the same definition
    torch.testing.assert_close(torch.cat(got).float(), want.float(), atol=2e-2, rtol=2.0**-7)
    assert _status() == 0


def test_graph_capture_of_a_decoding_step(cuda):
    import scree_b200 as scree
    from scree_b200 import paged
    from scree_b200.kernels.native import token_logprobs

    cache, slots, hs = _make(cuda, [300, 41], 16, 2, 64, torch.bfloat16, seed=5)
    q = scree.Array(torch.randn((2, 4, 64), device=cuda).to(torch.bfloat16), _i32([0, 1, 2], cuda))
    kv = scree.Array(torch.randn((2, 2, 64), device=cuda).to(torch.bfloat16), _i32([0, 1, 2], cuda))
    one = _i32([1, 1], cuda)
    head = torch.randn((4 * 64, 3000), device=cuda).to(torch.bfloat16)
    given = torch.tensor([5, 2999], device=cuda)

    def run():
        c = paged.paged_reserve(cache, slots, one)
        paged.paged_write(c, 0, slots, kv, kv)
        out = paged.paged_attention(q, c, 0, slots).values
        s = token_logprobs(out.view(2, -1) @ head, given, top_k=3)
        return c.table, c.lengths, c.refs, out, s.logp, s.entropy, s.top_logp, s.top_ids

    want = [t.clone() for t in run()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert _status() == 0


def test_speculative_decoding_example(cuda):
    """The example's drafted trees give the tokens of plain greedy decoding, up to the few
    places where two logits lie within rounding of one another, in fewer steps."""
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parent.parent / "examples" / "speculative_decoding.py"
    spec = importlib.util.spec_from_file_location("speculative_decoding", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    plain, fast, steps, cache = mod.main(cuda, new_tokens=16)
    # A near tie may send one sequence another way from there on; the others must agree.
    assert sum(p == f for p, f in zip(plain, fast)) >= len(plain) - 1
    assert steps < 16
    assert cache.lengths.tolist()[0] == cache.lengths.tolist()[1] == cache.lengths.tolist()[2] > 0
    used = int((cache.refs > 0).sum())
    assert (cache.refs[:used] > 0).all() and (cache.refs[used:] == 0).all() and _status() == 0


def test_attention_refusals(cuda):
    import scree_b200 as scree
    from scree_b200 import _lib, paged

    cache, slots, _ = _make(cuda, [40, 9], 16, 2, 64, torch.bfloat16, seed=6)
    q = torch.zeros((3, 4, 64), dtype=torch.bfloat16, device=cuda)
    offs = _i32([0, 2, 3], cuda)
    A = lambda t=q, o=offs: scree.Array(t, o)  # noqa: E731

    def site(call):
        call()
        st = _lib.device_status()
        assert st >> 16 == _lib.DEVERR_BAD_INPUT
        return st & 0xFFFF

    call = lambda **k: paged.paged_attention(k.get("q", A()), k.get("c", cache), 0, k.get("s", slots), mask=k.get("m"))  # noqa: E731
    assert site(lambda: call(s=_i32([0, 7], cuda))) == 70
    assert site(lambda: call(s=_i32([-1, 0], cuda))) == 70
    many = torch.zeros((70, 4, 64), dtype=torch.bfloat16, device=cuda)
    assert site(lambda: call(q=A(many, _i32([0, 41, 70], cuda)))) == 70  # more queries than tokens
    assert site(lambda: call(q=A(q, _i32([0, 4, 3], cuda)))) == 70       # offsets that go back
    big = paged.PagedCache(k=cache.k, v=cache.v, table=cache.table, refs=cache.refs,
                           lengths=torch.full_like(cache.lengths, 10**6))
    assert site(lambda: call(c=big)) == 70                                # more tokens than a table row
    holes = paged.PagedCache(k=cache.k, v=cache.v, table=torch.full_like(cache.table, -1), refs=cache.refs,
                             lengths=cache.lengths)
    assert site(lambda: call(c=holes)) == 71                              # a page id out of range
    wide, wslots, _ = _make(cuda, [80], 16, 2, 64, torch.bfloat16, seed=6)
    narrow = torch.zeros((70, 1), dtype=torch.int64, device=cuda)
    assert site(lambda: paged.paged_attention(A(many, _i32([0, 70], cuda)), wide, 0, wslots, mask=narrow)) == 70
    with pytest.raises(AssertionError, match="fp16 or bf16"):
        call(q=A(q.float()))
    with pytest.raises(AssertionError, match="dtype"):
        call(q=A(q.half()))
    with pytest.raises(AssertionError, match="multiple"):
        call(q=A(q[:, :3]))
    with pytest.raises(ValueError, match="2 entries"):
        call(s=slots[:1])
    with pytest.raises(TypeError, match="int64"):
        call(m=torch.zeros((3, 1), dtype=torch.int32, device=cuda))
    with pytest.raises(ValueError, match="mask must be"):
        call(m=torch.zeros((2, 1), dtype=torch.int64, device=cuda))
    with pytest.raises(ValueError, match="layer 1 of 1"):
        paged.paged_attention(A(), cache, 1, slots)
    small = paged.paged_cache(1, 4, 8, 2, 64, 2, 2, device=cuda)
    with pytest.raises(ValueError, match="multiple of 16"):
        call(c=small)
    odd = paged.paged_cache(1, 4, 16, 2, 96, 2, 2, device=cuda)
    with pytest.raises(NotImplementedError, match="head_dim 96"):
        paged.paged_attention(A(torch.zeros((3, 4, 96), dtype=torch.bfloat16, device=cuda)), odd, 0, slots)
    empty = call(q=A(q[:0], _i32([0, 0, 0], cuda)))
    assert empty.values.shape == (0, 4, 64) and _status() == 0


def test_attention_of_many_rows_on_views(cuda):
    """Queries as views: of a fused projection, heads first, one row for all tokens, a misaligned base."""
    import scree_b200 as scree
    from scree_b200 import paged

    lens, news = [300, 141], [45, 35]
    cache, slots, _ = _make(cuda, lens, 16, 2, 64, torch.bfloat16, seed=8)
    T, H, D = sum(news), 8, 64
    gen = torch.Generator().manual_seed(9)
    qkv = torch.randn((T, 3, H, D), generator=gen).to(torch.bfloat16).to(cuda)
    offs = _i32([0, 45, 80], cuda)
    call = lambda q: paged.paged_attention(scree.Array(q, offs), cache, 0, slots).values  # noqa: E731
    q = qkv[:, 1].contiguous()
    want = call(q)
    _compare(want, paged.paged_attention(scree.Array(q, offs), cache, 0, slots, return_lse=True)[1],
             _reference(q, cache, 0, slots.tolist(), lens, news, _causal(news)))
    assert torch.equal(call(qkv[:, 1]), want)
    assert torch.equal(call(q.transpose(0, 1).contiguous().transpose(0, 1)), want)
    odd = torch.empty(q.numel() + 1, dtype=torch.bfloat16, device=cuda)[1:].view(T, H, D).copy_(q)
    assert torch.equal(call(odd), want)
    assert torch.equal(call(q[:1].expand(T, H, D)), call(q[:1].repeat(T, 1, 1)))
    assert torch.equal(call(q[:, :1].expand(T, H, D)), call(q[:, :1].repeat(1, H, 1)))
    assert _status() == 0


def test_offsets_past_32_bits_many_rows(cuda):
    """As above for queries that take the tensor-core kernel, and an accept in the pools' last pages."""
    import scree_b200 as scree
    from scree_b200 import paged

    P, page, H, D = 2**21 + 64, 16, 1, 128
    if torch.cuda.mem_get_info()[0] < 40 * 2**30:
        pytest.skip("needs 40 GB")
    k = torch.empty((1, P, H, page, D), dtype=torch.bfloat16, device=cuda)
    v = torch.empty_like(k)
    refs = torch.ones(P, dtype=torch.int32, device=cuda)
    refs[-9:] = 0
    cache = paged.PagedCache(k=k, v=v, table=torch.full((1, 8), -1, dtype=torch.int32, device=cuda),
                             lengths=torch.zeros(1, dtype=torch.int32, device=cuda), refs=refs)
    slots, n, m = _i32([0], cuda), 100, 40
    cache = paged.paged_reserve(cache, slots, _i32([n], cuda))
    assert cache.table[0, 0].item() == P - 9
    gen = torch.Generator().manual_seed(4)
    kv = torch.randn((n, 2, H, D), generator=gen).to(torch.bfloat16).to(cuda)
    offs = _i32([0, n], cuda)
    paged.paged_write(cache, 0, slots, scree.Array(kv[:, 0], offs), scree.Array(kv[:, 1], offs))
    q = torch.randn((m, 2, D), generator=gen).to(torch.bfloat16).to(cuda)
    out, lse = paged.paged_attention(scree.Array(q, _i32([0, m], cuda)), cache, 0, slots, return_lse=True)
    _compare(out.values, lse, _reference(q, cache, 0, [0], [n], [m], _causal([m])))
    path = [1, 5, 6, 30, 39]
    cache = paged.paged_accept(cache, slots, _i32([m], cuda), torch.tensor([path], dtype=torch.int32, device=cuda))
    rows = _rows(cache, cache.k, 0, 0, n - m + len(path))
    assert np.array_equal(rows[n - m:, 0], to64(kv[[n - m + j for j in path], 0, 0]))
    assert cache.lengths.item() == n - m + len(path) and _status() == 0


def test_attention_refuses_a_scale_that_is_not_positive(cuda):
    from scree_b200 import _lib

    cache, slots, _ = _make(cuda, [40], 16, 2, 64, torch.bfloat16, seed=6)
    q = torch.zeros((1, 4, 64), dtype=torch.bfloat16, device=cuda)
    offs, out, lib = _i32([0, 1], cuda), torch.empty_like(q), _lib.load()
    S, M, P, page, H, D = cache._pools.sizes
    ws = torch.empty(lib.scree_attn_fwd_paged_workspace_size(1, 1, 4, 2, 64), dtype=torch.uint8, device=cuda)
    for scale in (0.0, -1.0, float("nan")):
        rc = lib.scree_attn_fwd_paged(
            q.data_ptr(), 256, 64, cache._pools.ref, 0, cache.table.data_ptr(), cache.lengths.data_ptr(), S, M, P, page,
            slots.data_ptr(), offs.data_ptr(), 0, 1, 1, 4, 64, _lib.BF16, scale, None, 0, out.data_ptr(), 256, 64, None,
            ws.data_ptr(), ws.numel(), _lib.stream_ptr(q.device))
        with pytest.raises(ValueError, match="scale"):
            _lib.check(rc, "paged_attention")
