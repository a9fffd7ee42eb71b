"""The order of waits in the tensor-core kernel of attention over pages, on the CPU.

A wait on an mbarrier names the parity of a phase, so it also returns at once while the
phase before the one meant is still under way.  The softmax warps wait for the V tile of
their round (ring of kStages places) only where the tile is masked; so what they have seen
before must imply that the place's last fill, tile v - kStages, has landed.  The model
below holds the happens-before edges of one CTA: the V warp, the MMA thread and the two
softmax groups, as the kernel's source orders them.
"""

import itertools
import re
from pathlib import Path

import pytest

SOURCE = Path(__file__).resolve().parent.parent / "scree_b200" / "csrc" / "attn_paged_tc.cu"
kStages = 3


class Order:
    """Happens-before: nodes in an order of creation that respects every edge's use."""

    def __init__(self):
        self.edges = {}

    def after(self, node, *before):
        self.edges.setdefault(node, set()).update(b for b in before if b is not None)
        return node

    def reach(self, node):
        seen, todo = set(), [node]
        while todo:
            for b in self.edges.get(todo.pop(), ()):
                if b not in seen:
                    seen.add(b)
                    todo.append(b)
        return seen


def unsafe_waits(pieces, s_first):
    """pieces: (tiles of rows, tiles of keys).  (piece, group, tile) of every wait on V that may
    meet a place whose last fill is still under way."""
    o = Order()
    # Rounds of a piece: (group, round of the group, tile), as the MMA thread issues their products.
    plan, v = [], 0
    for rows, keys in pieces:
        if rows == 1 and keys >= 2:
            plan.append((v, keys, True, [(j & 1, j >> 1, v + j) for j in range(keys)]))
        else:
            plan.append((v, keys, False, [(x, j, v + j) for j in range(keys) for x in range(rows)]))
        v += keys
    for t in range(v):  # the V warp: a place is free when the products of its last tile are done
        o.after(("load", t), ("load", t - 1) if t else None, ("products", t - kStages) if t >= kStages else None)
        o.after(("landed", t), ("load", t))
    # The MMA thread: one chain of steps; what it issues completes in order.
    step, done = None, None

    def issue(node):
        nonlocal step, done
        step = o.after(("issue",) + node, step)
        done = o.after(("done",) + node, step, done)
        return done

    last_of = {}  # of a group: the end of its last piece
    for k, (v0, keys, split, rounds) in enumerate(plan):
        def s_of(x, r):
            issue(("S", k, x, r))

        def product(x, r, t):
            nonlocal step
            step = o.after(("free", k, x, r), step, last_of.get(x) if r == 0 else None)
            step = o.after(("P half", k, x, r), step, ("half", k, x, r))
            issue(("PV1", k, x, r))
            step = o.after(("P full", k, x, r), step, ("full", k, x, r))
            return issue(("PV2", k, x, r))

        def v_wait(t):
            nonlocal step
            step = o.after(("V seen", t), step, ("landed", t))

        if split:
            s_of(0, 0)
            s_of(1, 0)
            for j, (x, r, t) in enumerate(rounds):
                v_wait(t)
                o.after(("products", t), product(x, r, t))
                if j + 2 < keys:
                    s_of(x, r + 1)
        else:
            groups = sorted({x for x, _, _ in rounds})
            for x in groups:
                s_of(x, 0)
            for j in range(keys):
                v_wait(v0 + j)
                for x in groups:
                    end = product(x, j, v0 + j)
                    if j + 1 < keys:
                        s_of(x, j + 1)
                o.after(("products", v0 + j), end)
        # The softmax groups.  (Waits on V add no edges: few tiles are masked.)
        for x in (0, 1):
            at = last_of.get(x)
            at = o.after(("record", k, x), at)
            mine = [(r, t) for y, r, t in rounds if y == x]
            for r, t in mine:
                scores = ("done", "S", k, x, r)
                o.after(("V wait", k, x, t), at, scores if s_first else None)
                at = o.after(("scores", k, x, r), at, scores)
                if r > 0:
                    at = o.after(("product seen", k, x, r), at, ("done", "PV2", k, x, r - 1))
                at = o.after(("half", k, x, r), at)
                at = o.after(("full", k, x, r), at)
            if mine:
                at = o.after(("piece done", k, x), at, ("done", "PV2", k, x, mine[-1][0]))
            last_of[x] = at
        if split:  # A joins B's half and frees both accumulators
            last_of[0] = o.after(("joined", k), last_of[0], last_of[1])
    bad = []
    for node in [n for n in o.edges if n[0] == "V wait"]:
        t = node[3]
        if t >= kStages and ("landed", t - kStages) not in o.reach(node):
            bad.append(node[1:])
    return bad


def _kernel_waits_for_scores_first():
    text = SOURCE.read_text()
    start = text.index("- softmax\n")
    v = re.search(r"ok = wait\(&v_full\[st\], vpos", text[start:])
    s = re.search(r"ok = wait\(&s_full\[x\], sc \+ j\)", text[start:])
    assert v and s, "the kernel's waits have changed: bring the model in line"
    return s.start() < v.start()


PIECES = [(1, 1), (1, 2), (1, 3), (1, 7), (2, 1), (2, 2), (2, 5)]


@pytest.mark.parametrize("first", PIECES)
def test_waits_on_v_name_one_phase(first):
    s_first = _kernel_waits_for_scores_first()
    for rest in itertools.chain([()], itertools.product(PIECES, repeat=2), itertools.product([(1, 1), (1, 4), (2, 2)], repeat=4)):
        pieces = [first, *rest]
        assert unsafe_waits(pieces, s_first) == [], pieces


def test_the_model_sees_waits_that_are_too_early():
    """Without the scores in front, group B may test tile 3 while V of tile 0 is landing."""
    assert (0, 1, 3) in unsafe_waits([(1, 4)], s_first=False)
    assert unsafe_waits([(1, 1), (1, 1), (1, 1), (1, 2)], s_first=False)
    assert unsafe_waits([(2, 9)], s_first=False) == []
