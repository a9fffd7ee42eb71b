"""The serving and scoring operators as a user's program calls them, and their plain forms.

Four kinds of case:

  attention  scores of new tokens (one each, or a tree of drafted tokens) against a paged K/V cache
  step       one speculative step of the cache: reserve room for the drafted tokens, write their
             K/V in every layer, keep the accepted path, give the rest back
  relocate   fork running sequences into siblings, free finished ones, compact the pool
  score      log probabilities of given tokens, entropies and top alternatives, with the gradient
             of the logits where the case trains

With ``own`` false everything below is elementary torch in 32 bits; with ``own`` true the calls are
the framework's own.  The cache operators return new bookkeeping tensors and update the pools in
place, so a pass repeats the same work on the same state.
"""

import math

import numpy as np
import torch

own = False

_DT = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


# ----------------------------------------------------------------------------------------- cases


def listed():
    return [
        # One conversation, one new token: the smallest call of a decoding loop.
        {"name": "decode_one", "op": "attention", "dtype": "bfloat16", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "seqs": 1, "mean": 640, "sigma": 0.0, "nodes": 1, "tree": False, "lse": False},
        # A full decoding batch with the length spread of the training benchmark's sequences.
        {"name": "decode_batch", "op": "attention", "dtype": "bfloat16", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "seqs": 64, "mean": 2048, "sigma": 0.6, "nodes": 1, "tree": False, "lse": False},
        # Two very long documents, few K/V heads: the work has to be split along the cache.
        {"name": "decode_long", "op": "attention", "dtype": "float16", "heads": 16, "kv_heads": 2, "dim": 64,
         "page": 64, "seqs": 2, "mean": 131071, "sigma": 0.3, "nodes": 1, "tree": False, "lse": True},
        # Verification of drafted trees for a serving batch.
        {"name": "verify_tree", "op": "attention", "dtype": "bfloat16", "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 32, "seqs": 16, "mean": 4096, "sigma": 0.6, "nodes": 61, "tree": True, "lse": False},
        # One drafted chain of a single conversation accepted in part.
        {"name": "step_one", "op": "step", "dtype": "bfloat16", "kv_heads": 8, "dim": 128, "page": 16, "layers": 2,
         "seqs": 1, "mean": 300, "sigma": 0.0, "nodes": 6, "depth": 4},
        # The same for a batch with full trees.
        {"name": "step_batch", "op": "step", "dtype": "bfloat16", "kv_heads": 8, "dim": 128, "page": 16, "layers": 4,
         "seqs": 64, "mean": 1024, "sigma": 0.6, "nodes": 64, "depth": 9},
        # Two samples drawn from one prompt.
        {"name": "relocate_small", "op": "relocate", "dtype": "float16", "kv_heads": 4, "dim": 64, "page": 32,
         "layers": 2, "seqs": 4, "mean": 200, "sigma": 0.4, "forks": 2, "freed": 1},
        # A busy server: samples forked, a quarter of the requests finished, the pool shrunk.
        {"name": "relocate_batch", "op": "relocate", "dtype": "bfloat16", "kv_heads": 8, "dim": 128, "page": 16,
         "layers": 4, "seqs": 64, "mean": 1024, "sigma": 0.6, "forks": 48, "freed": 16},
        # One decoded token with its alternatives.
        {"name": "score_one", "op": "score", "dtype": "bfloat16", "rows": 1, "vocab": 131072, "top": 20, "train": False},
        # A prompt scored with alternatives; an odd vocabulary, so rows start at any alignment.
        {"name": "score_prompt", "op": "score", "dtype": "bfloat16", "rows": 4099, "vocab": 65539, "top": 8,
         "train": False},
        # A small policy update in 32 bits.
        {"name": "train_small", "op": "score", "dtype": "float32", "rows": 119, "vocab": 32000, "top": 0, "train": True},
        # A batch of packed sequences of a policy update with an entropy bonus.
        {"name": "train_batch", "op": "score", "dtype": "bfloat16", "rows": 6144, "vocab": 128000, "top": 4,
         "train": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "step", "relocate", "score", "score"])
    dtype = rng.choice(["bfloat16", "float16"])
    if op == "attention":
        dim = rng.choice([32, 64, 128])
        kv = rng.choice([1, 2, 3, 4, 8])
        group = rng.choice([1, 2, 3, 4, 7, 8])
        tree = rng.random() < 0.6
        seqs = _log_int(rng, 1, 64)
        nodes = _log_int(rng, 2, 130) if tree else rng.choice([1, 1, 2, 5])
        # Bound tokens of cache (the keys read) and score elements by those of the largest listed case.
        mean = _log_int(rng, 1, 100000)
        mean = max(1, min(mean, 260000 // (seqs * 2)))
        mean = max(1, min(mean, int(2.0e9 / (seqs * nodes * kv * group * dim)) * 6))
        return {"op": op, "dtype": dtype, "heads": kv * group, "kv_heads": kv, "dim": dim,
                "page": rng.choice([16, 32, 64, 128]), "seqs": seqs, "mean": mean,
                "sigma": round(rng.uniform(0.0, 0.8), 2), "nodes": nodes, "tree": tree, "lse": rng.random() < 0.5}
    if op in ("step", "relocate"):
        seqs = _log_int(rng, 2, 64)
        case = {"op": op, "dtype": rng.choice(["bfloat16", "float16", "float32"]), "kv_heads": rng.choice([1, 2, 3, 8]),
                "dim": rng.choice([32, 64, 128]), "page": rng.choice([16, 32, 64]), "layers": rng.randint(1, 4),
                "seqs": seqs, "mean": _log_int(rng, 3, 700), "sigma": round(rng.uniform(0.0, 0.6), 2)}
        if op == "step":
            nodes = _log_int(rng, 1, 64)
            case.update(nodes=nodes, depth=rng.randint(1, min(nodes, 12)))
        else:
            case.update(forks=rng.randint(1, max(1, seqs * 3 // 4)), freed=rng.randint(0, seqs // 3))
        return case
    vocab = _log_int(rng, 500, 200000)
    rows = _log_int(rng, 1, min(8192, max(2, 300_000_000 // vocab)))
    return {"op": op, "dtype": rng.choice(["bfloat16", "float16", "float32"]), "rows": rows, "vocab": vocab,
            "top": rng.choice([0, 1, 5, 20, 32]), "train": rng.random() < 0.5}


def _lengths(case):
    """Tokens already cached per sequence: log-normal around the mean, the same for every seed."""
    rng = np.random.default_rng(1000 + case["seqs"])
    raw = rng.lognormal(math.log(case["mean"]), case["sigma"], case["seqs"])
    return [int(x) for x in np.clip(np.round(raw), 0 if case["sigma"] > 0 else 1, 3 * case["mean"])]


def _nodes(case):
    """New tokens per sequence: the full tree, or a smaller one where drafting stopped early."""
    rng = np.random.default_rng(2000 + case["seqs"])
    n = case["nodes"]
    if case["op"] == "attention" and not case["tree"]:
        return [n] * case["seqs"]
    return [n if b % 2 == 0 else int(rng.integers(max(1, n // 2), n + 1)) for b in range(case["seqs"])]


# ----------------------------------------------------------------------------------------- inputs


def _parents(rng, n):
    """A drafted tree: each node hangs under an earlier one, node 0 is the root."""
    return [-1] + [int(rng.integers(max(0, i - 8), i)) for i in range(1, n)]


def _cache_tables(case, lens, spare_slots, spare_pages, rng):
    """A fragmented page table: pages handed out in random order, spare ones in between."""
    pg = case["page"]
    used = [-(-n // pg) for n in lens]
    slots = len(lens) + spare_slots
    pages = sum(used) + spare_pages
    perm = rng.permutation(pages)
    width = max(used) + 2 + -(-case.get("nodes", 1) // pg)
    table = np.full((slots, width), -1, np.int32)
    refs = np.zeros(pages, np.int32)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = perm[at:at + u]
        refs[perm[at:at + u]] = 1
        at += u
    lengths = np.zeros(slots, np.int32)
    lengths[:len(lens)] = lens
    return table, lengths, refs, pages


def _pools(case, pages, layers, gen):
    shape = (layers, pages, case["kv_heads"], case["page"], case["dim"])
    k, v = (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(_DT[case["dtype"]])
            for _ in range(2))
    return k, v


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    op = case["op"]
    if op == "score":
        n, v = case["rows"], case["vocab"]
        dt = _DT[case["dtype"]]
        s["logits"] = torch.empty((n, v), dtype=dt, device="cuda")
        for r in range(0, n, 1024):
            part = s["logits"][r:r + 1024]
            part.copy_(torch.randn(part.shape, generator=gen, device="cuda") * 3.0)
        # Tokens of a vocabulary's padding are masked out, as samplers do.
        s["logits"][:, v - v // 64:] = -math.inf
        targets = torch.randint(0, v - v // 64, (n,), generator=gen, device="cuda")
        if n > 4:
            targets[::17] = -100  # prompt positions that do not count
        s["targets"] = targets
        if case["train"]:
            s["g_logp"] = torch.randn(n, generator=gen, device="cuda")
            s["g_entropy"] = torch.randn(n, generator=gen, device="cuda") * 0.01
            s["g_top"] = torch.randn((n, case["top"]), generator=gen, device="cuda") * 0.1
        return s

    lens = _lengths(case)
    if op == "attention":
        nodes = _nodes(case)
        # The new tokens' K/V are in the cache already when attention runs.
        table, lengths, refs, pages = _cache_tables(case, [a + b for a, b in zip(lens, nodes)], 1, 3, rng)
        T = sum(nodes)
        offs = np.concatenate([[0], np.cumsum(nodes)])
        s["host"] = (offs.tolist(), [a + b for a, b in zip(lens, nodes)])
        s["q"] = torch.randn((T, case["heads"], case["dim"]), generator=gen, device="cuda").to(_DT[case["dtype"]])
        s["layer"] = 0
        if case["tree"]:
            s["parents"] = _i32([p for n in nodes for p in _parents(rng, n)])
        s["offsets"] = _i32(offs)
        k, v = _pools(case, pages, 1, gen)
    elif op == "step":
        nodes = _nodes(case)
        grow = sum(-(-n // case["page"]) + 1 for n in nodes)
        table, lengths, refs, pages = _cache_tables(case, lens, 2, grow, rng)
        offs = np.concatenate([[0], np.cumsum(nodes)])
        T = int(offs[-1])
        k, v = _pools(case, pages, case["layers"], gen)
        s["new"] = [tuple(torch.randn((T, case["kv_heads"], case["dim"]), generator=gen, device="cuda")
                          .to(_DT[case["dtype"]]) for _ in range(2)) for _ in range(case["layers"])]
        path = np.full((len(nodes), case["depth"]), -1, np.int32)
        for b, n in enumerate(nodes):
            m = int(rng.integers(1, min(n, case["depth"]) + 1))
            path[b, :m] = np.sort(rng.choice(n, size=m, replace=False))
        s["offsets"], s["counts"], s["path"] = _i32(offs), _i32(nodes), _i32(path)
        s["host"] = offs.tolist()
    else:
        table, lengths, refs, pages = _cache_tables(case, lens, case["forks"], case["forks"] + 8, rng)
        k, v = _pools(case, pages, case["layers"], gen)
        order = rng.permutation(case["seqs"])
        live = order[case["freed"]:]
        s["freed"] = _i32(order[:case["freed"]])
        s["parents"] = _i32(live[rng.integers(0, len(live), case["forks"])])
        s["children"] = _i32(np.arange(case["seqs"], case["seqs"] + case["forks"]))
    s["k"], s["v"] = k, v
    s["table"], s["lengths"], s["refs"] = _i32(table), _i32(lengths), _i32(refs)
    s["slots"] = torch.arange(case["seqs"], dtype=torch.int32, device="cuda")
    if own:
        import scree_b200 as scree
        from scree_b200 import paged

        s["cache"] = paged.PagedCache(k=k, v=v, table=s["table"], lengths=s["lengths"], refs=s["refs"])
        if op == "attention":
            s["q_array"] = scree.Array(values=s["q"], offsets=s["offsets"])
            if case["tree"]:
                # Made once per step of a model, before its layers.
                s["mask"] = paged.tree_mask(scree.Array(values=s["parents"], offsets=s["offsets"]))
        elif op == "step":
            s["new_arrays"] = [tuple(scree.Array(values=t, offsets=s["offsets"]) for t in kv) for kv in s["new"]]
    return s


# ----------------------------------------------------------------------------------------- one pass


def run(state):
    op = state["case"]["op"]
    if op == "attention":
        return (_own_attention if own else _plain_attention)(state)
    if op == "step":
        return (_own_step if own else _plain_step)(state)
    if op == "relocate":
        return (_own_relocate if own else _plain_relocate)(state)
    return (_own_score if own else _plain_score)(state)


def _own_attention(s):
    from scree_b200 import paged

    out = paged.paged_attention(s["q_array"], s["cache"], s["layer"], s["slots"], mask=s.get("mask"),
                                return_lse=s["case"]["lse"])
    return {"out": out[0].values, "lse": out[1]} if s["case"]["lse"] else {"out": out.values}


def _own_step(s):
    from scree_b200 import paged

    cache = paged.paged_reserve(s["cache"], s["slots"], s["counts"])
    for layer, (k, v) in enumerate(s["new_arrays"]):
        paged.paged_write(cache, layer, s["slots"], k, v)
    cache = paged.paged_accept(cache, s["slots"], s["counts"], s["path"])
    return {"k": cache.k, "v": cache.v, "table": cache.table, "lengths": cache.lengths, "refs": cache.refs}


def _own_relocate(s):
    from scree_b200 import paged

    cache = paged.paged_fork(s["cache"], s["parents"], s["children"])
    cache = paged.paged_free(cache, s["freed"])
    cache = paged.paged_compact(cache)
    return {"k": cache.k, "v": cache.v, "table": cache.table, "lengths": cache.lengths, "refs": cache.refs}


def _own_score(s):
    from scree_b200.kernels import native

    if not s["case"]["train"]:
        r = native.token_logprobs(s["logits"], s["targets"], top_k=s["case"]["top"])
        return {"logp": r.logp, "entropy": r.entropy, "top_logp": r.top_logp, "top_ids": r.top_ids}
    logits = s["logits"].detach().requires_grad_(True)
    r = native.token_logprobs_autograd(logits, s["targets"], top_k=s["case"]["top"])
    outs, grads = [r.logp, r.entropy], [s["g_logp"], s["g_entropy"]]
    if s["case"]["top"]:
        outs.append(r.top_logp)
        grads.append(s["g_top"])
    torch.autograd.backward(outs, grads)
    return {"logp": r.logp.detach(), "entropy": r.entropy.detach(), "top_logp": r.top_logp.detach(),
            "top_ids": r.top_ids, "d_logits": logits.grad}


def _ancestors(parents, offs):
    """Per sequence the (n, n) truth table "j is i or an ancestor of i"."""
    out = []
    for b in range(len(offs) - 1):
        par = parents[offs[b]:offs[b + 1]].long()
        n = par.numel()
        up = torch.zeros((n, n), dtype=torch.float32, device=par.device)
        up[torch.arange(n, device=par.device), par.clamp(min=0)] = (par >= 0).float()
        seen = torch.eye(n, device=par.device) + up
        steps = 1
        while steps < n:
            seen = (seen @ seen).clamp(max=1)
            steps *= 2
        out.append(seen > 0)
    return out


def _plain_attention(s):
    case = s["case"]
    offs, lens = s["host"]
    pg, hk, D = case["page"], case["kv_heads"], case["dim"]
    g = case["heads"] // hk
    q, out = s["q"], torch.empty_like(s["q"])
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    masks = _ancestors(s["parents"], offs) if case["tree"] else None
    kp, vp = s["k"][s["layer"]], s["v"][s["layer"]]
    for b, L in enumerate(lens):
        n = offs[b + 1] - offs[b]
        pages = s["table"][b, :-(-L // pg)].long()
        k = kp[pages].transpose(0, 1).reshape(hk, -1, D)[:, :L].float()
        v = vp[pages].transpose(0, 1).reshape(hk, -1, D)[:, :L].float()
        x = q[offs[b]:offs[b + 1]].float().reshape(n, hk, g, D).permute(1, 2, 0, 3)
        sc = x @ k[:, None].transpose(-1, -2) / math.sqrt(D)
        tree = masks[b] if masks else torch.ones((n, n), device=q.device).tril() > 0
        sc[..., L - n:] = torch.where(tree, sc[..., L - n:], -math.inf)
        m = sc.amax(-1, keepdim=True)
        e = (sc - m).exp()
        l = e.sum(-1, keepdim=True)
        o = (e @ v[:, None]) / l
        out[offs[b]:offs[b + 1]] = o.permute(2, 0, 1, 3).reshape(n, -1, D).to(q.dtype)
        lse[offs[b]:offs[b + 1]] = (m + l.log())[..., 0].permute(2, 0, 1).reshape(n, -1)
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


def _plain_step(s):
    case, pg = s["case"], s["case"]["page"]
    slots, counts = s["slots"].long(), s["counts"]
    k, v = s["k"], s["v"]
    # Reserve: the lowest free pages, in the order of the batch.
    before = s["lengths"][slots]
    after = before + counts
    first, last = (before + pg - 1) // pg, (after + pg - 1) // pg
    need = last - first
    start = torch.cumsum(need, 0) - need
    free = torch.argsort((s["refs"] > 0).int(), stable=True)
    cols = torch.arange(s["table"].shape[1], device=k.device)
    fresh = (cols >= first[:, None]) & (cols < last[:, None])
    pick = free[(start[:, None] + cols - first[:, None]).clamp(0, free.numel() - 1)].int()
    table, lengths, refs = s["table"].clone(), s["lengths"].clone(), s["refs"].clone()
    table[slots] = torch.where(fresh, pick, table[slots])
    lengths[slots] = after
    ranks = torch.arange(free.numel(), device=k.device)
    refs[free] = torch.where(ranks < need.sum(), 1, refs[free])
    # Write every layer's rows.
    seq = torch.repeat_interleave(torch.arange(slots.numel(), device=k.device), counts,
                                  output_size=s["host"][-1])
    pos = before[seq] + torch.arange(seq.numel(), device=k.device) - s["offsets"][seq]
    page, row = table[slots[seq], pos // pg].long(), pos % pg
    for layer, (nk, nv) in enumerate(s["new"]):
        k[layer][page, :, row] = nk
        v[layer][page, :, row] = nv
    # Accept: rows of the path move up, the pages behind them are given back.
    path = s["path"]
    b, d = (path >= 0).nonzero(as_tuple=True)
    src, dst = before[b] + path[b, d], before[b] + d
    sp, sr = table[slots[b], src // pg].long(), (src % pg).long()
    dp, dr = table[slots[b], dst // pg].long(), (dst % pg).long()
    for pool in (k, v):
        pool[:, dp, :, dr] = pool[:, sp, :, sr].clone()
    kept = before + (path >= 0).sum(1, dtype=torch.int32)
    gone = (cols >= ((kept + pg - 1) // pg)[:, None]) & (cols < last[:, None])
    refs.index_add_(0, table[slots][gone].long(), torch.full((int(gone.sum()),), -1, dtype=torch.int32, device=k.device))
    table[slots] = torch.where(gone, -1, table[slots])
    lengths[slots] = kept
    return {"k": k, "v": v, "table": table, "lengths": lengths, "refs": refs}


def _plain_relocate(s):
    pg = s["case"]["page"]
    k, v = s["k"], s["v"]
    parents, children, freed = s["parents"].long(), s["children"].long(), s["freed"].long()
    table, lengths, refs = s["table"].clone(), s["lengths"].clone(), s["refs"].clone()
    cols = torch.arange(table.shape[1], device=k.device)
    # Fork: whole pages are shared, the rows of a part-filled one copied.
    n = lengths[parents]
    full, part = n // pg, n % pg
    rows = table[parents]
    shared = rows[cols < full[:, None]].long()
    refs.index_add_(0, shared, torch.ones_like(shared, dtype=torch.int32))
    need = (part > 0).int()
    free = torch.argsort((s["refs"] > 0).int(), stable=True)
    fresh = free[torch.cumsum(need, 0) - need]
    has = (part > 0).nonzero(as_tuple=True)[0]
    old, new = rows[has, full[has].long()].long(), fresh[has]
    keep = torch.arange(pg, device=k.device) < part[has, None]
    for pool in (k, v):
        pool[:, new] = torch.where(keep[None, :, None, :, None], pool[:, old], pool[:, new])
    rows[has, full[has].long()] = new.int()
    table[children] = rows
    lengths[children] = n
    refs[new] = 1
    # Free.
    held = table[freed][cols < ((lengths[freed] + pg - 1) // pg)[:, None]].long()
    refs.index_add_(0, held, torch.full_like(held, -1, dtype=torch.int32))
    table[freed] = -1
    lengths[freed] = 0
    # Compact: the used pages above the count of used pages fill the holes below it, in order.
    used = refs > 0
    ids = torch.arange(refs.numel(), device=k.device)
    below = ids < used.sum()
    src, dst = (used & ~below).nonzero(as_tuple=True)[0], (~used & below).nonzero(as_tuple=True)[0]
    for pool in (k, v):
        pool[:, dst] = pool[:, src]
    to = ids.int()
    to[src] = dst.int()
    table = torch.where(table >= 0, to[table.clamp(min=0).long()], -1)
    refs[dst] = refs[src]
    refs[src] = 0
    return {"k": k, "v": v, "table": table, "lengths": lengths, "refs": refs}


def _plain_score(s):
    case = s["case"]
    x_all, t_all, top = s["logits"], s["targets"], case["top"]
    n, V = x_all.shape
    dev = x_all.device
    r = {"logp": torch.empty(n, device=dev), "entropy": torch.empty(n, device=dev),
         "top_logp": torch.empty((n, top), device=dev),
         "top_ids": torch.empty((n, top), dtype=torch.int64, device=dev)}
    if case["train"]:
        r["d_logits"] = torch.empty_like(x_all)
    ids = torch.arange(V, device=dev)
    step = max(1, (1 << 27) // V)
    for a in range(0, n, step):
        rows = slice(a, min(n, a + step))
        x, t = x_all[rows].float() + 0.0, t_all[rows]
        m = x.amax(-1, keepdim=True)
        e = (x - m).exp()
        z = e.sum(-1, keepdim=True)
        lse = m + z.log()
        logp = x - lse
        p = e / z
        H = -torch.where(p > 0, p * logp, 0.0).sum(-1, keepdim=True)
        given = t >= 0
        r["logp"][rows] = torch.where(given, logp.gather(1, t.clamp(min=0)[:, None])[:, 0], 0.0)
        r["entropy"][rows] = H[:, 0]
        if top:
            # Order by value, then by lower index: both in one whole number.
            bits = x.view(torch.int32).long()
            key = torch.where(bits < 0, ~bits & 0xFFFFFFFF, bits | 0x80000000) * (1 << 30) + (V - 1 - ids)
            best = V - 1 - (key.topk(top, dim=1).values & ((1 << 30) - 1))
            del bits, key
            r["top_ids"][rows] = best
            r["top_logp"][rows] = logp.gather(1, best)
        if case["train"]:
            g = torch.where(given, s["g_logp"][rows], 0.0)[:, None]
            gh, gt = s["g_entropy"][rows][:, None], s["g_top"][rows]
            d = -p * (g + gt.sum(1, keepdim=True)) - gh * torch.where(p > 0, p * (logp + H), 0.0)
            d.scatter_add_(1, t.clamp(min=0)[:, None], g)
            if top:
                d.scatter_add_(1, best, gt)
            r["d_logits"][rows] = d.to(x_all.dtype)
    return r


# ----------------------------------------------------------------------------------------- work


def work(case):
    op = case["op"]
    if op == "score":
        size = {"float32": 4}.get(case["dtype"], 2)
        n, V, k = case["rows"], case["vocab"], case["top"]
        passes = 2 if case["train"] else 1  # logits in, and their gradient out
        return {"bytes": passes * n * V * size + n * (8 + 4 + 4 + 12 * k), "flops": (12 if case["train"] else 6) * n * V}
    size = {"float32": 4}.get(case["dtype"], 2)
    lens = _lengths(case)
    row = 2 * case["kv_heads"] * case["dim"] * size  # K and V of one token in one layer
    if op == "attention":
        nodes = _nodes(case)
        keys = sum(lens) + sum(nodes)
        q = sum(nodes) * case["heads"] * case["dim"]
        # Every node sees its context and at least itself.
        pairs = sum(n * (c + 1) for n, c in zip(nodes, lens))
        return {"bytes": keys * row + 2 * q * size + 4 * keys // case["page"],
                "flops": 4 * case["heads"] * case["dim"] * pairs}
    if op == "step":
        nodes = _nodes(case)
        moved = sum((min(n, case["depth"]) + 1) / 2 for n in nodes)  # the mean of the path's length
        pages = sum(-(-c // case["page"]) for c in lens)
        return {"bytes": int(2 * (sum(nodes) + moved) * row * case["layers"]) + 12 * pages, "flops": sum(nodes)}
    pg = case["page"]
    per = np.array([-(-c // pg) for c in lens], float)
    held, spare = per.sum(), case["forks"] + 8
    gone = case["freed"] * per.mean()
    part = np.mean([c % pg for c in lens]) * case["forks"]
    left = held - gone + case["forks"]
    # Pages stand in random order, so the part above the end of the used ones is used as densely as the rest.
    moved = left * (1 - left / (held + spare)) if left < held + spare else 0
    return {"bytes": int(2 * (part + moved * pg) * row * case["layers"] + 12 * held), "flops": int(held)}


# ----------------------------------------------------------------------------------------- in 64 bits


def exact(case, seed):
    """The definitions in 64 bits, one sequence, page or row at a time."""
    s = prepare(case, seed)
    op = case["op"]
    if op == "attention":
        return _exact_attention(s)
    if op == "step":
        return _exact_step(s)
    if op == "relocate":
        return _exact_relocate(s)
    return _exact_score(s)


def _exact_attention(s):
    case = s["case"]
    offs, lens = s["host"]
    H, hk, D, pg = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    parents = s["parents"].tolist() if case["tree"] else None
    table = s["table"].tolist()
    for b, L in enumerate(lens):
        lo, n = offs[b], offs[b + 1] - offs[b]
        seen = np.zeros((n, L), bool)
        seen[:, :L - n] = True
        for i in range(n):
            j = i
            while j >= 0:
                seen[i, L - n + j] = True
                j = parents[lo + j] if parents else j - 1
        hide = ~torch.tensor(seen, device="cuda")
        pages = torch.tensor(table[b][:(L - 1) // pg + 1], device="cuda")
        for h in range(hk):
            K = s["k"][0, pages, h].reshape(-1, D)[:L].double()
            V = s["v"][0, pages, h].reshape(-1, D)[:L].double()
            for qh in range(h * (H // hk), (h + 1) * (H // hk)):
                z = (s["q"][lo:lo + n, qh].double() @ K.T).mul_(D ** -0.5).masked_fill_(hide, -math.inf)
                lse[lo:lo + n, qh] = torch.logsumexp(z, 1)
                out[lo:lo + n, qh] = torch.exp(z - lse[lo:lo + n, qh, None]) @ V
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


def _exact_step(s):
    case, pg = s["case"], s["case"]["page"]
    table, lengths, refs = s["table"].tolist(), s["lengths"].tolist(), s["refs"].tolist()
    k, v = s["k"], s["v"]
    free = iter([p for p, r in enumerate(refs) if r == 0])
    offs = s["host"]
    for b, path in enumerate(s["path"].tolist()):
        base, n = lengths[b], offs[b + 1] - offs[b]
        for c in range(-(-base // pg), -(-(base + n) // pg)):
            table[b][c] = next(free)
            refs[table[b][c]] = 1
    for b, path in enumerate(s["path"].tolist()):
        base, n = lengths[b], offs[b + 1] - offs[b]
        pages = torch.tensor([table[b][(base + i) // pg] for i in range(n)], device="cuda")
        at = torch.tensor([(base + i) % pg for i in range(n)], device="cuda")
        accepted = [i for i in path if i >= 0]
        rows = accepted + list(range(len(accepted), n))  # what each row holds in the end
        pick = torch.tensor([offs[b] + i for i in rows], device="cuda")
        for layer, (nk, nv) in enumerate(s["new"]):
            k[layer, pages, :, at] = nk[pick]
            v[layer, pages, :, at] = nv[pick]
        end = base + len(accepted)
        for c in range(-(-end // pg), -(-(base + n) // pg)):
            refs[table[b][c]] = 0
            table[b][c] = -1
        lengths[b] = end
    return {"k": k, "v": v, "table": _i32(table), "lengths": _i32(lengths), "refs": _i32(refs)}


def _exact_relocate(s):
    pg = s["case"]["page"]
    table, lengths, refs = s["table"].tolist(), s["lengths"].tolist(), s["refs"].tolist()
    k, v = s["k"], s["v"]
    free = [p for p, r in enumerate(refs) if r == 0]
    for p, c in zip(s["parents"].tolist(), s["children"].tolist()):
        n = lengths[p]
        table[c], lengths[c] = list(table[p]), n
        for j in range(n // pg):
            refs[table[p][j]] += 1
        if n % pg:
            new, old = free.pop(0), table[p][n // pg]
            k[:, new, :, :n % pg] = k[:, old, :, :n % pg]
            v[:, new, :, :n % pg] = v[:, old, :, :n % pg]
            table[c][n // pg] = new
            refs[new] = 1
    for f in s["freed"].tolist():
        for j in range(-(-lengths[f] // pg)):
            refs[table[f][j]] -= 1
        table[f], lengths[f] = [-1] * len(table[f]), 0
    used = sum(r > 0 for r in refs)
    holes = [p for p in range(used) if refs[p] == 0]
    move = dict(zip([p for p in range(used, len(refs)) if refs[p] > 0], holes))
    for a, b in move.items():
        k[:, b], v[:, b] = k[:, a], v[:, a]
        refs[b], refs[a] = refs[a], 0
    table = [[move.get(p, p) for p in row] for row in table]
    return {"k": k, "v": v, "table": _i32(table), "lengths": _i32(lengths), "refs": _i32(refs)}


def _exact_score(s):
    case = s["case"]
    x_all, top = s["logits"], case["top"]
    n, V = x_all.shape
    r = {"logp": torch.zeros(n, dtype=torch.float64, device="cuda"),
         "entropy": torch.zeros(n, dtype=torch.float64, device="cuda"),
         "top_logp": torch.zeros((n, top), dtype=torch.float64, device="cuda"),
         "top_ids": torch.zeros((n, top), dtype=torch.int64, device="cuda")}
    if case["train"]:
        r["d_logits"] = torch.empty((n, V), dtype=torch.float64, device="cuda")
    step = max(1, (1 << 26) // V)
    for a in range(0, n, step):
        z = x_all[a:a + step].double()
        t = s["targets"][a:a + step]
        lp = z - torch.logsumexp(z, 1, keepdim=True)
        p = lp.exp()
        plp = p * lp.clamp(min=-1e4)
        H = -plp.sum(1)
        at = torch.arange(len(t), device="cuda")
        r["logp"][a:a + step] = torch.where(t >= 0, lp[at, t.clamp(min=0)], 0.0)
        r["entropy"][a:a + step] = H
        if top:
            order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top]
            r["top_ids"][a:a + step] = order
            r["top_logp"][a:a + step] = lp.gather(1, order)
        if case["train"]:
            one = torch.zeros_like(p)
            one[at, t.clamp(min=0)] = (t >= 0).double() * s["g_logp"][a:a + step].double()
            if top:
                one.scatter_add_(1, order, s["g_top"][a:a + step].double())
            gh = s["g_entropy"][a:a + step].double()[:, None]
            r["d_logits"][a:a + step] = one - p * one.sum(1, keepdim=True) - gh * (plp + p * H[:, None])
    return r
