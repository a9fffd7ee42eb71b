"""Token log probabilities, entropies, top alternatives and the logits' gradient
on the GPU, against their definitions in float64 on the same inputs.

Bounds.  The kernels work in fp32 (u = 2^-24) with ex2 of relative error 2^-22 and at
most 64 sequential adds per partial sum, so s1 has relative error below 2^-17 and
  |lse - ref|  <= 2^-17 + 4 u |lse| + 4 u |m|          (m = the row's maximum)
  |logp - ref| <= that + u |x_t|
  |H - ref|    <= 2^-16 (1 + E[m - x])                 (s2 / s1 has the same relative error)
The gradient's p has relative error r = 2^-17 + 8 u (|x| + |lse|) ln 2, and is multiplied by
(gs + gH (H + log p)); then comes half an ulp of the logits' type.
"""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
HALF_ULP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def _status():
    from scree_b200 import _lib

    return _lib.device_status()


def _ref(x, t, k):
    """x (N, V) float64 on any device, t (N,) -> logp, H, lse, top ids (definition, NaN first)."""
    m = x.amax(1)
    empty = m == -np.inf
    rest = torch.logsumexp(x - m[:, None], 1)  # apart from m: it may be too large to add to in 64 bits
    lse = m + rest
    lp = (x - m[:, None]) - rest[:, None]
    lp[empty] = -np.inf
    p = torch.where(empty[:, None], torch.zeros_like(lp), lp.exp())
    H = -torch.where(p == 0, torch.zeros_like(p), p * lp).sum(1)
    got = lp.gather(1, t.clamp(min=0)[:, None])[:, 0]
    logp = torch.where(t < 0, torch.zeros_like(got), got)
    key = torch.where(x.isnan(), torch.full_like(x, np.inf), x)
    # stable sorts: by value, then NaN in front
    order = torch.sort(key, dim=1, descending=True, stable=True).indices
    if x.isnan().any():
        nan_first = torch.sort(x.gather(1, order).isnan().int(), dim=1, descending=True, stable=True).indices
        order = order.gather(1, nan_first)
    ids = order[:, :k]
    return logp, H, lse, ids, lp.gather(1, ids), p, lp


def _check(x, t, k, got, double):
    logp, H, lse, ids, tlp, p, _ = _ref(double, t.long(), k)
    m = double.amax(1)
    fin = torch.isfinite(lse)
    big = 2.0**-17 + 4 * U * (lse.abs() + m.abs())
    dist = torch.where(p > 0, p * (m[:, None] - double).clamp(max=1e30), torch.zeros_like(p)).sum(1)

    def near(a, b, tol):
        a = a.double()
        same = (a == b) | (a.isnan() & b.isnan())
        bad = ~same & ~((a - b).abs() <= tol)
        assert not bad.any(), (a[bad][:4], b[bad][:4])

    xt = double.gather(1, t.long().clamp(min=0)[:, None])[:, 0].abs()
    near(got.logp[fin], logp[fin], (big + U * torch.where(torch.isfinite(xt), xt, torch.zeros_like(xt)))[fin])
    near(got.entropy[fin], H[fin], (2.0**-16 * (1 + dist))[fin])
    assert torch.equal(got.top_ids, ids)
    near(got.top_logp[fin], tlp[fin], (big[:, None] + U * torch.where(torch.isfinite(tlp), tlp.abs(), torch.zeros_like(tlp)))[fin])
    return fin


def _logits(N, V, dtype, cuda, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((N, V), generator=g) * scale).to(dtype).to(cuda), torch.randint(0, V, (N,), generator=g).to(cuda)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,V,k", [(1, 1, 1), (3, 2, 2), (5, 7, 3), (2, 255, 32), (4, 4097, 20), (3, 16384, 5),
                                   (2, 16385, 1), (2, 50257, 8), (1, 131072, 32), (2, 262147, 20), (700, 33, 0)])
def test_forward(cuda, dtype, N, V, k):
    from scree_b200.kernels.native import token_logprobs

    x, t = _logits(N, V, dtype, cuda, seed=V)
    _check(x, t, k, token_logprobs(x, t, top_k=k), x.double())
    assert _status() == 0


@pytest.mark.parametrize("N,V,k,dtype", [(3000, 5003, 5, torch.bfloat16), (1790, 40003, 32, torch.float32),
                                         (1, 1200001, 20, torch.bfloat16), (2, 600001, 9, torch.float32)])
def test_many_rows_and_long_rows(cuda, N, V, k, dtype):
    """Rows that follow one another in a CTA; rows of more chunks than a window holds."""
    from scree_b200.kernels.native import token_logprobs

    x, t = _logits(N, V, dtype, cuda, seed=1)
    x[N // 2] = torch.arange(V, device=cuda).to(torch.float32).mul(1.0 / V).to(dtype)  # rising
    x[-1, V // 3:] = x[-1, 0]  # equal from there on
    r = token_logprobs(x, t, top_k=k)
    for a in range(0, N, 500):
        rows = slice(a, a + 500)
        part = type(r)(*(y[rows] for y in r))
        _check(x[rows], t[rows], k, part, x[rows].double())
    assert _status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_strided_rows_and_any_alignment(cuda, dtype, shift):
    from scree_b200.kernels.native import token_logprobs, token_logprobs_autograd

    big, t = _logits(9, 20011, dtype, cuda, seed=shift)
    x = big[:, shift:shift + 17001]
    t = t.clamp(max=17000)
    _check(x, t, 6, token_logprobs(x, t.int(), top_k=6), x.double())
    y = big.t().contiguous().t()[:, shift:shift + 17001]  # unit stride down the column
    _check(x, t, 6, token_logprobs(y, t, top_k=6), x.double())
    a = big.detach().clone().requires_grad_(True)
    token_logprobs_autograd(a[:, shift:shift + 17001], t).logp.sum().backward()
    one = torch.ones(9, dtype=torch.float64, device=cuda)
    want, tol = _grad_ref(x.double(), t, 0, one, 0 * one, one[:, None][:, :0])
    got = a.grad[:, shift:shift + 17001].double()
    assert ((got - want).abs() <= tol + HALF_ULP[dtype] * (want.abs() + tol)).all()
    assert _status() == 0


def test_ties_rank_by_lower_index(cuda):
    from scree_b200.kernels.native import token_logprobs

    # Whole rows equal (more candidates than fit the ranking buffer), two values, +0 and -0.
    x = torch.zeros((4, 40000), dtype=torch.bfloat16, device=cuda)
    x[1, ::3] = 1
    x[2, ::2] = -0.0
    x[3, 39000:] = -1
    t = torch.zeros(4, dtype=torch.int64, device=cuda)
    r = token_logprobs(x, t, top_k=32)
    a = torch.arange(32, device=cuda)
    assert torch.equal(r.top_ids, torch.stack([a, 3 * a, a, a]))
    _check(x, t, 32, r, x.double())


def test_rows_that_rise_along_the_vocabulary(cuda):
    """Every element beats all before it: the candidate buffer overflows."""
    from scree_b200.kernels.native import token_logprobs

    x = torch.arange(60000, dtype=torch.float32, device=cuda).mul(1e-3).repeat(3, 1)
    x[1] = x[1].flip(0)
    t = torch.tensor([59999, 0, 5], device=cuda)
    _check(x, t, 32, token_logprobs(x, t, top_k=32), x.double())
    y = x.to(torch.bfloat16)  # steps of equal values
    _check(y, t, 32, token_logprobs(y, t, top_k=32), y.double())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_masked_infinite_and_nan_logits(cuda, dtype):
    from scree_b200.kernels.native import token_logprobs, token_logprobs_autograd

    x, t = _logits(8, 20000, dtype, cuda, seed=5)
    x[0, 100:] = -np.inf          # most of the vocabulary masked
    x[1] = -np.inf                # nothing left
    x[2] = torch.finfo(dtype).min  # masked by the type's lowest value throughout
    x[3, 7:] = torch.finfo(dtype).min
    x[4, 5] = np.nan
    x[5, 19999] = np.inf
    x[6, :] = -np.inf
    x[6, 123] = 2.0               # one token left
    t[:] = 50
    t[6], t[7] = 123, -100
    r = token_logprobs(x, t, top_k=4)
    fin = _check(x, t, 4, r, x.double())
    assert fin.tolist() == [True, False, True, True, False, False, True, True]
    assert r.logp[1] == -np.inf and r.entropy[1] == 0 and r.top_ids[1].tolist() == [0, 1, 2, 3]
    assert torch.isneginf(r.top_logp[1]).all()
    assert r.logp[4].isnan() and r.entropy[4].isnan() and r.top_ids[4, 0] == 5
    assert r.logp[5].isnan() and r.top_ids[5, 0] == 19999
    assert r.logp[6] == 0 and r.entropy[6] == 0 and r.logp[7] == 0
    y = x.detach().requires_grad_(True)
    q = token_logprobs_autograd(y, t, top_k=4)
    (q.logp[:4].sum() + 2 * q.entropy[:4].sum() + q.entropy[6:].sum() + q.top_logp[0, :2].sum()).backward()
    g = y.grad.double()
    assert torch.isfinite(g[[0, 1, 2, 3, 6, 7]]).all()
    assert (g[1] == 0).all() and (g[0, 100:] == 0).all()
    assert _status() == 0


def _grad_ref(x, t, k, gl, gh, gt):
    logp, H, lse, ids, _, p, lp = _ref(x, t, k)
    g = torch.where(t < 0, torch.zeros_like(gl), gl)
    one = torch.zeros_like(x)
    one.scatter_add_(1, t.clamp(min=0)[:, None], g[:, None])
    if k:
        one.scatter_add_(1, ids, gt)
    ent = torch.where(p > 0, H[:, None] + lp, torch.zeros_like(p))
    gs = one.sum(1, keepdim=True)
    d = one - p * (gs + gh[:, None] * ent)
    r = 2.0**-17 + 8 * U * (x.abs() + lse[:, None].abs())
    return d, p * (gs.abs() + gh[:, None].abs() * (ent.abs() + 1)) * r + U * one.abs()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,V,k", [(1, 1, 0), (3, 5, 5), (7, 4099, 0), (4, 16400, 3), (3, 50257, 20)])
@pytest.mark.parametrize("given", ["all", "logp", "entropy", "top"])
def test_gradient(cuda, dtype, N, V, k, given):
    from scree_b200.kernels.native import token_logprobs_autograd

    x, t = _logits(N, V, dtype, cuda, seed=V + 1)
    if N > 2:
        t[1] = -1
    g = torch.Generator().manual_seed(3)
    gl, gh, gt = (torch.randn(s, generator=g).to(cuda) for s in ((N,), (N,), (N, k)))
    if given != "all":
        gl, gh, gt = (v if given == n else torch.zeros_like(v) for n, v in (("logp", gl), ("entropy", gh), ("top", gt)))
    y = x.detach().requires_grad_(True)
    r = token_logprobs_autograd(y, t, top_k=k)
    pairs = [(r.logp, gl, "logp"), (r.entropy, gh, "entropy"), (r.top_logp, gt, "top")]
    outs = [(o, w) for o, w, n in pairs if (given in ("all", n)) and (o.numel() or n != "top" or given == n)]
    torch.autograd.backward([o for o, _ in outs], [w for _, w in outs])
    want, tol = _grad_ref(x.double(), t, k, gl.double(), gh.double(), gt.double())
    err = (y.grad.double() - want).abs()
    tiny = 2.0**-25 if dtype == torch.float16 else 0.0  # half of the smallest fp16 step
    assert (err <= tol + HALF_ULP[dtype] * (want.abs() + tol) + tiny).all(), float((err - tol).max())


def test_gradient_against_differences(cuda):
    """Central differences (h = 1e-5) of the float64 definition: their error is below
    h^2 * |third derivative| + 2^-52 |f| / h < 1e-9."""
    from scree_b200.kernels.native import token_logprobs_autograd

    N, V, k = 3, 11, 4
    x, t = _logits(N, V, torch.float32, cuda, seed=2, scale=1.0)
    t[2] = -5
    g = torch.Generator().manual_seed(4)
    gl, gh, gt = (torch.randn(s, generator=g, dtype=torch.float64).to(cuda) for s in ((N,), (N,), (N, k)))
    ids = _ref(x.double(), t, k)[3]

    def f(z):
        lp = torch.log_softmax(z, 1)
        logp = torch.where(t < 0, torch.zeros_like(gl), lp.gather(1, t.clamp(min=0)[:, None])[:, 0])
        return (gl * logp).sum() - (gh * (lp.exp() * lp).sum(1)).sum() + (gt * lp.gather(1, ids)).sum()

    want = torch.zeros((N, V), dtype=torch.float64, device=cuda)
    for i in range(N):
        for j in range(V):
            z = x.double().clone()
            z[i, j] += 1e-5
            hi = f(z)
            z[i, j] -= 2e-5
            want[i, j] = (hi - f(z)) / 2e-5
    y = x.detach().requires_grad_(True)
    r = token_logprobs_autograd(y, t, top_k=k)
    torch.autograd.backward([r.logp, r.entropy, r.top_logp], [gl.float(), gh.float(), gt.float()])
    _, tol = _grad_ref(x.double(), t, k, gl, gh, gt)
    # + 2e-7: the upstream gradients were rounded to fp32
    assert ((y.grad.double() - want).abs() <= tol + 1e-8 + 2.0**-22 * (1 + want.abs())).all()


def test_array_level_and_other_stream(cuda):
    import scree_b200 as scree
    from scree_b200.kernels import native, varlen_token_logprobs

    x, t = _logits(12, 3001, torch.bfloat16, cuda, seed=8)
    offs = torch.tensor([0, 5, 5, 12], dtype=torch.int32, device=cuda)
    want = native.token_logprobs(x, t, top_k=2)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        r = varlen_token_logprobs(scree.from_cu_seqlens(x, offs), scree.from_cu_seqlens(t, offs), top_k=2)
    side.synchronize()
    for a, b in zip(r, want):
        assert torch.equal(a.values, b) and a.offsets is offs
    assert _status() == 0


def test_refusals(cuda):
    from scree_b200 import _lib
    from scree_b200.kernels.native import token_logprobs

    x, t = _logits(4, 100, torch.float32, cuda)
    with pytest.raises(ValueError, match="top must be"):
        token_logprobs(x, t, top_k=33)
    with pytest.raises(ValueError, match="top must be"):
        token_logprobs(x[:, :5], t.clamp(max=4), top_k=6)
    with pytest.raises(ValueError, match="top must be"):
        token_logprobs(x, t, top_k=-1)
    with pytest.raises(AssertionError, match="targets"):
        token_logprobs(x, t[:3])
    with pytest.raises(AssertionError, match="int32 or int64"):
        token_logprobs(x, t.float())
    with pytest.raises(AssertionError, match="fp16, bf16 or fp32"):
        token_logprobs(x.double(), t)
    with pytest.raises(AssertionError, match="CUDA"):
        token_logprobs(x.cpu(), t.cpu())
    assert token_logprobs(x[:0], t[:0], top_k=3).top_ids.shape == (0, 3)
    t[1] = 100
    r = token_logprobs(x, t)
    assert r.logp[1].isnan() and torch.isfinite(r.logp[[0, 2, 3]]).all()
    st = _lib.device_status()
    assert st >> 16 == _lib.DEVERR_BAD_INPUT and st & 0xFFFF == 50
    assert _status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 3, 9, 2047, 8193, 16391])
def test_neighbouring_rows_do_not_matter(cuda, dtype, V):
    """Rows of odd lengths at every alignment, their neighbours NaN, the tensor between NaN."""
    from scree_b200.kernels import native

    for shift in range(0, 8, 3):
        for N in (1, 2, 5):
            x, t = _logits(N, V, dtype, cuda, seed=shift + N)
            k = min(V, 7)
            buf = torch.full((shift + 2 * N * V + 9,), float("nan"), dtype=dtype, device=cuda)
            rows = buf[shift:shift + 2 * N * V].view(N, 2, V)[:, 0]  # row stride 2 V
            rows.copy_(x)
            alone = native.token_logprobs(x, t, top_k=k)
            got = native.token_logprobs(rows, t, top_k=k)
            _check(x, t, k, got, x.double())
            assert torch.equal(got.top_ids, alone.top_ids)
            whole = buf[shift:shift + 2 * N * V].view(2 * N, V)      # every other row is NaN
            two = native.token_logprobs(whole, t.repeat_interleave(2), top_k=k)
            assert two.logp[1::2].isnan().all()
            _check(x, t, k, native.TokenLogprobs(*(r[::2] for r in two)), x.double())
    assert _status() == 0


@pytest.mark.parametrize("kept", [0, 1, 5, 31, 40])
def test_rows_masked_but_for_a_few_tokens(cuda, kept):
    """Constrained decoding: all logits -inf but a few; the rest rank by index."""
    from scree_b200.kernels import native

    N, V, k = 6, 150001, 32
    x = torch.full((N, V), -float("inf"), dtype=torch.bfloat16, device=cuda)
    g = torch.Generator().manual_seed(kept)
    for n in range(N):
        at = torch.randperm(V, generator=g)[:kept].to(cuda)
        x[n, at] = torch.randn(kept, generator=g).to(torch.bfloat16).to(cuda)
    t = x.float().argmax(1)
    got = native.token_logprobs(x, t, top_k=k)
    order = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(got.top_ids, order)
    if kept:
        _check(x, t, k, got, x.double())
    else:
        assert (got.logp == -float("inf")).all() and (got.entropy == 0).all()
    assert _status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [5, 1003, 8192])
def test_gradient_of_rows_at_every_alignment(cuda, dtype, V):
    """dx is contiguous; the logits' rows begin anywhere in their 16-byte blocks, NaN between them."""
    from scree_b200.kernels import native

    N = 9
    x, t = _logits(N, V, dtype, cuda, seed=V)
    g = torch.Generator().manual_seed(1)
    gl, gh, gt = (torch.randn(s, generator=g).to(cuda) for s in ((N,), (N,), (N, 2)))
    want, tol = _grad_ref(x.double(), t, 2, gl.double(), gh.double(), gt.double())
    tiny = 2.0**-25 if dtype == torch.float16 else 0.0
    for pad in range(0, 9):
        for shift in (0, 3):
            buf = torch.full((shift + N * (V + pad),), float("nan"), dtype=dtype, device=cuda)
            rows = buf[shift:].view(N, V + pad)[:, :V]
            rows.copy_(x)
            y = rows.detach().requires_grad_(True)
            r = native.token_logprobs_autograd(y, t, 2)
            torch.autograd.backward([r.logp, r.entropy, r.top_logp], [gl, gh, gt])
            err = (y.grad.double() - want).abs()
            assert (err <= tol + HALF_ULP[dtype] * (want.abs() + tol) + tiny).all(), (pad, shift)
    assert _status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("mask", [-1e4, -1e9, -1e30, 3000.0])
def test_rows_masked_with_large_numbers(cuda, dtype, mask):
    """Whole rows, and all that a thread reads before a row's last quarter, at one large number."""
    from scree_b200.kernels import native

    if dtype == torch.float16 and abs(mask) > 6e4:
        mask = -6e4
    N, V, k = 4, 30011, 6
    x, t = _logits(N, V, dtype, cuda, seed=11)
    x[:, :3 * V // 4] = mask
    x[1] = mask                      # a whole row
    x[2, 5] = 2.0                    # one token early on
    y = x.detach().requires_grad_(True)
    got = native.token_logprobs_autograd(y, t, k)
    _check(x, t, k, native.TokenLogprobs(*(r.detach() for r in got)), x.double())
    # The row of equal values is uniform whatever they are.
    flat = native.TokenLogprobs(*(r.detach()[1:2] for r in got))
    assert abs(flat.logp.item() + np.log(V)) <= 2.0**-15 and abs(flat.entropy.item() - np.log(V)) <= 2.0**-12
    g = torch.Generator().manual_seed(2)
    gl, gh, gt = (torch.randn(s, generator=g).to(cuda) for s in ((N,), (N,), (N, k)))
    torch.autograd.backward([got.logp, got.entropy, got.top_logp], [gl, gh, gt])
    want, tol = _grad_ref(x.double(), t, k, gl.double(), gh.double(), gt.double())
    tiny = 2.0**-25 if dtype == torch.float16 else 0.0
    err = (y.grad.double() - want).abs()
    assert (err <= tol + HALF_ULP[dtype] * (want.abs() + tol) + tiny).all()
    assert _status() == 0
