"""Edges of the token scores on the GPU: what their calls refuse, and how exact they are where
logits are far from 0.  References and bounds as in test_gpu_logprobs.py."""

import pytest
import torch
from test_gpu_logprobs import _logits, _status

pytestmark = pytest.mark.gpu


def test_gradient_of_ids_outside_the_vocabulary(cuda):
    """The C entry takes ids as they come: for those that are none nothing is written, in the
    gradient's rows or beside them, but what the whole row has of their weight."""
    from scree_b200 import _lib
    from scree_b200.kernels.native import token_logprobs_autograd

    N, V, k = 3, 1001, 3
    x, t = _logits(N, V, torch.float32, cuda, seed=4)
    y = x.detach().requires_grad_(True)
    r = token_logprobs_autograd(y, t, k)
    g = torch.ones((N, k), device=cuda)
    (want,) = torch.autograd.grad(r.top_logp, y, g)
    want = want.scatter_add(1, r.top_ids[:, 1:2], -g[:, :1])  # all but the second id's own element
    norm = torch.stack([x.amax(1), torch.logsumexp(x - x.amax(1, keepdim=True), 1)], 1)
    for bad in (V, V + 5, 2000, 2**40, -1):
        ids = r.top_ids.clone()
        ids[:, 1] = bad
        buf = torch.full((N * V + 4096,), 5.0, device=cuda)
        rc = _lib.load().scree_token_logprobs_bwd(
            x.data_ptr(), V, t.data_ptr(), 1, norm.data_ptr(), r.entropy.detach().contiguous().data_ptr(),
            ids.data_ptr(), None, None, g.data_ptr(), N, V, k, _lib.F32, buf.data_ptr(), _lib.stream_ptr(x.device))
        _lib.check(rc, "token_logprobs backward")
        st = _lib.device_status()
        assert st >> 16 == _lib.DEVERR_BAD_INPUT and st & 0xFFFF == 52
        assert (buf[N * V:] == 5).all()
        # (norm is torch's here: p to a few units in its last place)
        torch.testing.assert_close(buf[:N * V].view(N, V), want, atol=1e-5, rtol=1e-5)
    assert _status() == 0


def _far_logits(N, V, dtype, cuda):
    """Rows around levels from 20 to 1,000 of either sign (fp32 spacing up to 2^-14 there)."""
    x, t = _logits(N, V, torch.float32, cuda, seed=21)
    level = torch.tensor([20.0, 100.0, 333.3, 700.0, 1000.0, -100.0, -700.0, -1000.0], device=cuda)
    x = x + level.repeat(N // 8)[:, None]
    return x.clamp(-1020, 1020).to(dtype), t


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [4099, 32000, 131072])
def test_scores_do_not_depend_on_the_logits_level(cuda, dtype, V):
    """log p is a function of differences, x - m and log s1, each rounded to fp32 (u = 2^-24);
    s1's relative error is below 2^-17 wherever the row lies (test_gpu_logprobs.py)."""
    from scree_b200.kernels.native import token_logprobs

    u, k = 2.0**-24, 5
    x, t = _far_logits(24, V, dtype, cuda)
    got = token_logprobs(x, t, top_k=k)
    d = x.double() - x.double().amax(1, keepdim=True)
    rest = torch.logsumexp(d, 1, keepdim=True)
    lp = d - rest
    tol = 2.0**-17 + 4 * u * (rest.abs() + d.abs())
    at = lambda z, i: z.gather(1, i)  # noqa: E731
    assert ((got.logp[:, None].double() - at(lp, t[:, None])).abs() <= at(tol, t[:, None])).all()
    assert ((got.top_logp.double() - at(lp, got.top_ids)).abs() <= at(tol, got.top_ids)).all()
    H = -(lp.exp() * lp).sum(1)
    assert ((got.entropy.double() - H).abs() <= 2.0**-16 * (1 - (lp.exp() * d).sum(1))).all()
    assert _status() == 0


@pytest.mark.parametrize("V", [4099, 32000, 131072])
def test_gradient_does_not_depend_on_the_logits_level(cuda, V):
    """p's relative error comes from the same differences; fp32 logits keep it visible."""
    from scree_b200.kernels.native import token_logprobs_autograd

    u, k, N = 2.0**-24, 3, 24
    x, t = _far_logits(N, V, torch.float32, cuda)
    gen = torch.Generator().manual_seed(6)
    gl, gh, gt = (torch.randn(s, generator=gen).to(cuda) for s in ((N,), (N,), (N, k)))
    y = x.detach().requires_grad_(True)
    r = token_logprobs_autograd(y, t, k)
    torch.autograd.backward([r.logp, r.entropy, r.top_logp], [gl, gh, gt])
    d = x.double() - x.double().amax(1, keepdim=True)
    rest = torch.logsumexp(d, 1, keepdim=True)
    lp = d - rest
    p = lp.exp()
    H = -(p * lp).sum(1, keepdim=True)
    one = torch.zeros_like(p).scatter_add_(1, t[:, None], gl.double()[:, None]).scatter_add_(1, r.top_ids, gt.double())
    gs = one.sum(1, keepdim=True)
    ent = gh.double()[:, None] * (lp + H)
    want = one - p * (gs + ent)
    rel = 2.0**-17 + 8 * u * (d.abs() + rest.abs())
    tol = p * (gs.abs() + ent.abs() + gh.double().abs()[:, None]) * rel + u * (one.abs() + want.abs())
    assert ((y.grad.double() - want).abs() <= tol).all()
    assert _status() == 0


def test_a_second_derivative_is_refused(cuda):
    """The gradient is a kernel's output and no function of the logits to autograd: a term made of
    it would lose its own gradient."""
    from scree_b200.kernels.native import token_logprobs_autograd

    x, t = _logits(3, 50, torch.float32, cuda)
    y = x.detach().requires_grad_(True)
    w = torch.ones(3, device=cuda, requires_grad=True)
    r = token_logprobs_autograd(y, t)
    (g,) = torch.autograd.grad((r.logp * w).sum(), y, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (g.square().sum() + y.square().sum()).backward()
    y.grad = None
    token_logprobs_autograd(y, t).logp.sum().backward(create_graph=False)
    assert y.grad is not None and _status() == 0
