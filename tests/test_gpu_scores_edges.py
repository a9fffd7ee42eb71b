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
