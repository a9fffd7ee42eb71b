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
