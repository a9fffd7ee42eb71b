"""stream_ptr takes what torch.cuda.current_stream takes, and gives the same stream."""

import types

import pytest
import torch

from scree_b200 import _lib


@pytest.mark.parametrize("device", [None, 1, "cuda:1", "cuda", torch.device("cuda", 1), torch.device("cuda")])
def test_stream_of_any_way_to_name_a_device(monkeypatch, device):
    def index(d):
        if d is None or isinstance(d, int):
            return d or 0
        return torch.device(d).index or 0

    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: types.SimpleNamespace(cuda_stream=100 + index(d)))
    monkeypatch.setattr(_lib, "_raw_stream", lambda i: 100 + i)
    assert _lib.stream_ptr(device) == 100 + index(device)
