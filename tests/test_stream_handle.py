"""_lib.stream_handle takes what torch.cuda.current_stream takes: nothing, a device, its text or its index."""
import types

import pytest
import torch

from dilabhelmholtzoct_amd import _lib


def test_device_forms(monkeypatch):
    seen = []

    def current_stream(device=None):
        seen.append(device)
        return types.SimpleNamespace(cuda_stream=1000)
    monkeypatch.setattr(torch.cuda, "current_stream", current_stream)
    for device in (3, "cuda:2", "cuda", torch.device("cuda"), torch.device("cuda", 1)):
        assert _lib.stream_handle(device) == 1000
    assert seen == [3, "cuda:2", "cuda", torch.device("cuda"), torch.device("cuda", 1)]


@pytest.mark.gpu
def test_handles(cuda):
    side = torch.cuda.Stream()
    for stream in (torch.cuda.default_stream(), side):
        with torch.cuda.stream(stream):
            for device in (None, 0, "cuda", "cuda:0", torch.device("cuda"), torch.device("cuda", 0)):
                assert _lib.stream_handle(device) == stream.cuda_stream
    with pytest.raises(ValueError):
        _lib.stream_handle(torch.device("cpu"))
