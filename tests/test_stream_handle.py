"""_lib.stream_handle: the stream of the device that is named, however it is named (no GPU)."""
import pytest
import torch

from otfuse import _lib


@pytest.fixture
def streams(monkeypatch):
    """device i's current stream is 100 + i; device 2 is current"""
    class Stream:
        def __init__(self, i):
            self.cuda_stream = 100 + i

    def current_stream(device=None):
        if device is None:
            return Stream(2)
        if isinstance(device, int):
            return Stream(device)
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"Expected a cuda device, but got: {device}")
        return Stream(2 if device.index is None else device.index)

    monkeypatch.setattr(torch.cuda, "current_stream", current_stream)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 2)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 100 + i, raising=False)


@pytest.mark.parametrize("device,want", [(None, 102), (1, 101), (0, 100), ("cuda:1", 101), ("cuda", 102), (torch.device("cuda", 1), 101),
                                         (torch.device("cuda"), 102)])
def test_names_of_a_device(streams, device, want):
    assert _lib.stream_handle(device) == want


def test_a_host_device_is_refused(streams):
    for device in ("cpu", torch.device("cpu"), torch.device("cpu", 0)):
        with pytest.raises(ValueError):
            _lib.stream_handle(device)
