"""What a caller gives as a stream -- nothing, a torch stream, a handle -- is the stream that the call and its memory use."""
import types

import pytest
import torch

from sdr_amd import batch, dense


@pytest.fixture
def streams(monkeypatch):
    """torch's streams, without a device: by what they were asked for"""
    def external(handle, device=None):
        assert handle != 0, "a null handle asks for any stream of a pool"
        return types.SimpleNamespace(cuda_stream=handle, kind="external", device=device)

    default = types.SimpleNamespace(cuda_stream=0, kind="default")
    current = types.SimpleNamespace(cuda_stream=77, kind="current")
    monkeypatch.setattr(torch.cuda, "ExternalStream", external)
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: default)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: current)
    monkeypatch.setattr(dense, "_raw_stream", lambda device: current.cuda_stream)
    return types.SimpleNamespace(default=default, current=current)


def test_the_default_streams_handle_is_the_default_stream(streams):
    assert batch._torch_stream(0, 0) is streams.default
    assert batch._stream_handle(0, 0) == 0 and dense._handle(0, 0) == 0


def test_the_current_stream_other_handles_and_stream_objects(streams):
    assert batch._torch_stream(0, None) is streams.current
    assert batch._stream_handle(0, None) == 77 and dense._handle(0, None) == 77
    assert batch._torch_stream(0, 1234).cuda_stream == 1234 and dense._handle(0, 1234) == 1234
    own = types.SimpleNamespace(cuda_stream=55)
    assert batch._torch_stream(0, own).cuda_stream == 55 and dense._handle(0, own) == 55


def test_an_object_that_carries_a_handle_alone(streams):
    """it is enough for the calls; torch gets a stream of its own kind for it"""
    for handle, kind in ((55, "external"), (0, "default")):
        assert batch._torch_stream(0, types.SimpleNamespace(cuda_stream=handle)).kind == kind
