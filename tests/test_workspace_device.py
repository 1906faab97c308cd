"""Which recording a workspace belongs to, where the tensors' device is not the current one (CPU, with stand-ins: one
process here sees no two GPUs)."""

import pytest
import torch

from tinyvllm_b200 import _lib, attention


class _Lib:
    def __init__(self, captures):
        self.captures = captures                # stream -> capture id

    def tvk_stream_capture_id(self, out, stream):
        assert stream != 0                      # of whichever device is the current one, and never recording
        out._obj.value = self.captures.get(stream, 0)
        return 0


@pytest.fixture
def two_devices(monkeypatch):
    """Device 0 is the current one; device i's current stream is 100 + i.  Returns the recording streams."""
    captures = {}
    real_empty, real_device = torch.empty, torch.device
    monkeypatch.setattr(_lib, "lib", lambda: _Lib(captures))
    monkeypatch.setattr(_lib, "raw_stream", lambda index: 100 + index)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: captures.get(100, 0) != 0)
    monkeypatch.setattr(attention.torch, "empty", lambda n, dtype, device: real_empty(n, dtype=dtype, device="meta"))
    monkeypatch.setattr(attention, "_capture_workspaces", {})
    monkeypatch.setattr(attention, "_workspaces", {})
    monkeypatch.setattr(attention, "_workspace", lambda device, nbytes, kind: f"eager {real_device(device).index}")
    return captures


@pytest.mark.parametrize("index", [0, 1])
def test_a_recording_on_the_tensors_device_has_its_own_workspace(two_devices, index):
    assert attention.call_workspace(index, 1000, "decode_q8", 16) == f"eager {index}"
    two_devices[100 + index] = 7
    a = attention.call_workspace(index, 1000, "decode_q8", 16)
    assert isinstance(a, torch.Tensor) and a.numel() == 1000
    assert attention.call_workspace(index, 1000, "decode_q8", 16) is a            # the same recording
    assert attention.call_workspace(1 - index, 1000, "decode_q8", 16) == f"eager {1 - index}"
    two_devices[100 + index] = 8
    assert attention.call_workspace(index, 1000, "decode_q8", 16) is not a        # the next one


def test_a_default_stream_never_records(two_devices, monkeypatch):
    two_devices[101] = 7
    monkeypatch.setattr(_lib, "raw_stream", lambda index: 0)
    assert attention.call_workspace(1, 1000, "decode_q8", 16) == "eager 1"
