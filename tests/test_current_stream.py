"""The stream that the Python calls launch on, with and without torch's call for its raw handle."""
import types

import pytest
import torch

from inferno_amd import attention as A


@pytest.mark.parametrize("raw", [True, False])
def test_the_current_stream(monkeypatch, raw):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(cuda_stream=100 + device))
    if raw:
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 200 + device, raising=False)
    else:
        monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    assert A._device_stream() == (3, 203 if raw else 103)
    assert A._stream() == (203 if raw else 103)
