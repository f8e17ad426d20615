"""The operators find the current device and stream with torch's documented functions alone, should its short ways be missing."""
import importlib.util

import pytest
import torch


def documented(monkeypatch):
    """A second copy of the module, imported where the short ways do not exist."""
    import dgl_amd.attention as module
    for name in ("_cuda_getCurrentRawStream", "_cuda_getDevice"):
        monkeypatch.delattr(torch._C, name, raising=False)
    spec = importlib.util.spec_from_file_location("dgl_amd.attention_documented", module.__file__)
    copy = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(copy)
    monkeypatch.undo()
    return copy


def test_import_without_the_short_ways(monkeypatch):
    copy = documented(monkeypatch)
    assert copy._current_device is torch.cuda.current_device and callable(copy._raw_stream)


@pytest.mark.gpu
def test_same_stream_either_way(device, monkeypatch):
    import dgl_amd.attention as module
    copy = documented(monkeypatch)
    q = torch.randn(1, 2, 100, 16, device=device)
    s = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), s):
        with torch.cuda.stream(stream):
            assert copy._raw_stream(device.index) == module._raw_stream(device.index) == stream.cuda_stream
            assert copy._current_device() == module._current_device() == device.index
            a, b = copy.attention(q, q, q), module.attention(q, q, q)
        stream.synchronize()
        assert torch.equal(a, b)
