"""The stream and device that calls go to, with and without torch's raw stream getter."""

from types import SimpleNamespace

import pytest
import torch

from diffspec_mi355x import _ext


def test_handle_without_the_raw_getter(monkeypatch):
    seen = []
    monkeypatch.setattr(_ext, "_raw_stream", None)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d: seen.append(d) or SimpleNamespace(cuda_stream=77))
    assert _ext.stream_of(torch.device("cuda", 3)).value == 77
    assert seen == [torch.device("cuda", 3)]


def test_handle_of_the_raw_getter(monkeypatch):
    seen = []
    monkeypatch.setattr(_ext, "_raw_stream", lambda i: seen.append(i) or 55)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 2)
    assert _ext.stream_of(torch.device("cuda")).value == 55
    assert _ext.stream_of(torch.device("cuda", 1)).value == 55
    assert seen == [2, 1]


def test_device_context(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 2)
    assert _ext.on_device(torch.device("cuda", 2)) is _ext._HERE
    assert isinstance(_ext.on_device(torch.device("cuda", 1)), torch.cuda.device)


@pytest.mark.gpu
def test_handles_agree(gpu, monkeypatch):
    side = torch.cuda.Stream()
    for stream in (torch.cuda.default_stream(), side):
        with torch.cuda.stream(stream):
            want = torch.cuda.current_stream(gpu).cuda_stream or None
            assert _ext.stream_of(gpu).value == want == (stream.cuda_stream or None)
            with monkeypatch.context() as m:
                m.setattr(_ext, "_raw_stream", None)
                assert _ext.stream_of(gpu).value == want
