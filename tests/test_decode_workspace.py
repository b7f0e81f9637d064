"""Which buffer a 16-bit split-KV decode takes for its partials (no GPU: torch.cuda is a stand-in)."""

import contextlib

import pytest
import torch

from hcp_vllm_plugin_b200 import ops


class _Buffer:
    def __init__(self, n, dtype, device):
        self.n, self.device = n, device

    def numel(self):
        return self.n


class _Cuda:
    """Two GPUs, a current one, and the GPU whose current stream is being captured."""

    def __init__(self, monkeypatch, current, captured):
        self.current, self.captured = current, captured
        monkeypatch.setattr(ops, "_workspaces", {})
        monkeypatch.setattr(torch, "empty", _Buffer)
        monkeypatch.setattr(torch.cuda, "current_device", lambda: self.current)
        monkeypatch.setattr(torch.cuda, "device", self.device)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: self.current == self.captured)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: type("S", (), {"cuda_stream": 7})())

    @contextlib.contextmanager
    def device(self, device):
        before, self.current = self.current, torch.device(device).index
        yield
        self.current = before


@pytest.mark.parametrize("current", [0, 1])
def test_a_captured_call_on_another_gpu_keeps_its_buffer(monkeypatch, current):
    """The capture that counts is that of the call's GPU, whichever GPU is the current one: the captured
    call's buffer is its own, and no eager call's buffer comes out of a graph's memory."""
    _Cuda(monkeypatch, current, captured=1)
    here = [ops._workspace(torch.device("cuda", 1), 100) for _ in range(2)]
    assert here[0] is not here[1] and ops._workspaces == {}
    other = [ops._workspace(torch.device("cuda", 0), 100) for _ in range(2)]
    assert len(ops._workspaces) == 1
    assert other[0] is other[1] and other[0].device.index == 0


def test_eager_calls_share_the_streams_buffer(monkeypatch):
    _Cuda(monkeypatch, 0, captured=None)
    a, b = (ops._workspace(torch.device("cuda", 0), 100) for _ in range(2))
    assert a is b
