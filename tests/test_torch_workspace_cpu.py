"""Where the torch operators' workspaces are zero-filled: on the device of the
operator's tensors, whichever is current (CPU stand-ins for the devices)."""
import contextlib
import importlib

import pytest
import torch

kvq = importlib.import_module("cuda-operators_amd").kvq
torch_ops = importlib.import_module("cuda-operators_amd.torch_ops")


class Devices:
    """torch.cuda's current device, and what was done under which."""

    def __init__(self, monkeypatch, capturing=()):
        self.current, self.log = 0, []
        empty = torch.empty
        monkeypatch.setattr(torch, "empty", lambda n, dtype, device: empty(n, dtype=dtype))
        monkeypatch.setattr(torch.cuda, "device", self.device)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: self.current in capturing)
        monkeypatch.setattr(kvq, "workspace_init", lambda ws, nbytes=None, stream=None: self.log.append((self.current, nbytes, stream)))
        monkeypatch.setattr(torch_ops, "_workspaces", {})
        monkeypatch.setattr(torch_ops, "_retired", [])

    @contextlib.contextmanager
    def device(self, d):
        before, self.current = self.current, d.index if isinstance(d, torch.device) else d
        yield
        self.current = before


@pytest.mark.parametrize("index", [0, 1, 3])
def test_zero_filled_on_its_own_device(monkeypatch, index):
    devices = Devices(monkeypatch)
    key, device = ("op", index, 7), torch.device("cuda", index)
    ws = torch_ops._workspace(key, 1000, device)
    assert devices.log == [(index, 1000, None)] and devices.current == 0
    assert torch_ops._workspace(key, 900, device) is ws and len(devices.log) == 1
    assert torch_ops._workspace(key, 1500, device) is not ws
    assert devices.log[1:] == [(index, 2000, None)] and torch_ops._retired == [ws]


def test_capture_on_its_own_device(monkeypatch):
    """A workspace made while its device's stream is captured stays with that graph; a capture on another does not count."""
    devices = Devices(monkeypatch, capturing={1})
    ws = torch_ops._workspace(("op", 1, 7), 64, torch.device("cuda", 1))
    assert torch_ops._workspaces == {} and torch_ops._retired == [ws]
    torch_ops._workspace(("op", 2, 7), 64, torch.device("cuda", 2))
    assert list(torch_ops._workspaces) == [("op", 2, 7)] and [d for d, _, _ in devices.log] == [1, 2]
