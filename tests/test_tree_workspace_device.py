"""The workspace of a tree attention call is sized for the device that runs it, whichever device is
current."""

import types

import pytest
import torch

from dispec_amd import _lib
from dispec_amd.engine import hip_attn


@pytest.fixture()
def two_devices(monkeypatch):
    """Device 0 (current) needs 4096 bytes a sequence, device 1 twice as many."""
    current = [0]

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *a):
            current[0] = self.before

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(_lib, "lib", lambda: types.SimpleNamespace(
        dsp_paged_tree_workspace_bytes=lambda B, *a: 4096 * B * (1 + current[0])))
    monkeypatch.setattr(torch, "empty", lambda n, dtype, device: (4 * (n - 1), device))
    hip_attn._tree_ws_bytes.cache_clear()
    yield
    hip_attn._tree_ws_bytes.cache_clear()


def test_each_device_has_its_size(two_devices):
    args = (3, 8, 2, 128, 16, 1024)
    for device, need in (("cuda:0", 1), ("cuda:1", 2), ("cuda", 1), (1, 2), (torch.device("cuda:0"), 1)):
        assert hip_attn.tree_workspace(*args, device) == (3 * 4096 * need, device)
