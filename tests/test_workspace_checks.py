"""Workspace: whose buffer a call gets.  No GPU is needed: buffers are stand-ins, nothing is launched."""
import types

import pytest
import torch

from tqkv import int4, ops

KEY = (1, 4, 2, 5000, 128)


def _buffer(device, size=1 << 20):
    return types.SimpleNamespace(get_device=lambda: device, numel=lambda: size, data_ptr=lambda: 4096,
                                 device=torch.device("cuda", device))


@pytest.fixture
def sizes(monkeypatch):
    monkeypatch.setattr(int4, "_ws_bytes", {(i, KEY): 4096 for i in (0, 1)})


@pytest.mark.parametrize("named", ["cuda", "cuda:0"])
def test_a_buffer_of_another_device_is_refused(sizes, named):
    """A Workspace without an index takes the device of its first use, and serves no other."""
    ws = ops.Workspace(named)
    ws.buf = _buffer(0)
    assert int4._workspace(ws, 0, 0, KEY) == (4096, 1 << 20)
    with pytest.raises(ValueError, match="cuda:0.*cuda:1"):
        int4._workspace(ws, 1, 0, KEY)
    assert ops._workspace(ws, torch.device("cuda:0")) is ws
    with pytest.raises(ValueError, match="cuda:0.*cuda:1"):
        ops._workspace(ws, torch.device("cuda:1"))


def test_a_workspace_for_another_device_is_refused_before_it_has_a_buffer(sizes):
    ws = ops.Workspace("cuda:0")
    with pytest.raises(ValueError, match="cuda:0.*cuda:1"):
        int4._workspace(ws, 1, 0, KEY)
    with pytest.raises(ValueError, match="cuda:0.*cuda:1"):
        ops._workspace(ws, torch.device("cuda:1"))
