"""Workspace: whose buffer a call gets.  No GPU is needed: buffers are stand-ins, nothing is launched."""
import threading
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


def test_a_workspace_in_host_memory_is_refused(sizes):
    """Its buffer's address would go to a kernel."""
    ws = ops.Workspace("cpu")
    for _ in range(2):
        with pytest.raises(ValueError, match="workspace is on cpu"):
            int4._workspace(ws, 0, 0, KEY)
        with pytest.raises(ValueError, match="workspace is on cpu"):
            ops._workspace(ws, torch.device("cuda:0"))
        ws.buf = torch.empty(1 << 20, dtype=torch.uint8)


def _grow(monkeypatch, init):
    """A Workspace in host memory whose zeroing is `init`."""
    monkeypatch.setattr(ops, "load", lambda: types.SimpleNamespace(tqkv_workspace_init=init))
    return ops.Workspace("cpu"), types.SimpleNamespace(cuda_stream=0)


def test_a_buffer_is_handed_out_only_once_its_zeroing_is_enqueued(monkeypatch):
    """A second thread that meets a growing Workspace on the same stream must not launch with the new
    buffer ahead of its zeroing: the kernels' counters have to be zero."""
    began, done = threading.Event(), threading.Event()
    zeroed = []

    def init(ptr, size, stream):
        began.set()
        assert done.wait(20)
        zeroed.append(ptr)
        return 0

    ws, stream = _grow(monkeypatch, init)
    got = []
    threads = [threading.Thread(target=lambda: got.append((*ws.get(1000, stream), list(zeroed))))
               for _ in range(2)]
    threads[0].start()
    assert began.wait(20)
    threads[1].start()
    threads[1].join(0.3)
    early = list(got)
    done.set()
    for t in threads:
        t.join(20)
    assert early == []
    assert len(got) == 2 and got[0][:2] == got[1][:2] and all(p in z for p, _, z in got)
    assert len(zeroed) == 1 and ws._retired == []


def test_a_buffer_whose_zeroing_failed_is_not_kept(monkeypatch):
    answers = [5, 0]
    ws, stream = _grow(monkeypatch, lambda *a: answers.pop(0))
    monkeypatch.setattr(ops, "check", lambda name, status: (_ for _ in ()).throw(RuntimeError(name)) if status else None)
    with pytest.raises(RuntimeError):
        ws.get(1000, stream)
    assert ws.buf is None
    assert ws.get(1000, stream)[1] == 1000 and answers == []


def test_growing_keeps_what_was_handed_out(monkeypatch):
    ws, stream = _grow(monkeypatch, lambda *a: 0)
    first = ws.get(1000, stream)
    assert ws.get(900, stream) == first
    second = ws.get(1001, stream)
    assert second[1] == 2000 and [b.data_ptr() for b in ws._retired] == [first[0]]


def test_threads_of_one_stream_share_one_default_workspace(monkeypatch):
    """Two threads' first calls: one Workspace, so that no buffer is dropped while a launch uses it."""
    monkeypatch.setattr(int4, "_default_ws", {})
    monkeypatch.setattr(int4, "_ws_bytes", {(0, KEY): 4096})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    gate = threading.Barrier(2)

    class Slow:
        def __init__(self, device):
            try:
                gate.wait(0.5)
            except threading.BrokenBarrierError:
                pass

        def get(self, need):
            return id(self), need

    monkeypatch.setattr(int4, "Workspace", Slow)
    got = []
    threads = [threading.Thread(target=lambda: got.append(int4._workspace(None, 0, 7, KEY))) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(20)
    kept = int4._default_ws[(0, 7)]
    assert [g[0] for g in got] == [id(kept)] * 2
