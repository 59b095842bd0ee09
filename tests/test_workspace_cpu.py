"""`ops.workspace` on the CPU: the stream, its capture and the device stand in as fakes."""
import pytest
import torch

from unpopped_b200 import ops


@pytest.fixture
def fake(monkeypatch):
    state = dict(stream=7, capturing=False, device=0)
    monkeypatch.setattr(ops, "_raw_stream", lambda index: state["stream"])
    monkeypatch.setattr(ops, "_ws_cache", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    monkeypatch.setattr(torch.cuda, "current_device", lambda: state["device"])
    return state


def test_a_capture_has_workspaces_of_its_own(fake):
    on = torch.device("cpu", 0)
    eager = ops.workspace("t", 512, on)
    eager.fill_(3)
    assert ops.workspace("t", 300, on) is eager
    fake["capturing"] = True
    one, two = ops.workspace("t", 512, on), ops.workspace("t", 4096, on)
    first = ops.workspace("u", 100, on)
    assert len({t.data_ptr() for t in (eager, one, two, first)}) == 4
    assert all(int(t.sum()) == 0 for t in (one, two, first)) and two.numel() == 4096
    fake["capturing"] = False
    assert ops.workspace("t", 512, on) is eager
    # what a graph holds is not what an eager call takes, nor what one outgrows
    assert ops.workspace("u", 100, on).data_ptr() != first.data_ptr()
    assert ops.workspace("t", 4096, on).data_ptr() != two.data_ptr()


def test_a_device_without_an_index_is_the_current_one(fake, monkeypatch):
    def stream_of(index):
        if not isinstance(index, int):
            raise RuntimeError("a device's index is a number")
        return {0: 7, 1: 8}[index]

    monkeypatch.setattr(ops, "_raw_stream", stream_of)
    plain = ops.workspace("t", 64, torch.device("cpu"))
    assert ops.workspace("t", 64, torch.device("cpu", 0)) is plain
    fake["device"] = 1
    assert ops.workspace("t", 64, torch.device("cpu")) is not plain
    assert set(ops._ws_cache) == {("t", 0, 7), ("t", 1, 8)}
    asked = []
    monkeypatch.setattr(ops, "workspace_status", lambda ws: asked.append(ws) or 0)
    ops.check_workspace("t", torch.device("cpu", 0))
    fake["device"] = 0
    ops.check_workspace("t", torch.device("cpu"))
    ops.check_workspace("none", torch.device("cpu"))
    assert len(asked) == 2 and all(a is plain for a in asked)
