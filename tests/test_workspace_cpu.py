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
