"""What `ops.workspace_status` and `ops.check_workspace` leave behind, on the CPU: the library and the stream stand in as fakes."""
import pytest
import torch

from unpopped_b200 import _lib, ops


class Library:
    def __init__(self, status):
        self.status = status

    def up_sm100_workspace_status(self, at, stream):
        return self.status

    def up_sm100_last_error(self):
        return b""


@pytest.fixture
def cached(monkeypatch):
    ws = torch.full((4096,), 3, dtype=torch.uint8)
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 7)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(ops, "_ws_cache", {("t", 0, 7): ws})
    return ws


def test_a_wait_that_ran_out_leaves_a_workspace_of_zeros(monkeypatch, cached):
    monkeypatch.setattr(_lib, "load", lambda: Library(_lib.UP_ERR_DEVICE_TIMEOUT))
    own = torch.full((300,), 5, dtype=torch.uint8)
    assert ops.workspace_status(own) == _lib.UP_ERR_DEVICE_TIMEOUT and not bool(own.any())
    with pytest.raises(_lib.UpError):
        ops.check_workspace("t", torch.device("cpu", 0))
    assert not bool(cached.any()) and ops.workspace("t", 4096, torch.device("cpu", 0)) is cached


@pytest.mark.parametrize("status", [_lib.UP_OK, _lib.UP_ERR_CUDA])
def test_any_other_status_leaves_it_as_it_is(monkeypatch, cached, status):
    monkeypatch.setattr(_lib, "load", lambda: Library(status))
    assert ops.workspace_status(cached) == status and bool((cached == 3).all())
