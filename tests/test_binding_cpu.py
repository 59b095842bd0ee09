"""The serving operators' Python calls as a build product (no GPU): when they are built anew, what works without them."""
import os
import sys

import pytest
import torch

from unpopped_b200 import _lib, build, ops


@pytest.fixture
def unbound(monkeypatch):
    """No binding for this Python and torch."""
    import unpopped_b200

    monkeypatch.setattr(ops, "_bound", None)
    monkeypatch.setitem(sys.modules, "unpopped_b200._bind", None)
    monkeypatch.delattr(unpopped_b200, "_bind", raising=False)


def test_dequant_needs_the_c_library_only(unbound, monkeypatch):
    seen = []

    class Library:
        def up_sm100_dequant_i4_bf16(self, *args):
            seen.append(args)
            return 0

    w, scale = torch.zeros(3, 32, dtype=torch.uint8), torch.zeros(3, 2).half()
    with pytest.raises(TypeError):  # the tensors' check, not the binding's absence
        ops.dequant_i4(w, scale, 32)
    monkeypatch.setattr(_lib, "load", Library)
    monkeypatch.setattr(ops, "_cuda", lambda t, name: None)
    monkeypatch.setattr(ops, "_stream", lambda t: 5)
    out = ops.dequant_i4(w, scale, 32)
    assert out.shape == (3, 64) and out.dtype == torch.bfloat16
    assert ops.dequant_i4(w, scale, 32, out) is out
    assert seen == [(w.data_ptr(), scale.data_ptr(), 3, 64, 32, out.data_ptr(), 5)] * 2


def test_the_serving_operators_say_what_is_missing(unbound):
    x = torch.zeros(1, 1, 32)
    for call in (lambda: ops.rope(x, None, x), lambda: ops.kv4_append(x, x, (), x), lambda: ops.kv4_attention(x, (), x, x)):
        with pytest.raises(ImportError, match="unpopped_b200.build"):
            call()


def test_the_binding_is_named_and_built_for_its_python_and_torch(tmp_path, monkeypatch):
    assert build.BIND.endswith(".so") and "cpython" in os.path.basename(build.BIND)
    made, note = tmp_path / "bind.so", tmp_path / "bind.txt"
    made.write_bytes(b"")
    monkeypatch.setattr(build, "BIND", str(made))
    monkeypatch.setattr(build, "BIND_MADE_WITH", str(note))
    cmd = build._bind_command()
    assert build._bind_stale(cmd)  # nothing says what it was made with
    note.write_text(build._bind_made_with(cmd))
    assert not build._bind_stale(cmd)
    monkeypatch.setattr(torch, "__version__", "0.0")
    assert build._bind_stale(cmd)
    note.write_text(build._bind_made_with(cmd))
    assert not build._bind_stale(cmd)
    monkeypatch.setattr(sys, "version", "4.0")
    assert build._bind_stale(cmd)


def test_without_torch_there_is_the_c_library(monkeypatch, capsys):
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name: None)
    monkeypatch.setattr(build.subprocess, "run", lambda *a, **k: pytest.fail("nothing is compiled"))
    build._build_bind()
    assert "without" in capsys.readouterr().err
