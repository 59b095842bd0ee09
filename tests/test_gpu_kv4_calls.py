"""How `ops.kv4_attention` takes its arguments."""
import numpy as np
import pytest
import torch
from kv4_exact import cache_of

from unpopped_b200 import ops

pytestmark = pytest.mark.gpu


def one():
    g = torch.Generator(device="cuda").manual_seed(3)
    cache, table = cache_of(torch.randn(2, 1, 50, 1, 64, generator=g, device="cuda"), 16, 32)
    return torch.randn(1, 4, 64, generator=g, device="cuda").half(), cache, table, torch.tensor([50], device="cuda").int()


def test_want_lse_is_any_truth_value():
    args = one()
    out, lse = ops.kv4_attention(*args, want_lse=True)
    for yes in (1, np.bool_(True), "lse"):
        got = ops.kv4_attention(*args, want_lse=yes)
        assert isinstance(got, tuple) and torch.equal(got[0], out) and torch.equal(got[1], lse)
    for no in (0, None, np.bool_(False), []):
        assert torch.equal(ops.kv4_attention(*args, want_lse=no), out)
    with pytest.raises(RuntimeError):  # a tensor of several elements has no truth value
        ops.kv4_attention(*args, want_lse=torch.ones(2))


def test_a_workspace_is_contiguous():
    """Its size is that of its elements, which a view with other strides does not have behind it."""
    args = one()
    for ws in (torch.zeros(1, dtype=torch.uint8, device="cuda").expand(64 << 20),
               torch.zeros(32 << 20, 2, dtype=torch.uint8, device="cuda")[:, 0]):
        with pytest.raises(ValueError):
            ops.kv4_attention(*args, ws=ws)
    want = ops.kv4_attention(*args)
    assert torch.equal(ops.kv4_attention(*args, ws=torch.zeros(4 << 20, dtype=torch.float32, device="cuda")), want)
