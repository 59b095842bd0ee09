"""Sizes that up_sm100_kv4_attention refuses before it launches anything (no GPU)."""
import ctypes

import pytest

from unpopped_b200 import _lib
from unpopped_b200._lib import EK, UP_ERR_UNSUPPORTED, UpKv4Cache

P = 1 << 20  # an aligned address that is never read


@pytest.mark.parametrize("batch", [(1 << 30) + 1, (1 << 31) - 100, (1 << 31) - 1])
def test_more_sequences_than_the_kernels_count(batch):
    """A block's threads share the sequences out as (batch + 127) / 128 each, in 32 bits: past 2^31 - 128 that wraps round."""
    cache = UpKv4Cache(P, P, P, P, 4, 2, 16, 64, 32)
    got = _lib.load().up_sm100_kv4_attention(P, EK["F16"], 3, 4, 256, 64, ctypes.byref(cache), P, 4, 4, P, P, batch, 1, 0, 1.0, P,
                                             256, 64, None, 4, P, 1 << 40, None)
    assert got == UP_ERR_UNSUPPORTED
