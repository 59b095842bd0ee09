"""examples/decode_4bit.py: the serving operators run together as a decoding loop."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def test_prompts_at_once_and_token_by_token_give_the_same_logits():
    """A prompt fed whole and one token a step write the same cache and see the same tokens; what differs is the rounding
    of the probabilities (to f16, against references that differ) and of the bf16 activations that follow from it:
    measured against the logits' norm, a few bf16 units (2^-8) over the 2 layers' six roundings."""
    import decode_4bit as ex

    model = ex.Model()
    prompts = [list(range(5, 45)), [7], list(range(100, 117))]
    whole = ex.step(model, ex.Sequences(model, 3), prompts).float()
    one = ex.Sequences(model, 3)
    last = [None] * 3
    for t in range(40):
        feed = [p[t:t + 1] for p in prompts]
        logits = ex.step(model, one, feed).float()
        for b, f in enumerate(feed):
            if f:
                last[b] = logits[b]
    got = torch.stack(last)
    assert bool(torch.isfinite(whole).all())
    assert float((got - whole).norm() / whole.norm()) <= 6 * 2.0 ** -8


def test_generation_is_reproducible():
    import decode_4bit as ex

    model = ex.Model()
    prompts = [[1], list(range(30)), [3, 4, 5]]
    first = ex.generate(model, prompts, 6)
    assert ex.generate(model, prompts, 6) == first and all(len(t) == 6 for t in first)
