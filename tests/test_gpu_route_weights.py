"""The weights of routing, each held to a bound of its own row's logits."""
import pytest
import torch

import f8_exact as ex
from unpopped_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
STEP = 2.0 ** -24  # half a step of f32
ZERO = -104.0      # exp of less rounds to 0 in f32


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def check(logits, k, score="softmax", renormalise=True, gain=1.0):
    """Whole numbers are equal. A weight's half steps: four of an exponential (2 steps) and, by a rounded difference from the row's largest
    logit, as many as that difference, 104 at most, below which exp is 0; both once more for the sum; its additions (31 in a lane and 5 over the
    lanes of all experts, 5 of the chosen); of a sigmoid its sum and quotient, twice; the quotient and the product by gain. Results below 2^-126 are
    multiples of 2^-149: some of these, 2^-146."""
    got = ops.expert_route(logits, k, score, renormalise, gain)
    want = ex.routed(logits, k, score, renormalise, gain)
    for name, a, b in zip(("ids", "weights", "rows", "slots", "offsets"), got, want):
        if name != "weights":
            assert torch.equal(a.cpu(), b), name
    l, ids = logits.double().cpu(), want[0].long()
    chosen = l.gather(1, ids.clamp(min=0)).masked_fill(ids < 0, float("nan"))
    seen = chosen if renormalise else torch.where(l == float("-inf"), torch.full_like(l, float("nan")), l)
    top = seen.nan_to_num(-1e300).amax(1, keepdim=True)
    far = (top - seen).nan_to_num(0).amax(1, keepdim=True).clamp(max=104)
    if score == "sigmoid":
        far = torch.where((top < 0) & torch.tensor(renormalise), far, torch.zeros_like(far))
    halves = 2 * (far + 4) + (5 if renormalise else 36) + 4 + 2
    rel = halves * STEP
    assert float(rel.max()) < 1e-4
    expected = want[1]
    if score == "sigmoid":  # scores are f32's: where the largest is 0 there are no shares
        expected = torch.where((top < ZERO) if renormalise else (chosen < ZERO), torch.zeros_like(expected), expected)
    off = (got[1].double().cpu() - expected).abs()
    assert bool((off <= rel * expected.abs() + 2.0 ** -146 * max(1.0, gain)).all()), float((off / (rel * expected.abs() + 2.0 ** -146)).max())
    return got


@pytest.mark.parametrize("tokens", [9, 200])
@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("low", [-60, -80, -87, -88.5, -89, -95, -102])
def test_a_sigmoid_of_logits_far_below_0(low, renormalise, tokens):
    """Scores that are no normal numbers in f32, whose shares are ordinary ones; single rows have larger logits too."""
    logits = low + torch.rand(tokens, 40, generator=gen(tokens), device=DEV)
    logits[3::7] -= 10 * torch.rand(len(logits[3::7]), 40, generator=gen(1), device=DEV)
    logits[3::7, 0] = low + 1
    logits[1, 5], logits[2, 5] = -30.0, 2.0
    got = check(logits, 4, "sigmoid", renormalise)
    assert bool((got[1].sum(1) - 1).abs().max() < 1e-5) or not renormalise


@pytest.mark.parametrize("low", [-106, -800, -1e30])
def test_a_sigmoid_of_logits_whose_scores_are_0(low):
    logits = torch.full((70, 20), float(low), device=DEV)
    logits[1, 3], logits[2, 4] = -5.0, 3.0
    got = check(logits, 3, "sigmoid")
    assert not bool(got[1][3:].any()) and float(got[1][1, 0]) == 1 and bool((got[1][1:3, 1:] < 2.0 ** -140).all())  # exp(-101) is 10 times 2^-149
    check(logits, 3, "sigmoid", False, 2.0)
