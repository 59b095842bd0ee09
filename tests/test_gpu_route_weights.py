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


@pytest.mark.parametrize("tokens", [70, 700])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
def test_masked_experts(tokens, score, renormalise):
    """Rows that have fewer experts than are asked for, or none."""
    g = gen(tokens)
    logits = 3 * torch.randn(tokens, 50, generator=g, device=DEV)
    logits[torch.rand(tokens, 50, generator=g, device=DEV) < 0.9] = float("-inf")
    logits[5] = float("-inf")
    logits[-tokens // 4:] = float("-inf")
    check(logits, 8, score, renormalise, 1.0 if renormalise else 2.5)


@pytest.mark.parametrize("experts,k", [(40, 8), (64, 6), (256, 8), (256, 32), (1000, 32)])
@pytest.mark.parametrize("score,renormalise", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_equal_logits(experts, k, score, renormalise):
    """More experts than a warp has lanes reach the k-th largest logit."""
    logits = torch.randint(0, 3, (150, experts), generator=gen(experts), device=DEV).float()
    logits[0] = 0.0
    logits[1] = -0.0
    logits[2, :k - 1] = 5.0
    logits[3] = torch.arange(experts, device=DEV) % 32
    logits[4] = torch.arange(experts, device=DEV) // 32
    logits[7] = float("-inf")
    logits[7, 3::7] = -20.0
    check(logits, k, score, renormalise)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("value", [-3e38, -1e30, 1e30, 3e38])
def test_logits_of_any_finite_size(score, value):
    """A row of one huge value, beside ordinary rows whose bound does not know of it."""
    logits = torch.randn(40, 30, generator=gen(7), device=DEV)
    logits[7] = value
    logits[9, 4] = value
    got = check(logits, 5, score)
    if score == "softmax" or value > 0:
        assert bool(((got[1][7] - 0.2).abs() < 1e-6).all())
