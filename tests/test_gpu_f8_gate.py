"""The gate of f8_quantise to f32's precision: silu(x) * u by f32's own exponential and quotient."""
import pytest
import torch

import f8_exact as ex
from unpopped_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
STEP = 2.0 ** -24  # half a step of f32


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def gates(seed, tokens, k, spread, dtype):
    g = gen(seed)
    x = torch.randn(tokens, 2 * k, generator=g, device=DEV)
    x[:, :k] *= spread
    x[:, k:] *= torch.exp(torch.randn(tokens, 1, generator=g, device=DEV))
    return x.to(dtype)


def off_by(q, s, y, rel):
    """Whether scales and values are those of y, known to `rel` of itself. A scale has two roundings more; a code divides by it with two more again, so
    it is y / scale to 2 rel and four roundings, and half a step of 2^-4 of e4m3 (of 2^-10 below 2^-6)."""
    k = y.shape[1]
    pad = torch.nn.functional.pad(y, (0, -k % 128)).unflatten(1, (-1, 128))
    want = pad.abs().amax(2) / 448
    assert bool(((s.double() - want).abs() <= want * (rel + 2 * STEP)).all())
    v = y / want.repeat_interleave(128, 1)[:, :k]
    off = (q.double() - v).abs()
    assert bool((off <= (v.abs() * 2.0 ** -4).clamp(min=2.0 ** -10) + v.abs() * (2 * rel + 4 * STEP)).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,k,spread", [(1, 16, 1), (7, 400, 3), (33, 2048, 1), (33, 2048, 6), (300, 1040, 20)])
def test_the_gate_is_within_f32s_roundings(dtype, tokens, k, spread):
    """exp to 2 steps (4 half steps), weighed with e / (1 + e); the sum, the quotient and the product by u half a step each."""
    x = gates(k, tokens, k, spread, dtype)
    q, s = ops.f8_quantise(x, gate=True)
    d = x.double()
    off_by(q, s, d[:, :k] * torch.sigmoid(d[:, :k]) * d[:, k:], 7 * STEP)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("spread", [1, 8, 30])
def test_the_gate_is_the_f32_formula_bit_for_bit(dtype, spread):
    """x / (1 + exp(-x)) * u in f32, wherever exp(-x) is a number."""
    x = gates(spread, 200, 1040, spread, dtype).clamp(min=-88)
    q, s = ops.f8_quantise(x, gate=True)
    f = x.float()
    y = f[:, :1040] / (1 + (-f[:, :1040]).exp()) * f[:, 1040:]
    wq, ws = ex.quantised(y)
    assert torch.equal(s, ws) and torch.equal(q.float(), wq.float())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_gate_where_exp_leaves_f32(dtype):
    """From -88.7 down 1 / (1 + exp(-x)) goes by halves of the exponential: 2 steps of each (8 half steps), three products."""
    g = gen(3)
    x = torch.empty(64, 256, device=DEV)
    x[:, :128] = torch.linspace(-108, -86, 64, device=DEV)[:, None] - torch.rand(64, 128, generator=g, device=DEV)
    x[:, 128:] = torch.randn(64, 128, generator=g, device=DEV).sign() * (1 + torch.rand(64, 128, generator=g, device=DEV)) * 1e37
    x = x.to(dtype)
    q, s = ops.f8_quantise(x, gate=True)
    d = x.double()
    off_by(q, s, d[:, :128] * torch.sigmoid(d[:, :128]) * d[:, 128:], 11 * STEP)


def test_the_gate_of_values_that_are_not_finite():
    """As the formula's: an infinite or NaN y is NaN in its place only."""
    x = torch.randn(5, 256, generator=gen(4), device=DEV)
    x[0, 3], x[1, 4], x[2, 5], x[3, 130] = float("inf"), float("-inf"), float("nan"), float("inf")
    q, s = ops.f8_quantise(x, gate=True)
    y = x[:, :128] / (1 + (-x[:, :128]).exp()) * x[:, 128:]
    wq, ws = ex.quantised(y)
    assert torch.equal(s, ws) and torch.equal(q.float().nan_to_num(-1), wq.float().nan_to_num(-1))
    assert [int(r.isnan().sum()) for r in q.float()] == [1, 1, 1, 1, 0]


@pytest.mark.parametrize("dtype", TYPES)
def test_the_gate_of_gathered_rows_with_values_far_below_0(dtype):
    """Rows by number, some of them none, of a wider tensor; here and there an x below -88.7 among ordinary ones."""
    g = gen(5)
    x = torch.randn(9, 2, 2 * 272, generator=g, device=DEV)
    x[:, :, 3:272:31] = -100 * torch.rand(9, 2, 9, generator=g, device=DEV) - 60
    x = x.to(dtype)[:, 1]
    rows = torch.tensor([8, 0, -1, 9, 3, 3, 2 ** 31 - 1, -2 ** 31, 7], dtype=torch.int32, device=DEV)
    q, s = ops.f8_quantise(x, rows, gate=True)
    keep = (rows >= 0) & (rows < 9)
    all_q, all_s = ops.f8_quantise(x.contiguous(), gate=True)
    at = rows[keep].long()
    assert torch.equal(q[keep].float(), all_q.float()[at]) and torch.equal(s[keep], all_s[at])
    assert not bool(q[~keep].float().any()) and not bool(s[~keep].any())
    d = x.double()
    off_by(all_q, all_s, d[:, :272] * torch.sigmoid(d[:, :272]) * d[:, 272:], 11 * STEP)
