"""Routing to experts, the experts' sum, and a layer of them against their definitions in 64 bits (tests/f8_exact.py)."""
import pytest
import torch

import f8_exact as ex
from unpopped_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def check_route(logits, k, score="softmax", renormalise=True, gain=1.0):
    """Whole numbers are equal. A weight: exp (2 steps of its value and, by the f32 difference l - max, half a step of |l - max|),
    a sum of at most 1024 in 6 levels of a warp and 32 in a lane, a quotient, a product."""
    got = ops.expert_route(logits, k, score, renormalise, gain)
    want = ex.routed(logits, k, score, renormalise, gain)
    for name, a, b in zip(("ids", "weights", "rows", "slots", "offsets"), got, want):
        if name != "weights":
            assert torch.equal(a.cpu(), b), name
    w, e = got[1].double().cpu(), want[1]
    spread = logits.double().nan_to_num(0, 0, 0).abs().max().item()
    rel = (2 * spread + 60) * 2.0 ** -24
    assert bool((((w - e).abs() <= rel * e.abs() + 2.0 ** -140) | (w.isnan() & e.isnan())).all())
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score,renormalise", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("tokens,experts,k", [(1, 1, 1), (1, 128, 8), (5, 60, 6), (128, 33, 4), (129, 8, 8), (300, 256, 8), (40, 1024, 32), (200, 500, 3)])
def test_route(dtype, score, renormalise, tokens, experts, k):
    logits = (2 * torch.randn(tokens, experts, generator=gen(tokens + experts), device=DEV)).to(dtype)
    check_route(logits, k, score, renormalise, 1.0 if renormalise else 2.5)


@pytest.mark.parametrize("tokens", [1, 127, 128, 129, 256, 257, 5000])
def test_route_of_equal_logits_takes_the_lowest(tokens):
    logits = torch.randint(-2, 3, (tokens, 40), generator=gen(tokens), device=DEV).float()
    logits[logits == 0] *= -1  # zeros of both signs are equal
    logits[::3] = 1.0
    check_route(logits, 7)


@pytest.mark.parametrize("tokens", [70, 700])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_of_masked_experts(tokens, score):
    g = gen(tokens)
    logits = torch.randn(tokens, 50, generator=g, device=DEV)
    logits[torch.rand(tokens, 50, generator=g, device=DEV) < 0.9] = float("-inf")
    logits[5] = float("-inf")
    logits[-tokens // 4:] = float("-inf")
    logits[7, :] = -3e38
    _, _, rows, _, offsets = check_route(logits, 8, score)
    assert bool((rows[int(offsets[-1]):] == -1).all())
    check_route(torch.full((tokens, 50), float("-inf"), device=DEV), 8, score)


def test_route_of_values_that_are_not_finite():
    logits = torch.randn(140, 40, generator=gen(1), device=DEV)
    logits[3, 7] = float("nan")
    logits[3, 3] = float("inf")
    logits[130, 9] = logits[130, 2] = float("nan")
    ids, w, *_ = ops.expert_route(logits, 4)
    want = ex.routed(logits, 4, "softmax", True)
    assert torch.equal(ids.cpu(), want[0]) and ids[3, :2].tolist() == [7, 3] and ids[130, :2].tolist() == [2, 9]
    assert bool(w[3].isnan().all()) and bool(w[4].isfinite().all())
    logits = torch.randn(3, 40, generator=gen(2), device=DEV)
    logits[1, 4] = float("inf")
    assert ops.expert_route(logits, 2, "sigmoid", False)[1][1, 0] == 1.0


def test_route_of_many_tokens():
    """More than 256 blocks of 128 tokens: a block has several tiles."""
    logits = torch.randn(40000, 16, generator=gen(4), device=DEV)
    ids, w, rows, slots, offsets = ops.expert_route(logits, 2)
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :2]
    assert torch.equal(ids.long(), order)
    by = torch.sort(order.flatten(), stable=True).indices
    assert torch.equal(rows.long(), by // 2)
    assert torch.equal(slots.flatten()[by].long(), torch.arange(80000, device=DEV))
    assert torch.equal(offsets[1:].long(), torch.bincount(order.flatten(), minlength=16).cumsum(0))


@pytest.mark.parametrize("tokens", [63, 64, 65, 96, 97, 1000, 4736, 4737, 9473, 14209, 18944, 18945, 32768, 32769])
@pytest.mark.parametrize("experts,k", [(16, 2), (200, 8)])
def test_route_where_the_blocks_tiles_change(tokens, experts, k):
    """One launch or two, tiles of 32 to 128 tokens, blocks of one tile or more; every ninth token is padding."""
    logits = torch.randn(tokens, experts, generator=gen(tokens), device=DEV)
    logits[::9] = float("-inf")
    ids, w, rows, slots, offsets = ops.expert_route(logits, k)
    there = torch.ones(tokens, dtype=torch.bool, device=DEV)
    there[::9] = False
    top = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(ids[there].long(), top[there]) and bool((ids[~there] == -1).all()) and bool((slots[~there] == -1).all())
    pairs = int(there.sum()) * k
    flat = torch.where(there[:, None], top, experts).flatten()
    by = torch.sort(flat, stable=True).indices[:pairs]
    assert torch.equal(rows[:pairs].long(), by // k) and bool((rows[pairs:] == -1).all())
    assert torch.equal(slots.flatten()[by].long(), torch.arange(pairs, device=DEV))
    assert torch.equal(offsets[1:].long(), torch.bincount(flat, minlength=experts + 1)[:experts].cumsum(0)) and int(offsets[0]) == 0


def test_route_of_views_and_no_tokens():
    wide = torch.randn(50, 3, 64, generator=gen(6), device=DEV)
    check_route(wide[:, 1], 4)
    ids, w, rows, slots, offsets = ops.expert_route(wide[:0, 1], 4)
    assert ids.shape == (0, 4) and rows.shape == (0,) and offsets.tolist() == [0] * 65


def test_route_refusals():
    l = torch.zeros(4, 64, device=DEV)
    for call in (lambda: ops.expert_route(l, 0), lambda: ops.expert_route(l, 65), lambda: ops.expert_route(l, 2, "tanh"),
                 lambda: ops.expert_route(l.double(), 2), lambda: ops.expert_route(l.t(), 2), lambda: ops.expert_route(l[0], 1)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(_lib.UpError):
        ops.expert_route(l, 33)
    with pytest.raises(_lib.UpError):
        ops.expert_route(torch.zeros(2, 1025, device=DEV), 2)
    with pytest.raises(TypeError):
        ops.expert_route(l.cpu(), 2)


# ---- the sum ----
def check_combine(y, slots, weights, add=None, out=None):
    got = ops.expert_combine(y, slots, weights, add, out)
    there = (slots >= 0) & (slots < y.shape[0])
    picked = y.double()[slots.long().clamp(0, max(0, y.shape[0] - 1))] if y.shape[0] else torch.zeros(slots.shape + (y.shape[1],), device=DEV)
    terms = torch.where(there[..., None], picked * weights.double()[..., None], torch.zeros_like(picked, dtype=torch.float64))
    want, size = terms.sum(1), terms.abs().sum(1)
    if add is not None:
        want, size = want + add.double(), size + add.double().abs()
    steps = (slots.shape[1] + 1) * 2.0 ** -24  # one fused multiply and add a term
    off = (got.double() - want).abs()
    assert bool((off <= steps * size + ex.HALF_STEP[y.dtype] * (want.abs() + steps * size) + ex.SMALLEST[y.dtype]).all())
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,k,n", [(1, 1, 1), (1, 8, 4096), (7, 3, 130), (33, 9, 64), (40, 2, 1001), (5, 32, 8)])
@pytest.mark.parametrize("with_add", [False, True])
def test_combine(dtype, tokens, k, n, with_add):
    g = gen(n)
    rows = tokens * k
    y = torch.randn(rows, n, generator=g, device=DEV).to(dtype)
    slots = torch.randint(-1, rows + 2, (tokens, k), generator=g, device=DEV, dtype=torch.int32)
    check_combine(y, slots, torch.rand(tokens, k, generator=g, device=DEV),
                  torch.randn(tokens, n, generator=g, device=DEV).to(dtype) if with_add else None)


def test_combine_of_views_in_place_and_of_rows_that_are_left_out():
    g = gen(8)
    wide = torch.randn(30, 3, 136, generator=g, device=DEV).bfloat16()
    slots = torch.tensor([[0, 29], [-1, -1], [30, 5], [2 ** 31 - 1, -2 ** 31]], dtype=torch.int32, device=DEV)
    w = torch.tensor([[1, 2], [float("nan")] * 2, [float("nan"), 0.5], [1, 1]], device=DEV)
    add = torch.randn(4, 136, generator=g, device=DEV).bfloat16()
    y = wide[:, 1]
    w2 = torch.where(w.isnan(), torch.zeros_like(w), w)
    want = check_combine(y, slots, w2, add)
    assert torch.equal(ops.expert_combine(y, slots, w, add), want)  # weights of slots that are left out are not looked at
    assert torch.equal(want[1], add[1]) and torch.equal(want[3], add[3])
    out = add.clone()
    assert ops.expert_combine(y, slots, w, out, out) is out and torch.equal(out, want)
    odd = torch.randn(30, 137, generator=g, device=DEV).bfloat16()[:, 1:]  # rows that do not start on 16 bytes
    check_combine(odd, slots, w2, add)
    assert not bool(check_combine(y[:0], slots, w2).any())
    for bad in (dict(slots=slots.long()), dict(weights=w.double()), dict(weights=w[:2]), dict(add=add.float()), dict(add=add[:2]),
                dict(out=out[:, :8]), dict(y=y.double()), dict(y=y[0])):
        a = dict(y=y, slots=slots, weights=w2, add=None, out=None)
        a.update(bad)
        with pytest.raises(ValueError):
            ops.expert_combine(**a)


def test_offsets_that_pass_32_bits():
    """Logits and rows of more than 2^31 values."""
    tokens, experts, k = 4300000, 512, 2
    logits = torch.zeros(tokens, experts, device=DEV, dtype=torch.float16)
    logits[:, 7] = -1
    logits[-1, 500], logits[-2, 7] = 2, 3
    ids, weights, rows, slots, offsets = ops.expert_route(logits, k)
    del logits
    assert bool((ids[:-2] == torch.tensor([0, 1], device=DEV)).all()) and ids[-2:].tolist() == [[7, 0], [500, 0]]
    assert offsets[[0, 1, 2, 7, 8, 500, 501, 512]].tolist() == [0, tokens, 2 * tokens - 2, 2 * tokens - 2, 2 * tokens - 1, 2 * tokens - 1,
                                                                2 * tokens, 2 * tokens]
    assert slots[-2:].tolist() == [[2 * tokens - 2, tokens - 2], [2 * tokens - 1, tokens - 1]]
    assert torch.equal(rows[:tokens], torch.arange(tokens, device=DEV, dtype=torch.int32)) and rows[-2:].tolist() == [tokens - 2, tokens - 1]
    assert torch.equal(rows[slots.long()], torch.arange(tokens, device=DEV, dtype=torch.int32)[:, None].expand(tokens, k))
    del ids, weights, rows, slots
    g = gen(17)
    y = torch.zeros(300000, 8192, device=DEV, dtype=torch.bfloat16)
    y[-40:] = torch.randn(40, 8192, generator=g, device=DEV).bfloat16()
    slots = torch.randint(299960, 300000, (9, 3), generator=g, device=DEV, dtype=torch.int32)
    w = torch.rand(9, 3, generator=g, device=DEV)
    got = ops.expert_combine(y, slots, w)
    assert torch.equal(got, check_combine(y[-40:].clone(), slots - 299960, w))


# ---- a layer ----
def layer(x, router, up, up_s, down, down_s, k, add=None):
    ids, weights, rows, slots, offsets = ops.expert_route(torch.matmul(x.float(), router.t()), k)
    q, s = ops.f8_quantise(x, rows)
    h = ops.f8_expert_matmul(q, s, up, up_s, offsets)
    q, s = ops.f8_quantise(h, gate=True)
    return ops.expert_combine(ops.f8_expert_matmul(q, s, down, down_s, offsets), slots, weights, add)


@pytest.mark.parametrize("tokens", [1, 5, 64, 300])
def test_a_layer_of_experts(tokens):
    """The operators together, against the layer in 64 bits on the quantised weights and unquantised activations. Each activation
    is off by half a step of e4m3 (2^-4 of it, or 2^-10 of a scale that is 1/448 of its block's largest); these errors have no
    common sign, so of a sum of n terms they leave about 1/sqrt(n): the layer's 2-norm is off by at most 2^-4 for each of the two
    quantised inputs, and by three roundings to bf16."""
    e, d, f, k = 16, 512, 384, 4
    g = gen(tokens)
    x = torch.randn(tokens, d, generator=g, device=DEV).bfloat16()
    router = torch.randn(e, d, generator=g, device=DEV) / d ** 0.5
    up, up_s = ops.f8_quantise_weight(torch.randn(e, 2 * f, d, generator=g, device=DEV).bfloat16() / d ** 0.5)
    down, down_s = ops.f8_quantise_weight(torch.randn(e, d, f, generator=g, device=DEV).bfloat16() / f ** 0.5)
    got = layer(x, router, up, up_s, down, down_s, k, add=x)

    def plain(q, s):
        return q.double() * s.double().repeat_interleave(128, -1)[..., :q.shape[-1]].repeat_interleave(128, -2)[..., :q.shape[-2], :]

    u, v = plain(up, up_s), plain(down, down_s)
    logits = torch.matmul(x.float(), router.t())
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    w = torch.softmax(logits.double().gather(1, ids), 1)
    want = x.double()
    for j in range(k):
        h = torch.einsum("td,tfd->tf", x.double(), u[ids[:, j]])
        h = h[:, :f] * torch.sigmoid(h[:, :f]) * h[:, f:]
        want = want + w[:, j, None] * torch.einsum("tf,tdf->td", h, v[ids[:, j]])
    assert float((got.double() - want).norm() / (want - x.double()).norm()) <= 2 * 2.0 ** -4 + 3 * 2.0 ** -8
    # once more, captured and replayed on other tokens
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(static, router, up, up_s, down, down_s, k, add=static)
    other = torch.randn(tokens, d, generator=g, device=DEV).bfloat16()
    static.copy_(other)
    graph.replay()
    assert torch.equal(out, layer(other, router, up, up_s, down, down_s, k, add=other))


@pytest.mark.parametrize("experts,k", [(40, 8), (64, 6), (256, 8), (256, 32), (1000, 32)])
def test_route_where_more_experts_than_a_warp_has_lanes_reach_the_bound(experts, k):
    """Few distinct logits: hundreds of equal ones around the k-th, in one lane and in all of them."""
    logits = torch.randint(0, 3, (150, experts), generator=gen(experts), device=DEV).float()
    logits[0] = 0.0
    logits[1] = -0.0
    logits[2, :k - 1] = 5.0
    logits[3] = torch.arange(experts, device=DEV) % 32  # a lane's keys are equal, the lanes' differ
    logits[4] = torch.arange(experts, device=DEV) // 32
    logits[5] = float("inf")
    logits[6] = float("nan")
    logits[7] = -float("inf")
    logits[7, 3::7] = -1e30
    check_route(logits, k, "sigmoid")
    check_route(logits[:5], k, "softmax", False)


@pytest.mark.parametrize("tokens", [10, 200])
def test_a_layer_of_a_padded_batch(tokens):
    """Padded tokens have no experts: their rows are the residual, and the others are what they are alone."""
    e, d, f, k = 8, 256, 128, 3
    g = gen(tokens)
    x = torch.randn(tokens, d, generator=g, device=DEV).bfloat16()
    x[tokens // 2:] = float("nan")  # what lies in padded rows is not looked at
    logits = torch.randn(tokens, e, generator=g, device=DEV)
    logits[tokens // 2:] = float("-inf")
    up, up_s = ops.f8_quantise_weight(torch.randn(e, 2 * f, d, generator=g, device=DEV).bfloat16())
    down, down_s = ops.f8_quantise_weight(torch.randn(e, d, f, generator=g, device=DEV).bfloat16())

    def run(x, logits, add):
        ids, weights, rows, slots, offsets = ops.expert_route(logits, k)
        h = ops.f8_expert_matmul(*ops.f8_quantise(x, rows), up, up_s, offsets)
        y = ops.f8_expert_matmul(*ops.f8_quantise(h, gate=True), down, down_s, offsets)
        return ops.expert_combine(y, slots, weights, add)

    add = torch.randn(tokens, d, generator=g, device=DEV).bfloat16()
    out, n = run(x, logits, add), tokens // 2
    assert torch.equal(out[n:], add[n:]) and bool(out.isfinite().all())
    want = run(x[:n], logits[:n], add[:n])
    # With other counts of rows tiles may be split elsewhere and sums be added in another order: a code of h may then be its neighbour, 2^-3 of
    # one of 128 terms of no common sign, 2^-3 / sqrt(128) = 2^-6.5 of a row's size
    assert bool(((out[:n].double() - want.double()).abs() <= want.double().abs() * 2.0 ** -6 + 2.0 ** -6 * want.double().abs().max()).all())


def test_combine_of_no_slots():
    add = torch.randn(5, 24, generator=gen(1), device=DEV).bfloat16()
    y = torch.randn(3, 24, generator=gen(2), device=DEV).bfloat16()
    none, w = torch.empty(5, 0, dtype=torch.int32, device=DEV), torch.empty(5, 0, device=DEV)
    assert torch.equal(ops.expert_combine(y, none, w, add), add) and not bool(ops.expert_combine(y, none, w).any())
