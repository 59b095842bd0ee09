"""8-bit products whose two scales are far apart, or both far from 1: their product leaves f32 where the result need not."""
import pytest
import torch

import f8_exact as ex
import f8_walk
from unpopped_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
# few rows, rows of 128 x 128 tiles, of 128 x 256 ones and of pairs; tiles that are shared, and a last block of k that is short
SHAPES = [(1, 200, 400), (21, 384, 4096), (40, 300, 272), (300, 1000, 528), (600, 4096, 1040), (300, 300, 8192), (1100, 4096, 528), (384, 4096, 4096), (513, 2051, 8192),
          (1100, 4111, 8208), (2000, 2051, 8208)]


def test_the_shapes_take_every_form():
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert {f8_walk.form(m, n, k, 1, sms) for m, n, k in SHAPES} == set(f8_walk.FORMS)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def near(g, exponent, *shape):
    return ((1 + torch.rand(*shape, generator=g, device=DEV, dtype=torch.float64)) * 2.0 ** exponent).float()


def check(got, x, xs, w, ws):
    """The bound of every product, and for each block some halves of f32's smallest number for the roundings below its normal ones. Where the definition
    is beyond the type it is infinite."""
    want, size = ex.product(x, xs, w, ws)
    bound = ex.product_bound(want, size, x.shape[1], got.dtype) + ex.blocks(x.shape[1]) * 2.0 ** -148
    off = (got.double() - want).abs()
    good = off <= bound
    good |= got.isinf() & (got.sign() == want.sign()) & (want.abs() + bound >= torch.finfo(got.dtype).max)
    assert bool(good.all()), (int((~good).sum()), float((off / bound)[~good].nan_to_num(-1).max()))


def codes(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV).mul_(150).clamp_(-448, 448).to(ex.F8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("low", [(-70, -72), (-20, -122), (-126, -16), (-10, -140)])
def test_a_product_of_scales_below_f32s_normal_numbers(m, n, k, dtype, low):
    """x * w is a few bits of 2^-149, v * x * w some 2^-120."""
    g = gen(m)
    x, w = codes(g, m, k), codes(g, n, k)
    xs, ws = near(g, low[0], m, ex.blocks(k)), near(g, low[1], ex.blocks(n), ex.blocks(k))
    xs[::3] = near(g, 0, *xs[::3].shape)  # among rows whose product is an ordinary number
    xs[1::5] = 0
    check(ops.f8_matmul(x, xs, w, ws, dtype=dtype), x, xs, w, ws)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("high", [(66, 64), (4, 126), (126, 5)])
def test_a_product_of_scales_above_f32(m, n, k, dtype, high):
    """x * w is above 2^128; a block's sum of few products of 2^-9 by 2^-9 is below 2^-15, and often 0."""
    g = gen(k)
    x, w = (torch.zeros(s, k, device=DEV) for s in (m, n))
    x[:, ::7], w[:, ::14] = 2.0 ** -9, -2.0 ** -9
    x[:, 128:256] = 0
    x, w = x.to(ex.F8), w.to(ex.F8)
    xs, ws = near(g, high[0], m, ex.blocks(k)), near(g, high[1], ex.blocks(n), ex.blocks(k))
    xs[1::3] = near(g, -high[1], *xs[1::3].shape)
    xs[2::5] = 0
    got = ops.f8_matmul(x, xs, w, ws, dtype=dtype)
    check(got, x, xs, w, ws)
    assert bool(got.isfinite().all())


@pytest.mark.parametrize("m,n,k", [(21, 384, 4096), (200, 2048, 2048), (600, 4096, 2064), (1100, 4096, 2064), (300, 300, 8192)])
@pytest.mark.parametrize("where", [[3], [0, 9], [14, 15]])
def test_single_blocks_of_such_scales(m, n, k, where):
    """Of blocks whose other scales, or codes, are 0."""
    g = gen(n)
    x, w = codes(g, m, k), codes(g, n, k)
    xs, ws = torch.zeros(m, ex.blocks(k), device=DEV), near(g, -75, ex.blocks(n), ex.blocks(k))
    xs[:, where] = near(g, -70, m, len(where))
    xs[5], xs[9] = near(g, 60, ex.blocks(k)), 0
    check(ops.f8_matmul(x, xs, w, ws, dtype=torch.float32), x, xs, w, ws)


def test_by_expert_of_scales_far_apart():
    g = gen(9)
    sizes = torch.tensor([0, 5, 0, 140, 1, 33, 300, 0])
    m, n, k = int(sizes.sum()), 264, 656
    offsets = torch.zeros(9, dtype=torch.int32)
    offsets[1:] = sizes.cumsum(0)
    x, w = codes(g, m, k), codes(g, 8, n, k)
    xs, ws = near(g, -60, m, ex.blocks(k)), near(g, -83, 8, ex.blocks(n), ex.blocks(k))
    got = ops.f8_expert_matmul(x, xs, w, ws, offsets.to(DEV), dtype=torch.float32)
    for e in range(8):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        check(got[lo:hi], x[lo:hi], xs[lo:hi], w[e], ws[e]) if hi > lo else None


def test_scales_that_are_not_finite():
    """An infinite scale gives infinities or NaN in its rows only, a NaN NaN."""
    g = gen(10)
    for m, n, k in SHAPES[1:4]:
        x, w = codes(g, m, k), codes(g, n, k)
        xs, ws = near(g, 0, m, ex.blocks(k)), near(g, 0, ex.blocks(n), ex.blocks(k))
        want = ops.f8_matmul(x, xs, w, ws, dtype=torch.float32)
        xs = xs.clone()
        xs[3, 1], xs[7, 0] = float("inf"), float("nan")
        got = ops.f8_matmul(x, xs, w, ws, dtype=torch.float32)
        assert not bool(got[3].isfinite().any()) and bool(got[7].isnan().all())
        keep = torch.ones(m, dtype=torch.bool, device=DEV)
        keep[[3, 7]] = False
        assert torch.equal(got[keep], want[keep])
