"""Rotary positions on the GPU (`ops.rope`, `rope_backward`, `rope_table`) against a plain implementation in 64 bits.

Bound of a rotated value: two products and a sum, each rounded to f32 (u = 2^-24), then the type's rounding:
|got - exact| <= 3u (|x0 c| + |x1 s|) + half an ulp of the type. Copied dimensions are equal bit for bit."""
import math

import pytest
import torch

from unpopped_b200 import _lib, ops

pytestmark = pytest.mark.gpu
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


def table_of(n, rot, dev="cuda"):
    f = 10000.0 ** (-torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / max(rot, 1))
    a = torch.arange(n, device=dev, dtype=torch.float64)[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float().reshape(n, rot)


def exact(x, pos, table, layout, sign=1.0):
    """(values, error bound before the final rounding) of x [..., heads, dim] at pos [...], in 64 bits."""
    rot = table.shape[1]
    y = x.double().clone()
    bound = torch.zeros_like(y)
    c, s = table.double()[pos][..., None, :rot // 2], sign * table.double()[pos][..., None, rot // 2:]
    i = torch.arange(rot // 2, device=x.device)
    a, b = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
    x0, x1 = y[..., a], y[..., b]
    bound[..., a] = (x0 * c).abs() + (x1 * s).abs()
    bound[..., b] = (x1 * c).abs() + (x0 * s).abs()
    y[..., a], y[..., b] = x0 * c - x1 * s, x1 * c + x0 * s
    return y, bound * 3 * 2.0 ** -24


def check(got, x, pos, table, layout, sign=1.0):
    want, bound = exact(x, pos, table, layout, sign)
    rot = table.shape[1]
    assert torch.equal(got[..., rot:], x[..., rot:])
    off = (got.double() - want).abs()
    assert bool((off <= bound + want.abs() * HALF_ULP[x.dtype] * 1.001 + TINY[x.dtype]).all()), float(off.max())


@pytest.mark.parametrize("kind", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,dim,rot", [(1, 1, 2, 2), (1, 64, 128, 128), (7, 3, 80, 80), (33, 5, 96, 32),
                                                  (130, 2, 64, 0), (19, 3, 7, 6), (5, 2, 100, 20), (257, 9, 256, 128)])
def test_forward_and_gradient_match_64_bits(kind, layout, tokens, heads, dim, rot):
    g = torch.Generator(device="cuda").manual_seed(tokens * 1000 + dim)
    x = torch.randn(tokens, heads, dim, generator=g, device="cuda").to(kind)
    pos = torch.randint(0, 500, (tokens,), generator=g, device="cuda")
    table = table_of(500, rot)
    check(ops.rope(x, pos, table, layout), x, pos, table, layout)
    check(ops.rope(x, pos.int(), table, layout), x, pos, table, layout)
    check(ops.rope_backward(x, pos, table, layout), x, pos, table, layout, -1.0)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient_matches_differences(layout):
    """The map is linear, so <g, rope(x + h e) - rope(x)> / h is the gradient's element up to f32 rounding of a few
    units of |g| |x| 2^-24 / h; with h = 1 and values of order 1 that is below 2^-18."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(3, 2, 24, generator=g, device="cuda")
    grad = torch.randn(3, 2, 24, generator=g, device="cuda")
    pos = torch.tensor([0, 17, 499], device="cuda")
    table = table_of(500, 16)
    dx = ops.rope_backward(grad, pos, table, layout)
    base = ops.rope(x, pos, table, layout).double()
    for t, h, d in [(0, 0, 0), (1, 1, 1), (2, 0, 8), (2, 1, 15), (1, 0, 16), (0, 1, 23), (1, 1, 7)]:
        e = x.clone()
        e[t, h, d] += 1.0
        step = e[t, h, d].double() - x[t, h, d].double()
        diff = ((ops.rope(e, pos, table, layout).double() - base) * grad.double()).sum() / step
        assert abs(float(diff - dx[t, h, d].double())) <= 2.0 ** -18


def test_gain_scales_the_gradient_too():
    x = torch.randn(4, 2, 32, device="cuda")
    pos = torch.arange(4, device="cuda")
    table = ops.rope_table(8, 32, gain=1.25)
    check(ops.rope(x, pos, table), x, pos, table, "half")
    check(ops.rope_backward(x, pos, table), x, pos, table, "half", -1.0)


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_strides_batches_and_in_place(kind):
    table = table_of(64, 32)
    packed = torch.randn(3, 10, 12, 64, device="cuda").to(kind)  # [batch, seq, heads of q, k and v, dim]
    q = packed[:, :, 2:7]
    pos = torch.randint(0, 64, (3, 10), device="cuda")
    want = ops.rope(q.contiguous(), pos, table)
    check(want, q, pos, table, "half")
    assert torch.equal(ops.rope(q, pos, table), want)
    # heads before tokens
    hm = q.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    out = torch.empty(3, 5, 10, 64, device="cuda", dtype=kind).permute(0, 2, 1, 3)
    assert torch.equal(ops.rope(hm, pos, table, out=out), want)
    # an odd row stride, and rows that are not 16-byte aligned
    odd = torch.empty(3, 10, 5, 67, device="cuda", dtype=kind)[..., 1:65]
    odd.copy_(q)
    assert torch.equal(ops.rope(odd, pos, table), want)
    # one row of positions for all sequences, and none
    one = pos[1].contiguous()
    assert torch.equal(ops.rope(q, one, table), ops.rope(q.contiguous(), one.expand(3, 10).contiguous(), table))
    seq = torch.arange(10, device="cuda")
    assert torch.equal(ops.rope(q, None, table), ops.rope(q, seq, table))
    # in place, leaving the neighbours alone
    before = packed.clone()
    assert ops.rope(q, pos, table, out=q).data_ptr() == q.data_ptr()
    assert torch.equal(q, want)
    assert torch.equal(packed[:, :, :2], before[:, :, :2]) and torch.equal(packed[:, :, 7:], before[:, :, 7:])


def test_a_position_outside_the_table_gives_nan_there_only():
    table = table_of(8, 16)
    for dim in (32, 18):  # the vector and the general kernel
        x = torch.randn(4, 2, dim, device="cuda")
        y = ops.rope(x, torch.tensor([0, -1, 8, 7], device="cuda"), table)
        assert bool(y[1:3, :, :16].isnan().all())
        assert torch.equal(y[:, :, 16:], x[:, :, 16:])
        check(y[[0, 3]], x[[0, 3]], torch.tensor([0, 7], device="cuda"), table, "half")


def test_empty_and_another_stream():
    table = table_of(8, 16)
    assert ops.rope(torch.empty(0, 4, 32, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"),
                    table).shape == (0, 4, 32)
    x = torch.randn(300, 8, 32, device="cuda")
    pos = torch.arange(300, device="cuda") % 8
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = ops.rope(x, pos, table)
    torch.cuda.current_stream().wait_stream(s)
    check(y, x, pos, table, "half")


def test_refusals():
    table = table_of(8, 16)
    x = torch.randn(4, 2, 32, device="cuda")
    pos = torch.arange(4, device="cuda")
    for bad in (lambda: ops.rope(x.double(), pos, table), lambda: ops.rope(x[0], pos, table),
                lambda: ops.rope(x.transpose(1, 2), pos, table), lambda: ops.rope(x, pos[:3], table),
                lambda: ops.rope(x, pos.float(), table), lambda: ops.rope(x, pos, table.double()),
                lambda: ops.rope(x, pos, table.t()), lambda: ops.rope(x, pos, table, out=x[:2]),
                lambda: ops.rope(x, pos.cpu(), table)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        ops.rope(x.cpu(), pos, table)
    with pytest.raises(KeyError):
        ops.rope(x, pos, table, "thirds")
    with pytest.raises(_lib.UpError):  # a rotation wider than the head
        ops.rope(x, pos, table_of(8, 64))
    with pytest.raises(_lib.UpError):  # an odd one
        ops.rope(x, pos, torch.zeros(8, 15, device="cuda"))
    with pytest.raises(_lib.UpError):  # output rows that overlap
        ops.rope(x, pos, table, out=torch.empty(1, 1, 32, device="cuda").expand(4, 2, 32))


def frequencies(rot, base, scaling):
    f = []
    for i in range(rot // 2):
        b = base
        if scaling and scaling[0] == "base" and rot > 2:
            b = base * scaling[1] ** (rot / (rot - 2))
        v = b ** (-2 * i / rot)
        if scaling and scaling[0] == "linear":
            v /= scaling[1]
        if scaling and scaling[0] in ("wavelength", "ramp"):
            kind, factor, low, high, orig = scaling
            if kind == "wavelength":
                w = 2 * math.pi / v
                t = min(max((orig / w - low) / (high - low), 0.0), 1.0)
            else:
                at = [rot * math.log(orig / (2 * math.pi * n)) / (2 * math.log(base)) for n in (high, low)]
                lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
                t = 1.0 - min(max((i - lo) / ((hi - lo) or 0.001), 0.0), 1.0)
            v = (1 - t) * v / factor + t * v
        f.append(v)
    return torch.tensor(f, dtype=torch.float64, device="cuda")


@pytest.mark.parametrize("rot", [2, 20, 128])
@pytest.mark.parametrize("scaling", [None, ("linear", 4.0), ("base", 8.0), ("wavelength", 8.0, 1.0, 4.0, 8192),
                                     ("ramp", 16.0, 1.0, 32.0, 4096)])
def test_table(rot, scaling):
    """f64 throughout: an angle of up to 4095 has an f64 error below 2^-38, so f32 rounding (2^-24 of at most the gain)
    decides; the two sides may round a tie apart."""
    got = ops.rope_table(4096, rot, 500000.0, scaling, gain=1.5)
    a = torch.arange(4096, device="cuda", dtype=torch.float64)[:, None] * frequencies(rot, 500000.0, scaling)
    want = 1.5 * torch.cat([a.cos(), a.sin()], 1)
    assert float((got.double() - want).abs().max()) <= 1.5 * 2.0 ** -24


def test_table_refusals():
    for scaling in (("linear",), ("cubic", 2.0), ("ramp", 2.0)):
        with pytest.raises(ValueError):
            ops.rope_table(8, 16, scaling=scaling)
    for kw in (dict(rot=15), dict(rot=16, base=1.0), dict(rot=16, scaling=("linear", 0.0)),
               dict(rot=16, scaling=("wavelength", 2.0, 4.0, 1.0, 8192))):
        with pytest.raises(_lib.UpError):
            ops.rope_table(8, **kw)
