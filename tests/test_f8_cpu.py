"""The 8-bit operators' and the experts' C entries without a GPU: what they refuse before any launch, their interfaces, and the
definitions that the GPU tests compare with."""
import ctypes
import os
import re

import numpy as np
import pytest
import torch

import f8_exact as ex
from unpopped_b200 import _lib, build
from unpopped_b200.interface import kernel_interface

EK, P = _lib.EK, 1 << 20  # a 16-byte aligned address that no refused call touches
OK, INVALID, UNSUPPORTED = _lib.UP_OK, _lib.UP_ERR_INVALID, _lib.UP_ERR_UNSUPPORTED


@pytest.fixture(scope="module")
def L():
    return _lib.load()


def quantise(L, **change):
    a = dict(x=P, dtype=EK["BF16"], tokens=4, stride=256, rows=None, n=4, k=256, gate=0, q=P, scale=P, sr=1, sb=4)
    a.update(change)
    return L.up_sm100_f8_quantise(*a.values(), None)


@pytest.mark.parametrize("change,status", [
    (dict(tokens=-1), INVALID), (dict(n=5), INVALID), (dict(dtype=EK["F64"]), UNSUPPORTED), (dict(dtype=EK["FP8_E4M3FN"]), UNSUPPORTED),
    (dict(k=264, stride=264), UNSUPPORTED), (dict(x=None), INVALID), (dict(q=None), INVALID), (dict(scale=None), INVALID),
    (dict(stride=240), INVALID), (dict(gate=1), INVALID), (dict(x=P + 8), UNSUPPORTED), (dict(stride=260), UNSUPPORTED),
    (dict(q=P + 8), UNSUPPORTED), (dict(sr=-1), INVALID), (dict(k=1 << 31, stride=1 << 31), UNSUPPORTED),
    (dict(tokens=0, n=0), OK), (dict(k=0, stride=0), OK),
])
def test_quantise_refusals(L, change, status):
    assert quantise(L, **change) == status


def weight(L, **change):
    a = dict(w=P, dtype=EK["F16"], experts=2, n=130, k=144, se=130 * 144, sn=144, q=P, scale=P)
    a.update(change)
    return L.up_sm100_f8_quantise_weight(*a.values(), None)


@pytest.mark.parametrize("change,status", [
    (dict(experts=-1), INVALID), (dict(dtype=EK["I8"]), UNSUPPORTED), (dict(k=136), UNSUPPORTED), (dict(sn=128), INVALID),
    (dict(sn=148), UNSUPPORTED), (dict(se=130 * 144 + 4), UNSUPPORTED), (dict(w=P + 8), UNSUPPORTED), (dict(w=None), INVALID),
    (dict(experts=1 << 31), UNSUPPORTED), (dict(n=0), OK), (dict(experts=0), OK),
])
def test_quantise_weight_refusals(L, change, status):
    assert weight(L, **change) == status


def matmul(L, **change):
    a = dict(x=P, m=4, stride=256, xs=P, xm=1, xb=4, w=P, ws=P, experts=1, n=130, k=256, offsets=None, out=P, dtype=EK["BF16"], os=130,
             space=P, bytes=1 << 40)
    a.update(change)
    return L.up_sm100_f8_matmul(*a.values(), None)


@pytest.mark.parametrize("change,status", [
    (dict(m=-1), INVALID), (dict(experts=0), INVALID), (dict(experts=2), INVALID), (dict(experts=1025, offsets=P), UNSUPPORTED),
    (dict(k=0), UNSUPPORTED), (dict(k=264, stride=272), UNSUPPORTED), (dict(dtype=EK["F64"]), UNSUPPORTED), (dict(stride=240), INVALID),
    (dict(stride=264), UNSUPPORTED), (dict(x=P + 8), UNSUPPORTED), (dict(w=P + 8), UNSUPPORTED), (dict(os=129), INVALID),
    (dict(x=None), INVALID), (dict(xs=None), INVALID), (dict(w=None), INVALID), (dict(ws=None), INVALID), (dict(out=None), INVALID),
    (dict(space=None), INVALID), (dict(xm=-1), INVALID), (dict(m=1 << 31), UNSUPPORTED), (dict(n=1 << 31, os=1 << 31), UNSUPPORTED),
    (dict(n=1 << 29, os=1 << 29, k=1 << 20, stride=1 << 20), UNSUPPORTED), (dict(m=0), OK), (dict(n=0, os=0), OK),
])
def test_matmul_refusals(L, change, status):
    assert matmul(L, **change) == status


def route(L, **change):
    a = dict(l=P, dtype=EK["F32"], tokens=4, experts=64, stride=64, k=2, score=0, renormalise=1, gain=1.0, ids=P, weights=P, rows=P, slots=P,
             offsets=P, space=P, bytes=1 << 40)
    a.update(change)
    return L.up_sm100_expert_route(*a.values(), None)


@pytest.mark.parametrize("change,status", [
    (dict(tokens=-1), INVALID), (dict(experts=0, k=0), INVALID), (dict(k=0), INVALID), (dict(k=65), INVALID), (dict(k=33), UNSUPPORTED),
    (dict(experts=1025, stride=1025), UNSUPPORTED), (dict(stride=63), INVALID), (dict(score=2), INVALID), (dict(dtype=EK["I32"]), UNSUPPORTED),
    (dict(tokens=1 << 31), UNSUPPORTED), (dict(l=None), INVALID), (dict(ids=None), INVALID), (dict(offsets=None), INVALID),
    (dict(space=P + 16), INVALID), (dict(tokens=1000, bytes=256), INVALID),
])
def test_route_refusals(L, change, status):
    assert route(L, **change) == status


def combine(L, **change):
    a = dict(y=P, dtype=EK["BF16"], rows=8, ys=64, n=64, slots=P, weights=P, tokens=4, k=2, add=None, adds=0, out=P, os=64)
    a.update(change)
    return L.up_sm100_expert_combine(*a.values(), None)


@pytest.mark.parametrize("change,status", [
    (dict(rows=-1), INVALID), (dict(dtype=EK["I32"]), UNSUPPORTED), (dict(y=None), INVALID), (dict(out=None), INVALID), (dict(slots=None), INVALID),
    (dict(ys=63), INVALID), (dict(os=63), INVALID), (dict(add=P, adds=63), INVALID), (dict(k=-1), INVALID), (dict(tokens=0), OK), (dict(n=0), OK),
])
def test_combine_refusals(L, change, status):
    assert combine(L, **change) == status


@pytest.mark.parametrize("name", ["F8_QUANTISE", "F8_MATMUL", "EXPERT_ROUTE", "EXPERT_COMBINE"])
def test_interfaces(name):
    ki = kernel_interface(_lib.SERVING_KERNEL[name])
    assert hasattr(_lib.load(), ki.entry_symbol) and ki.entry_symbol in _lib.SIGNATURES
    source = {"F8_QUANTISE": "f8_quantise.cu", "F8_MATMUL": "f8_matmul.cu"}.get(name, "experts.cu")
    assert ki.revision_hash == build.revision_hash(os.path.join(build.CSRC, source))


def test_a_workspaces_counters_are_what_is_to_be_zeroed():
    with open(os.path.join(build.ROOT, "include", "up_sm100.h")) as f:
        counters = int(re.search(r"#define UP_F8_COUNTER_BYTES (\d+)", f.read()).group(1))
    assert counters == 8192 and _lib.load().up_sm100_f8_matmul_workspace_bytes(0, 1, 8, 8) == counters


def test_a_plan_never_lowers_to_them():
    L = _lib.load()
    for kernel in _lib.SERVING_KERNEL.values():
        assert L.up_sm100_launch(kernel, None, 0, None, 0, None, 0, None, 0, None) != OK


# ---- the definitions that the GPU tests use, against numbers worked out by hand ----
def test_the_definition_of_the_product():
    x = torch.zeros(2, 144)
    x[0, 0], x[0, 130], x[1, 128] = 2.0, 3.0, 0.5
    w = torch.zeros(130, 144)
    w[0, 0], w[129, 130], w[129, 128] = 4.0, 8.0, 16.0
    xs = torch.tensor([[0.5, 2.0], [1.0, 4.0]])
    ws = torch.tensor([[1.0, 10.0], [100.0, 1000.0]])
    out, size = ex.product(x.to(ex.F8), xs, w.to(ex.F8), ws)
    want = torch.zeros(2, 130, dtype=torch.float64)
    want[0, 0] = 2 * 4 * 0.5 * 1
    want[0, 129] = 3 * 8 * 2.0 * 1000
    want[1, 129] = 0.5 * 16 * 4 * 1000
    assert torch.equal(out, want) and torch.equal(size, want)


def test_the_definition_of_quantisation():
    y = torch.zeros(1, 256)
    y[0, 0], y[0, 1], y[0, 2], y[0, 128] = 448.0, -1.0625, 17.0, float("inf")
    q, s = ex.quantised(y)
    # 448 * f32(1/448) is 1 or next to it; 1.0625 lies between 1 and 1.125 (ties to the even 1), 17 between 16 and 18 (to 16)
    assert abs(float(s[0, 0]) - 1) <= 2.0 ** -23 and float(s[0, 1]) == 0
    assert q.float()[0, :3].tolist() == [448.0, -1.0, 16.0] and np.isnan(float(q.float()[0, 128]))


def test_the_definition_of_routing():
    l = torch.tensor([[1.0, 3.0, 3.0, float("-inf")], [float("-inf")] * 4, [0.0, float("nan"), 5.0, 5.0]])
    ids, w, rows, slots, offsets = ex.routed(l, 3, "softmax", True)
    assert ids.tolist() == [[1, 2, 0], [-1, -1, -1], [1, 2, 3]]
    assert offsets.tolist() == [0, 1, 3, 5, 6] and rows.tolist() == [0, 0, 2, 0, 2, 2, -1, -1, -1]
    assert slots.tolist() == [[1, 3, 0], [-1, -1, -1], [2, 4, 5]]
    assert torch.allclose(w[0], torch.softmax(torch.tensor([3.0, 3.0, 1.0], dtype=torch.float64), 0)) and not w[1].any()


# ---- the schedule of the products' tiles, restated ----
def shares(units, owners, most):
    """(first unit of each owner, owner of a unit) as the kernel computes them."""
    sharers = min(max(most, 1), owners)
    base, more = units // sharers, units - units // sharers * sharers

    def first(o):
        return o * base + min(o, more)

    def owner_of(u):
        return u // (base + 1) if u < more * (base + 1) else more + (u - more * (base + 1)) // base

    return sharers, first, owner_of


@pytest.mark.parametrize("owners", [1, 2, 74, 148])
def test_every_unit_has_one_owner(owners):
    for units in list(range(1, 400)) + [4096, 99991]:
        for least in (1, 2, 8, 16):
            sharers, first, owner_of = shares(units, owners, units // least)
            bounds = [first(o) for o in range(sharers)] + [units]
            assert bounds[0] == 0 and all(a < b for a, b in zip(bounds, bounds[1:]))
            for o in range(sharers):
                assert owner_of(bounds[o]) == o and owner_of(bounds[o + 1] - 1) == o


@pytest.mark.parametrize("wide", [2, 3, 7, 32, 129])
def test_panels_hold_every_tile_once(wide):
    """Tiles of many rows: 16 tiles' weights at a time, token by token, the last panel with fewer."""
    for across in (1, 2, 15, 16, 17, 33, 70):
        seen = set()
        for at in range(wide * across):
            panel = at // (16 * wide)
            left, n = at - panel * 16 * wide, min(16, across - panel * 16)
            place, tile = left // n, panel * 16 + left % n
            assert place < wide and tile < across
            seen.add((tile, place))
        assert len(seen) == wide * across


def test_owners_a_tile_by_a_float_quotient():
    """(most + 0.5) / rest, off by up to four steps of f32, has the whole part of most / rest: it is 0.5 / rest from a whole number at least."""
    for rest in range(1, 2033):
        for most in (0, 1, rest - 1, rest, rest + 1, 2 * rest - 1, 2 * rest, 5 * rest - 1, 5 * rest, 2032):
            exact = (most + 0.5) / rest
            assert int(exact * (1 - 2.0 ** -21)) == int(exact * (1 + 2.0 ** -21)) == most // rest


@pytest.mark.parametrize("tokens,step", [(32, 16), (128, 128), (256, 256)])
def test_a_groups_tiles_hold_its_rows(tokens, step):
    for rows in range(1, 3000):
        wide = -(-rows // tokens)
        each = -(-(-(-rows // wide)) // step) * step
        sizes = [min(each, rows - i * each) for i in range(wide)]
        assert all(0 < n <= tokens for n in sizes) and sum(sizes) == rows
