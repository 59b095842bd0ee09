"""8-bit quantisation and products against their definitions in 64 bits (tests/f8_exact.py)."""
import pytest
import torch

import f8_exact as ex
from unpopped_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
F8 = ex.F8
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def codes(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV).mul_(150).clamp_(-448, 448).to(F8)


def scales(g, *shape):
    return torch.exp(torch.randn(*shape, generator=g, device=DEV) * 2) * 1e-3


def problem(seed, m, n, k, experts=None):
    g = gen(seed)
    e = () if experts is None else (experts,)
    return (codes(g, m, k), scales(g, ex.blocks(k), m).t(), codes(g, *e, n, k), scales(g, *e, ex.blocks(n), ex.blocks(k)))


def check(got, x, xs, w, ws):
    want, size = ex.product(x, xs, w, ws)
    bound = ex.product_bound(want, size, x.shape[1], got.dtype)
    off = (got.double() - want).abs()
    good = off <= bound
    if got.dtype == torch.float16:  # what is 65520 or more, half a step above the largest value, 65504, rounds to infinity
        good |= got.isinf() & (got.sign() == want.sign()) & (want.abs() + bound >= 65520)
    assert bool(good.all()), float((off / bound).max())


# ---- quantisation: bit for bit ----
def same(got, want):
    """e4m3 values alike, NaN where NaN."""
    a, b = got.float(), want.float()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,k", [(1, 16), (1, 128), (3, 144), (17, 1040), (130, 256), (5, 8192)])
def test_quantise(dtype, tokens, k):
    x = (torch.randn(tokens, k, generator=gen(k), device=DEV) * torch.exp(3 * torch.randn(tokens, 1, generator=gen(1), device=DEV))).to(dtype)
    q, s = ops.f8_quantise(x)
    wq, ws = ex.quantised(x.float())
    assert torch.equal(s, ws) and same(q, wq) and q.dtype == F8 and s.stride() == (1, tokens)


@pytest.mark.parametrize("dtype", TYPES)
def test_quantise_takes_rows_by_number(dtype):
    base = torch.randn(9, 3, 272, generator=gen(2), device=DEV).to(dtype)
    x = base[:, 1]  # rows of a wider tensor
    rows = torch.tensor([8, 0, 0, -1, 9, 3, 2 ** 31 - 1, -2 ** 31, 7], dtype=torch.int32, device=DEV)
    q, s = ops.f8_quantise(x, rows)
    keep = (rows >= 0) & (rows < 9)
    wq, ws = ex.quantised(x.float())
    at = rows[keep].long()
    assert same(q[keep], wq.float()[at].to(F8)) and torch.equal(s[keep], ws[at])
    assert not bool(q[~keep].float().any()) and not bool(s[~keep].any())


def test_quantise_of_values_that_are_not_finite_and_of_tiny_ones():
    x = torch.randn(6, 384, generator=gen(3), device=DEV)
    x[0, 5], x[0, 130], x[1, 200] = float("inf"), float("-inf"), float("nan")
    x[2, :128] = float("nan")       # a block of nothing else
    x[3, :128] = 0.0
    x[3, 128:256] = 2.0 ** -120     # its scale would be below 2^-126
    x[4, :128] = 448 * 2.0 ** -126  # its scale is just that
    x[5, :128] = 3.4e38
    q, s = ops.f8_quantise(x)
    wq, ws = ex.quantised(x)
    assert torch.equal(s, ws) and same(q, wq)
    assert float(s[3, 1]) == 0 and not bool(q[3, 128:256].float().any()) and float(s[4, 0]) == 2.0 ** -126
    assert bool(q[2, :128].float().isnan().all()) and float(s[2, 0]) == 0 and bool(q[0, 5].float().isnan())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,k", [(1, 16), (7, 400), (33, 2048)])
def test_quantise_with_a_gate(dtype, tokens, k):
    """y is within 2^-19 of silu(g) u: exp of an argument rounded to f32 (|g| < 16: 2^-20 at most, weighed with at most 1 of
    the result), a sum, an approximate quotient of 2 steps and two products. The scale is off by as much and two roundings;
    a code by that much of its value and half a step of 2^-4, of 2^-10 below 2^-6."""
    x = torch.randn(tokens, 2 * k, generator=gen(k), device=DEV).to(dtype)
    q, s = ops.f8_quantise(x, gate=True)
    d = x.double()
    y = d[:, :k] * torch.sigmoid(d[:, :k]) * d[:, k:]
    pad = torch.nn.functional.pad(y, (0, -k % 128)).unflatten(1, (-1, 128))
    want = pad.abs().amax(2) / 448
    assert bool(((s.double() - want).abs() <= want * (2.0 ** -19 + 2.0 ** -23)).all())
    v = y / want.repeat_interleave(128, 1)[:, :k]
    off = (q.double() - v).abs()
    assert bool((off <= (v.abs() * 2.0 ** -4).clamp(min=2.0 ** -10) + v.abs() * 2.0 ** -18).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantise_with_a_gate_far_from_0(dtype):
    """x down to -126, where exp(-x) leaves f32 or its reciprocal does, times u up to 1e37: silu(x) u is a plain number. The argument |x| / 2
    of exp, times log2(e), is below 128: its rounding is 2^-18 at most and its factor's as much, e^ of them 2^-17 of exp, which counts twice."""
    g = gen(41)
    x = torch.empty(64, 256, device=DEV)
    x[:, :128] = -126 * torch.rand(64, 1, generator=g, device=DEV) - torch.rand(64, 128, generator=g, device=DEV)
    x[:32, :128] = torch.linspace(-100, -80, 128, device=DEV)
    x[:, 128:] = torch.randn(64, 128, generator=g, device=DEV).sign() * (1 + torch.rand(64, 128, generator=g, device=DEV)) * 5e36
    x = x.to(dtype)
    q, s = ops.f8_quantise(x, gate=True)
    d = x.double()
    y = d[:, :128] * torch.sigmoid(d[:, :128]) * d[:, 128:]
    want = y.abs().amax(1, keepdim=True) / 448
    there = want >= 2.0 ** -125  # smaller scales are 0
    assert bool(there[:32].all())
    assert bool(((s.double() - want).abs() <= want * (2.0 ** -16 + 2.0 ** -23))[there].all())
    v = y / want
    off = (q.double() - v).abs()
    assert bool(((off <= (v.abs() * 2.0 ** -4).clamp(min=2.0 ** -10) + v.abs() * 2.0 ** -15) | ~there).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 16), (130, 144), (257, 384), (3, 130, 272), (2, 128, 128)])
def test_quantise_weight(dtype, shape):
    w = (torch.randn(*shape, generator=gen(shape[-1]), device=DEV) * 0.02).to(dtype)
    w.view(-1)[7] = float("inf")
    q, s = ops.f8_quantise_weight(w)
    for e, each in enumerate(w if w.dim() == 3 else [w]):
        wq, ws = ex.quantised(each.float(), 128)
        assert torch.equal(s[e] if w.dim() == 3 else s, ws) and same(q[e] if w.dim() == 3 else q, wq)


# ---- one matrix ----
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 128, 128), (1, 200, 2064), (2, 640, 4096), (16, 129, 144), (17, 256, 272), (61, 300, 400),
                                   (127, 127, 1280), (128, 128, 128), (129, 384, 656), (300, 1000, 528), (513, 520, 1152)])
def test_matmul(dtype, m, n, k):
    x, xs, w, ws = problem(m + n + k, m, n, k)
    check(ops.f8_matmul(x, xs, w, ws, dtype=dtype), x, xs, w, ws)


@pytest.mark.parametrize("m,n,k", [(1, 28672, 1024), (4, 8192, 8192), (40, 1024, 8192), (700, 2048, 2048), (4096, 1152, 1024)])
def test_matmul_of_many_tiles(m, n, k):
    x, xs, w, ws = problem(m, m, n, k)
    check(ops.f8_matmul(x, xs, w, ws, dtype=torch.float32), x, xs, w, ws)
    ops.check_workspace("f8", torch.device(DEV))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(30, 1003, 2064), (60, 8192, 1024), (600, 2064, 2048), (600, 2051, 2048), (1100, 4096, 528), (1100, 4111, 528),
                                   (2100, 4104, 1040), (4100, 2049, 512), (4100, 2304, 512)])
def test_matmul_of_many_rows_whose_outputs_lie_oddly(m, n, k, dtype):
    """Outputs whose rows begin on 32 bytes or anywhere, last tiles of few columns or rows, for few rows and for many."""
    x, xs, w, ws = problem(m + n, m, n, k)
    check(ops.f8_matmul(x, xs, w, ws, dtype=dtype), x, xs, w, ws)


@pytest.mark.parametrize("m,n,k", [(1, 130, 65552), (33, 300, 20496), (130, 130, 16400), (200, 300, 20480), (257, 513, 8208), (520, 300, 16384),
                                   (300, 4096, 8192)])
def test_matmul_of_few_tiles_that_many_share(m, n, k):
    x, xs, w, ws = problem(m + k, m, n, k)
    got = ops.f8_matmul(x, xs, w, ws, dtype=torch.float32)
    check(got, x, xs, w, ws)
    assert torch.equal(ops.f8_matmul(x, xs, w, ws, dtype=torch.float32), got)


@pytest.mark.parametrize("m,n,k", [(2100, 2049, 24576), (9000, 4500, 5136)])
def test_matmul_of_more_rows_than_l2_holds(m, n, k):
    """The tiles go by panels; every eighth row and all columns are looked at."""
    x, xs, w, ws = problem(m + n, m, n, k)
    check(ops.f8_matmul(x, xs, w, ws)[::8], x[::8], xs[::8], w, ws)


def test_matmul_of_views():
    """Rows of a wider x and out, scales by rows and broadcast, a column slice of a projection's output."""
    m, n, k = 37, 200, 272
    g = gen(5)
    x = codes(g, m, 3 * 320).view(m, 3, 320)[:, 1, :k]
    w, ws = codes(g, n, k), scales(g, 2, 3)
    for xs in (scales(g, m, 3), scales(g, m, 5)[:, 1:4], scales(g, 3).expand(m, 3), scales(g, m, 1).expand(m, 3)):
        wide = torch.full((m, n + 57), 7.0, device=DEV, dtype=torch.bfloat16)
        out = wide[:, 13:13 + n]
        assert ops.f8_matmul(x, xs, w, ws, out=out) is out
        check(out, x, xs, w, ws)
        assert bool((wide[:, :13] == 7).all()) and bool((wide[:, 13 + n:] == 7).all())


def test_matmul_gives_the_same_bits_each_time():
    x, xs, w, ws = problem(9, 33, 384, 8192)
    first = ops.f8_matmul(x, xs, w, ws, dtype=torch.float32)
    for _ in range(20):
        assert torch.equal(ops.f8_matmul(x, xs, w, ws, dtype=torch.float32), first)


def test_a_nan_reaches_its_row_or_column_only():
    x, xs, w, ws = problem(10, 40, 300, 512)
    want = ops.f8_matmul(x, xs, w, ws, dtype=torch.float32)
    xn, wn = x.clone(), w.clone()
    xn.view(torch.uint8)[3, 100] = 0x7f
    wn.view(torch.uint8)[200, 300] = 0xff
    got = ops.f8_matmul(xn, xs, wn, ws, dtype=torch.float32)
    assert bool(got[3].isnan().all()) and bool(got[:, 200].isnan().all())
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[3] = False
    keep[:, 200] = False
    assert torch.equal(got[keep], want[keep])


# ---- by expert ----
def sizes_case(name, experts, g):
    if name == "even":
        return [9] * experts
    if name == "empty ones":
        return [0, 5, 0, 0, 140, 1, 0, 33][:experts] + [0] * max(0, experts - 8)
    if name == "one has all":
        return [0] * (experts - 1) + [200]
    if name == "ones":
        return [1] * experts
    return torch.randint(0, 90, (experts,), generator=torch.Generator().manual_seed(g)).tolist()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("name", ["even", "empty ones", "one has all", "ones", "random"])
@pytest.mark.parametrize("experts,n,k", [(8, 136, 272), (8, 256, 128), (33, 72, 400)])
def test_expert_matmul(dtype, name, experts, n, k):
    sizes = sizes_case(name, experts, n)
    m = sum(sizes)
    x, xs, w, ws = problem(m, m, n, k, experts)
    offsets = torch.tensor([0] + sizes, device=DEV).cumsum(0).to(torch.int32)
    got = ops.f8_expert_matmul(x, xs, w, ws, offsets, dtype=dtype)
    want, size, _ = ex.by_expert(x, xs, w, ws, offsets)
    assert bool(((got.double() - want).abs() <= ex.product_bound(want, size, k, dtype)).all())


@pytest.mark.parametrize("experts,sizes,n,k", [(64, (0, 500), 1407, 528), (64, (0, 500), 1408, 528), (8, (100, 3000), 2048, 1024),
                                               (8, (100, 400), 1030, 8192), (3, (0, 40), 384, 16400)])
def test_expert_matmul_of_large_groups(experts, sizes, n, k):
    g = torch.Generator().manual_seed(n)
    rows = torch.randint(*sizes, (experts,), generator=g)
    m = int(rows.sum())
    x, xs, w, ws = problem(n, m, n, k, experts)
    offsets = torch.zeros(experts + 1, dtype=torch.int32)
    offsets[1:] = rows.cumsum(0)
    got = ops.f8_expert_matmul(x, xs, w, ws, offsets.to(DEV))
    want, size, _ = ex.by_expert(x, xs, w, ws, offsets)
    assert bool(((got.double() - want).abs() <= ex.product_bound(want, size, k, torch.bfloat16)).all())


@pytest.mark.parametrize("experts", [1, 31, 32, 33, 300, 1024])
def test_expert_matmul_of_many_experts(experts):
    g = torch.Generator().manual_seed(experts)
    sizes = torch.randint(0, 4, (experts,), generator=g)
    sizes[0] += 1
    m, n, k = int(sizes.sum()), 40, 144
    x, xs, w, ws = problem(experts, m, n, k, experts)
    offsets = torch.zeros(experts + 1, dtype=torch.int32)
    offsets[1:] = sizes.cumsum(0)
    got = ops.f8_expert_matmul(x, xs, w, ws, offsets.to(DEV), dtype=torch.float32)
    want, size, _ = ex.by_expert(x, xs, w, ws, offsets)
    assert bool(((got.double() - want).abs() <= ex.product_bound(want, size, k, torch.float32)).all())


@pytest.mark.parametrize("offsets", [[3, 3, 7, 10], [0, 0, 0, 0], [10, 0, 5, 60], [-5, 4, 2, 1000], [60, 60, 60, 60], [100, 200, 300, 400],
                                     [-2 ** 31, 2 ** 31 - 1, 0, 5]])
def test_rows_that_no_expert_has_stay(offsets):
    x, xs, w, ws = problem(3, 60, 130, 256, 3)
    at = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    out = torch.full((60, 130), 5.0, device=DEV)
    ops.f8_expert_matmul(x, xs, w, ws, at, out=out)
    want, size, bounds = ex.by_expert(x, xs, w, ws, at)
    has = torch.zeros(60, dtype=torch.bool, device=DEV)
    has[bounds[0]:bounds[-1]] = True
    assert bool((out[~has] == 5).all())
    assert bool(((out.double() - want).abs() <= ex.product_bound(want, size, 256, torch.float32))[has].all())


def test_one_expert_is_the_dense_product():
    x, xs, w, ws = problem(12, 70, 200, 528)
    offsets = torch.tensor([0, 70], dtype=torch.int32, device=DEV)
    assert torch.equal(ops.f8_expert_matmul(x, xs, w[None], ws[None], offsets), ops.f8_matmul(x, xs, w, ws))


# ---- calls ----
def test_empty_calls():
    x, xs, w, ws = problem(1, 4, 130, 128)
    assert ops.f8_matmul(x[:0], xs[:0], w, ws).shape == (0, 130)
    assert ops.f8_matmul(x, xs, w[:0], ws[:0]).shape == (4, 0)
    q, s = ops.f8_quantise(torch.empty(0, 256, device=DEV))
    assert q.shape == (0, 256) and s.shape == (0, 2)
    q, s = ops.f8_quantise(torch.empty(0, 256, device=DEV), torch.tensor([0, 5], dtype=torch.int32, device=DEV))
    assert not bool(q.float().any()) and not bool(s.any())


def test_another_stream_and_a_graph():
    x, xs, w, ws = problem(14, 21, 384, 4096)
    want = ops.f8_matmul(x, xs, w, ws)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.f8_matmul(x, xs, w, ws)
    s.synchronize()
    assert torch.equal(other, want)
    graphs = []
    for _ in range(2):  # two graphs that do not share a workspace, replayed beside each other
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.f8_matmul(x, xs, w, ws)
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for (g, out), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert torch.equal(out, want)


def test_two_streams_at_once_and_calls_of_every_size_after_one_another():
    """Each stream's workspace serves calls of every form; the two streams' calls run beside each other."""
    problems = [problem(i, m, n, k) for i, (m, n, k) in enumerate([(1, 4096, 4096), (700, 2048, 1024), (20, 384, 8192), (2100, 4096, 512),
                                                                  (300, 300, 8192), (1, 1, 16), (129, 1000, 2048)])]
    want = [ops.f8_matmul(*p) for p in problems]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for turn in range(6):
        for i, p in enumerate(problems):
            for j, st in enumerate(streams):
                with torch.cuda.stream(st):
                    got.append((i, ops.f8_matmul(*problems[(i + 3 * j) % len(problems)]), (i + 3 * j) % len(problems)))
    torch.cuda.synchronize()
    for _, out, i in got:
        assert torch.equal(out, want[i])
    ops.check_workspace("f8", torch.device(DEV))


def test_a_call_right_behind_the_one_that_makes_its_operands():
    """Launches begin before the ones before them end: operands, scales, offsets and a workspace come from the launch right before."""
    g = gen(31)
    x = torch.randn(700, 1024, generator=g, device=DEV).bfloat16()
    w = torch.randn(600, 1024, generator=g, device=DEV).bfloat16()
    wq, wsc = ops.f8_quantise_weight(w)
    first = None
    for _ in range(30):
        q, sc = ops.f8_quantise(x)
        y = ops.f8_matmul(q, sc, wq, wsc)
        q2, sc2 = ops.f8_quantise(y[:, :512])
        z = ops.f8_matmul(q2, sc2, wq[:, :512].contiguous(), wsc[:, :4].contiguous(), dtype=torch.float32)
        if first is None:
            torch.cuda.synchronize()
            check(y, q, sc, wq, wsc)
            check(z, q2, sc2, wq[:, :512].contiguous(), wsc[:, :4].contiguous())
            first = y, z
        assert torch.equal(first[0], y) and torch.equal(first[1], z)


def test_offsets_that_pass_32_bits():
    """Outputs of more than 2^32 bytes and 2^31 values; activations and weights of more than 2^32 bytes."""
    g = gen(32)
    m, n, k = 70000, 32768, 16
    x, xs, w, ws = problem(33, m, n, k)
    out = torch.empty(m, n, device=DEV, dtype=torch.bfloat16)
    ops.f8_matmul(x, xs, w, ws, out=out)
    for at in (0, 32768, 65535, 69000):
        check(out[at:at + 64], x[at:at + 64], xs[at:at + 64], w, ws)
    del out
    rows, k = 270000, 8192
    big = torch.zeros(rows, k, device=DEV, dtype=torch.bfloat16)
    for at in (0, rows // 2 + 1, rows - 300):
        big[at:at + 300] = torch.randn(300, k, generator=g, device=DEV).bfloat16()
    q, sc = ops.f8_quantise(big)
    for at in (0, rows // 2 + 1, rows - 300):
        wq, wsc = ex.quantised(big[at:at + 300].float())
        assert same(q[at:at + 300], wq) and torch.equal(sc[at:at + 300], wsc)
    del big
    w, ws = codes(g, 24, k), scales(g, 1, 64)
    got = ops.f8_matmul(q, sc, w, ws, dtype=torch.float32)
    check(got[-300:], q[-300:], sc[-300:], w, ws)
    del q, sc, got
    experts, n = 70, 8192
    w = torch.zeros(experts, n, k, device=DEV, dtype=torch.uint8)
    w[-1] = codes(g, n, k).view(torch.uint8)
    w, ws = w.view(F8), scales(g, experts, 64, 64)
    x, xs = codes(g, 5, k), scales(g, 64, 5).t()
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=DEV)
    offsets[-1] = 5
    check(ops.f8_expert_matmul(x, xs, w, ws, offsets), x, xs, w[-1], ws[-1])


def test_a_workspace_of_the_callers():
    x, xs, w, ws = problem(15, 21, 384, 4096)
    n = _lib.load().up_sm100_f8_matmul_workspace_bytes(21, 1, 384, 4096)
    space = torch.full((n,), 0x5a, dtype=torch.uint8, device=DEV)
    space[:8192] = 0
    for _ in range(3):
        assert torch.equal(ops.f8_matmul(x, xs, w, ws, ws=space), ops.f8_matmul(x, xs, w, ws))
    assert ops.workspace_status(space) == _lib.UP_OK and not bool(space[:8192].any())
    with pytest.raises(_lib.UpError):
        ops.f8_matmul(x, xs, w, ws, ws=space[:8192])


def test_refusals_of_tensors():
    x, xs, w, ws = problem(16, 21, 384, 256)
    bad = [dict(x=x.float()), dict(x=x[:, :128]), dict(xs=xs[:, :1]), dict(xs=xs.double()), dict(xs=xs[:20]), dict(w=w[:, :128]),
           dict(w=w.float()), dict(w=w.t()), dict(ws=ws[:2]), dict(ws=ws.t()), dict(dtype=torch.float64), dict(dtype=torch.int32),
           dict(out=torch.empty(21, 383, device=DEV)), dict(out=torch.empty(21, 384, device=DEV, dtype=torch.float64)),
           dict(out=torch.empty(384, 21, device=DEV).t()), dict(xs=xs.cpu()), dict(x=x[0])]
    for change in bad:
        a = dict(x=x, xs=xs, w=w, ws=ws, dtype=torch.bfloat16, out=None)
        a.update(change)
        with pytest.raises((ValueError, TypeError)):
            ops.f8_matmul(a["x"], a["xs"], a["w"], a["ws"], dtype=a["dtype"], out=a["out"])
    k = 136  # no multiple of 16
    with pytest.raises(_lib.UpError):
        ops.f8_matmul(codes(gen(1), 3, k), scales(gen(1), 3, 2), codes(gen(1), 5, k), scales(gen(1), 1, 2))
    with pytest.raises(_lib.UpError):  # rows that are not 16 bytes apart
        ops.f8_matmul(codes(gen(1), 3, 136)[:, :128], scales(gen(1), 3, 1), codes(gen(1), 5, 128), scales(gen(1), 1, 1))
    with pytest.raises(TypeError):
        ops.f8_expert_matmul(x, xs, w[None], ws[None], None)
    with pytest.raises(ValueError):
        ops.f8_expert_matmul(x, xs, w[None], ws[None], torch.zeros(3, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError):
        ops.f8_expert_matmul(x, xs, w[None], ws[None], torch.zeros(2, dtype=torch.int64, device=DEV))
    with pytest.raises(_lib.UpError):
        ops.f8_quantise(torch.zeros(3, 136, device=DEV)[:, :120])
    with pytest.raises(ValueError):
        ops.f8_quantise(torch.zeros(3, 135, device=DEV), gate=True)
    with pytest.raises(ValueError):
        ops.f8_quantise(torch.zeros(3, 128, device=DEV, dtype=torch.float64))
