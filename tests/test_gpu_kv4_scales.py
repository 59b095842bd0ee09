"""Attention over caches whose scales lie far apart, under both kernels: tokens that a row does not see, weights far below a
row's largest, values that are not finite. Bounds: kv4_exact.py."""
import pytest
import torch
from kv4_exact import cache_of, exact, many_rows

from unpopped_b200 import ops

pytestmark = pytest.mark.gpu


def tokens_of(n, kv, dim, seed, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(2, 1, n, kv, dim, generator=g, device="cuda") * size


def cu_of(*counts):
    return torch.tensor((0,) + counts, device="cuda").cumsum(0).int()


def within(got, want, tol, rows=slice(None)):
    """Whether got is within tol of want, infinite where want rounds to that; and the largest error over its bound."""
    past = want.abs() > torch.finfo(got.dtype).max * (1 + 2.0 ** -12)  # (f16: from 65520 on)
    off = torch.where(past & (got == want.sign() * float("inf")), torch.zeros_like(want), (got.double() - want).abs())[rows]
    return bool((off <= tol[rows]).all()), float((off / tol[rows]).max())


MANY = [  # dim, group, query heads a key/value head, query tokens: the kernel for many query rows
    (128, 128, 75, 200), (128, 32, 75, 200), (64, 64, 115, 200), (64, 32, 115, 200)]
FEW = [(128, 128, 4, 200), (128, 32, 4, 200), (64, 32, 1, 8), (256, 64, 3, 20), (96, 96, 5, 30)]


def hidden(dim, group, ratio, nq, which, kind, many):
    """One token is a million times the others. Rows that causality or the window keeps from it are as exact as without it."""
    n, j, window = 260, 254, 100
    assert many_rows(nq, 1, ratio, 1, dim) == many
    x = tokens_of(n, 1, dim, dim + group, 0.3)
    x[which, 0, j] *= 4e5 / x[which, 0, j].abs().amax()  # a scale of 57143
    x[which, 0, 150] *= 4e5 / x[which, 0, 150].abs().amax()
    cache, table = cache_of(x, 16, group)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(ratio)
    q = (3 * torch.randn(nq, ratio, dim, generator=g, device="cuda")).to(kind)
    cu = cu_of(nq)
    out, lse = ops.kv4_attention(q, cache, table, lens, cu_q=cu, window=window, want_lse=True)
    want, want_lse, tol, tol_lse = exact(q, cache, table, lens, cu, window=window)
    pos = n - nq + torch.arange(nq, device="cuda")
    blind = (pos < j) & ((pos < 150) | (pos >= 150 + window))
    assert int(blind.sum()) > 0
    assert within(out, want, tol, blind)[0], within(out, want, tol, blind)[1]
    assert within(lse, want_lse, tol_lse, blind)[0], within(lse, want_lse, tol_lse, blind)[1]
    assert within(out, want, tol)[0] and within(lse, want_lse, tol_lse)[0]


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("dim,group,ratio,nq", MANY)
def test_many_rows_keep_their_precision_beside_a_hidden_token(dim, group, ratio, nq, which, kind):
    hidden(dim, group, ratio, nq, which, kind, True)


def not_finite(dim, group, ratio, nq, bad, many):
    """The logsumexp does not depend on the values; outputs that the value does not multiply keep their precision where few
    query rows share a tile, and are NaN where many do."""
    n, j = 260, 200
    assert many_rows(nq, 1, ratio, 1, dim) == many
    cache, table = cache_of(tokens_of(n, 1, dim, dim + group), 16, group)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    q = torch.randn(nq, ratio, dim, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").bfloat16()
    cu = cu_of(nq)
    want, want_lse, tol, tol_lse = exact(q, cache, table, lens, cu)
    cache[3][int(table[0, j // 16]), 0, j % 16, 0] = bad
    out, lse = ops.kv4_attention(q, cache, table, lens, cu_q=cu, want_lse=True)
    assert within(lse, want_lse, tol_lse)[0]
    sees = n - nq + torch.arange(nq, device="cuda") >= j
    assert within(out, want, tol, ~sees)[0] if bool((~sees).any()) else True
    assert not bool(torch.isfinite(out[sees][..., :group]).any())
    if many:
        assert bool(out[sees].isnan().all())
    elif group < dim:
        rest = (sees.nonzero()[:, 0], slice(None), slice(group, None))
        assert within(out, want, tol, rest)[0], within(out, want, tol, rest)[1]


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dim,group,ratio,nq", MANY)
def test_many_rows_keep_the_logsumexp_of_a_value_that_is_not_finite(dim, group, ratio, nq, bad):
    not_finite(dim, group, ratio, nq, bad, True)


@pytest.mark.parametrize("dim,ratio,nq", [(128, 64, 150), (64, 115, 150)])
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
def test_many_rows_keep_many_small_weights(dim, ratio, nq, kind):
    """One token with a value of 0 takes nearly all of the weight; 65536 others with weights of 2^-25.6 hold 2^-9.6 of it
    between them, which is all of the output."""
    n = 65537
    assert many_rows(nq, 1, ratio, 1, dim)
    pages = -(-n // 4096)
    cache = ops.kv4_cache(pages, 1, dim, 4096, dim)
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    cache[0].fill_(0x99), cache[1].fill_(0x77)  # -7 and 7 throughout
    cache[2].fill_(25.6 * 0.6931471805599453 / (7 * dim)), cache[3].fill_(1.0 / 7)
    cache[2][0, 0, 5] = cache[3][0, 0, 5] = 0.0
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    q = torch.ones(nq, ratio, dim, device="cuda").to(kind)
    cu = cu_of(nq)
    out, lse = ops.kv4_attention(q, cache, table, lens, cu_q=cu, causal=False, scale=1.0, want_lse=True)
    want, want_lse, tol, tol_lse = exact(q[:1, :1], cache, table, lens, cu_of(1), causal=False, scale=1.0)
    assert 2.0 ** -10 < float(want.min()) < 2.0 ** -9
    off = (out.double() - want).abs().max()
    assert float(off) <= float(tol.min()), (float(off), float(tol.min()))
    assert float((lse.double() - want_lse).abs().max()) <= float(tol_lse.min())


def grow_and_shrink(dim, group, ratio, nq, kind, many):
    """Values between 2^-12 and 2^12 of the first ones, up and down again, and keys that grow: against 64 bits."""
    n = 700
    assert many_rows(nq, 1, ratio, 1, dim) == many
    x = tokens_of(n, 1, dim, dim)
    j = torch.arange(n, device="cuda")
    x[0] *= (0.1 + j / 300)[:, None, None]
    x[1] *= torch.exp2(12 * torch.sin(j / 50.0))[:, None, None]
    cache, table = cache_of(x, 16, group)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    q = torch.randn(nq, ratio, dim, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(kind)
    for window in (0, 50):
        cu = cu_of(nq)
        out, lse = ops.kv4_attention(q, cache, table, lens, cu_q=cu, window=window, want_lse=True)
        want, want_lse, tol, tol_lse = exact(q, cache, table, lens, cu, window=window)
        assert within(out, want, tol)[0], within(out, want, tol)[1]
        assert within(lse, want_lse, tol_lse)[0], within(lse, want_lse, tol_lse)[1]


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,group,ratio,nq", MANY)
def test_many_rows_over_values_that_grow_and_shrink(dim, group, ratio, nq, kind):
    grow_and_shrink(dim, group, ratio, nq, kind, True)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("dim,group,ratio,nq", FEW)
def test_few_rows_keep_their_precision_beside_a_hidden_token(dim, group, ratio, nq, which, kind):
    hidden(dim, group, ratio, nq, which, kind, False)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dim,group,ratio,nq", FEW)
def test_few_rows_keep_the_others_precision_beside_a_value_that_is_not_finite(dim, group, ratio, nq, bad):
    not_finite(dim, group, ratio, nq, bad, False)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,group,ratio,nq", FEW)
def test_few_rows_over_values_that_grow_and_shrink(dim, group, ratio, nq, kind):
    grow_and_shrink(dim, group, ratio, nq, kind, False)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
def test_few_rows_keep_many_small_weights(dim, kind):
    """The same with a heavy token for each of a block's four warps, and sequences (over the same pages) enough that each is
    the work of few blocks."""
    n, batch = 65537, 600
    pages = -(-n // 4096)
    cache = ops.kv4_cache(pages, 1, dim, 4096, dim)
    cache[0].fill_(0x99), cache[1].fill_(0x77)
    cache[2].fill_(25.6 * 0.6931471805599453 / (7 * dim)), cache[3].fill_(1.0 / 7)
    for j in (5, 37, 69, 101):
        cache[2][0, 0, j] = cache[3][0, 0, j] = 0.0
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(batch, pages).contiguous()
    lens = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    q = torch.ones(batch, 2, dim, device="cuda").to(kind)
    assert not many_rows(batch, batch, 2, 1, dim)
    out, lse = ops.kv4_attention(q, cache, table, lens, scale=1.0, want_lse=True)
    want, want_lse, tol, tol_lse = exact(q[:1], cache, table[:1], lens[:1], scale=1.0)
    assert float((out.double() - want).abs().max()) <= float(tol.min()) < float(want.min()) / 4
    assert float((lse.double() - want_lse).abs().max()) <= float(tol_lse.min())
