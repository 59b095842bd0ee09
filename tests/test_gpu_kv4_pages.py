"""Caches with no pages, and pages that are not there, under both attention kernels."""
import pytest
import torch
from kv4_exact import cache_of, exact, many_rows

from unpopped_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,kv,dim,many", [(600, 16, 128, True), (900, 16, 64, True), (3, 16, 128, False), (5, 2, 96, False)])
def test_a_cache_of_no_pages_is_not_read(tokens, kv, dim, many):
    """Every token is left out: 0 and -infinity. With pages of 4096 a page is larger than all queries together."""
    assert many_rows(tokens, 1, kv, kv, dim) == many
    cache = ops.kv4_cache(0, kv, dim, 4096, 32)
    q = torch.randn(tokens, kv, dim, device="cuda").half()
    cu = torch.tensor([0, tokens], dtype=torch.int32, device="cuda")
    lens = torch.tensor([4096], dtype=torch.int32, device="cuda")
    for page in (0, 5, -1):
        table = torch.tensor([[page]], dtype=torch.int32, device="cuda")
        out, lse = ops.kv4_attention(q, cache, table, lens, cu_q=cu, causal=False, want_lse=True)
        assert bool((out == 0).all()) and bool((lse == float("-inf")).all())


@pytest.mark.parametrize("dim,many", [(128, True), (64, True), (96, False)])
def test_runs_without_a_page_count_as_absent(dim, many):
    """Pages of 8 tokens, every third one outside the cache: the rest, against 64 bits."""
    n, kv, ratio, nq = 300, 2, 100, 160
    assert many_rows(nq, 1, kv * ratio, kv, dim) == many
    x = torch.randn(2, 1, n, kv, dim, generator=torch.Generator(device="cuda").manual_seed(dim), device="cuda")
    cache, table = cache_of(x, 8, 32)
    q = torch.randn(nq, kv * ratio, dim, device="cuda").half()
    cu = torch.tensor([0, nq], dtype=torch.int32, device="cuda")
    gone = table.clone()
    gone[0, ::3] = torch.tensor([-1, 10 ** 6], device="cuda").repeat(7)[:gone[0, ::3].numel()].int()
    got, lse = ops.kv4_attention(q, cache, gone, torch.tensor([n], dtype=torch.int32, device="cuda"), cu_q=cu, causal=False,
                                 want_lse=True)
    kept = table[:, [i for i in range(table.shape[1]) if i % 3]].contiguous()
    left = sum(min(8, n - 8 * i) for i in range(table.shape[1]) if i % 3)
    want, want_lse, tol, tol_lse = exact(q, cache, kept, torch.tensor([left]), cu, causal=False)
    assert bool(((got.double() - want).abs() <= tol).all())
    assert bool(((lse.double() - want_lse).abs() <= tol_lse).all())
