"""Both attention kernels held to the bounds of kv4_exact.py: the logits' are f32's everywhere, the rounding of nibble *
v_scale is allowed where it is made (many query rows, bf16 outputs) and nowhere else."""
import pytest
import torch
from kv4_exact import HALF_ULP, cache_of, exact, many_rows

from unpopped_b200 import ops

pytestmark = pytest.mark.gpu
GROUPS = [(32, 32), (64, 32), (64, 64), (96, 32), (96, 96), (128, 32), (128, 64), (128, 128), (160, 32), (192, 96), (224, 224),
          (256, 64), (256, 256)]


def check(dim, group, kv, ratio, lens, nq, kind, causal=True, window=0, page=16, scale=None, many=False):
    assert many_rows(sum(nq), len(lens), kv * ratio, kv, dim) == many
    g = torch.Generator(device="cuda").manual_seed(dim * 31 + group + ratio)
    x = torch.randn(2, len(lens), max(lens), kv, dim, generator=g, device="cuda")
    cache, table = cache_of(x, page, group, dim)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0] + nq, device="cuda").cumsum(0).int()
    q = torch.randn(sum(nq), kv * ratio, dim, generator=g, device="cuda").to(kind)
    out, lse = ops.kv4_attention(q, cache, table, n, cu_q=cu, causal=causal, window=window, scale=scale, want_lse=True)
    want, want_lse, tol, tol_lse = exact(q, cache, table, n, cu, causal, window, scale)
    off = (out.double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())
    empty = want_lse == float("-inf")
    assert torch.equal(lse.double() == float("-inf"), empty) and bool((out[empty] == 0).all())
    off_lse = (lse.double() - want_lse)[~empty].abs()
    assert bool((off_lse <= tol_lse[~empty]).all()), float((off_lse / tol_lse[~empty]).max())
    # roundings are independent, with a mean square of a third of their bound each
    u = HALF_ULP[kind] + 2.0 ** -11 * (2 if many and kind == torch.bfloat16 else 1)
    assert float((out.double() - want).norm() / want.norm()) <= u
    ops.check_workspace("kv4", q.device)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("ratio", [1, 5, 8, 16])
@pytest.mark.parametrize("dim,group", GROUPS)
def test_single_tokens(dim, group, ratio, kind):
    lens = [0, 1, 8, 31, 33, 127, 129, 1001]
    check(dim, group, 2, ratio, lens, [1] * len(lens), kind)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 37), (False, 0), (False, 200)])
@pytest.mark.parametrize("dim,group", GROUPS)
def test_a_few_tokens_a_sequence(dim, group, causal, window, kind):
    check(dim, group, 2, 3, [40, 9, 3, 0, 700, 255], [5, 1, 8, 2, 0, 130], kind, causal, window, page=8)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 37), (False, 0), (True, 300)])
@pytest.mark.parametrize("dim,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
def test_many_rows(dim, group, causal, window, kind):
    check(dim, group, 2, 29, [900, 513, 300, 0, 128, 129], [900, 250, 1, 3, 128, 200], kind, causal, window, page=32, many=True)


@pytest.mark.parametrize("dim,group", [(64, 64), (128, 32)])
@pytest.mark.parametrize("scale", [-0.2, 3.0, 0.0])
def test_other_scales_of_the_logits(dim, group, scale):
    for ratio, many in ((3, False), (100, True)):
        check(dim, group, 1, ratio, [300, 65], [150, 65], torch.float16, scale=scale, many=many, page=64)
