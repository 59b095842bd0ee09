"""`ops.dequant_i4` on both sides of the choice between its kernels: 3 rows a SM, rows of 6144."""
import pytest
import torch

from unpopped_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k,group", [(8, 8), (128, 32), (6144, 128), (6152, 8), (8192, 64)])
@pytest.mark.parametrize("n", [1, 444, 445, 700])
def test_every_row_count(n, k, group):
    g = torch.Generator(device="cuda").manual_seed(n + k)
    w = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scale = torch.rand(n, k // group, generator=g, device="cuda").half()
    v = torch.stack([w & 15, w >> 4], -1).flatten(1).int()
    want = (torch.where(v > 7, v - 16, v).float() * scale.float().repeat_interleave(group, 1)).bfloat16()
    assert torch.equal(ops.dequant_i4(w, scale, group), want)
