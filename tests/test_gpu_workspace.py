"""A workspace that a launch left in the middle: the error word is set and counters of unfinished tiles are above zero. After the check that
reports it the next calls are right again."""
import pytest
import torch

import f8_exact as ex
from unpopped_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
HEADER = 64  # bytes; the error word is the fourth


def plant(ws, counters):
    """As a launch that gave up may leave it: every counter has seen an arrival."""
    words = ws[:HEADER + 4 * counters].view(torch.int32)
    words[HEADER // 4:] = 1
    words[3] = 1


def cached(kind):
    return ops._ws_cache[ops._ws_key(kind, torch.device("cuda", torch.cuda.current_device()))]


def recovers(kind, counters, call):
    want = call()
    ops.check_workspace(kind, DEV)
    plant(cached(kind), counters)
    with pytest.raises(_lib.UpError):
        ops.check_workspace(kind, DEV)
    for _ in range(3):
        assert torch.equal(call(), want)
    ops.check_workspace(kind, DEV)


def f8_problem(m, n, k):
    g = torch.Generator(device=DEV).manual_seed(m)
    x = torch.randn(m, k, generator=g, device=DEV).mul_(150).clamp_(-448, 448).to(ex.F8)
    w = torch.randn(n, k, generator=g, device=DEV).mul_(150).clamp_(-448, 448).to(ex.F8)
    return x, torch.rand(m, ex.blocks(k), generator=g, device=DEV), w, torch.rand(ex.blocks(n), ex.blocks(k), generator=g, device=DEV)


@pytest.mark.parametrize("m,n,k", [(1, 384, 8192), (300, 300, 8192), (1100, 1030, 8192)])
def test_f8_products(m, n, k):
    """Shapes whose tiles are shared."""
    p = f8_problem(m, n, k)
    recovers("f8", 8192 // 4 - HEADER // 4, lambda: ops.f8_matmul(*p, dtype=torch.float32))


def test_f8_products_in_a_workspace_of_the_callers():
    p = f8_problem(33, 384, 8192)
    space = torch.zeros(_lib.load().up_sm100_f8_matmul_workspace_bytes(33, 1, 384, 8192), dtype=torch.uint8, device=DEV)
    want = ops.f8_matmul(*p, dtype=torch.float32, ws=space)
    plant(space, 8192 // 4 - HEADER // 4)
    assert ops.workspace_status(space) == _lib.UP_ERR_DEVICE_TIMEOUT
    assert torch.equal(ops.f8_matmul(*p, dtype=torch.float32, ws=space), want)
    assert ops.workspace_status(space) == _lib.UP_OK


def test_w4a16():
    m, n, k, group = 4, 1024, 4096, 128
    g = torch.Generator(device=DEV).manual_seed(5)
    w = torch.randint(0, 256, (n, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    scale = torch.rand(n, k // group, generator=g, device=DEV).half()
    x = torch.randn(m, k, generator=g, device=DEV).bfloat16()
    recovers("w4a16", n // 128, lambda: ops.w4a16(w, scale, x, group))


def test_kv4_attention():
    g = torch.Generator(device=DEV).manual_seed(6)
    cache = ops.kv4_cache(64, 2, 64, device=DEV)
    k = torch.randn(1000, 2, 64, generator=g, device=DEV).bfloat16()
    ops.kv4_append(k, k, cache, torch.arange(1000, device=DEV, dtype=torch.int32))
    table = torch.arange(63, device=DEV, dtype=torch.int32)[None]
    lens, cu = torch.tensor([1000], dtype=torch.int32, device=DEV), torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    q = torch.randn(1, 4, 64, generator=g, device=DEV).bfloat16()
    recovers("kv4", 256, lambda: ops.kv4_attention(q, cache, table, lens, cu))


@pytest.mark.parametrize("m,n,k", [(1, 384, 8192), (384, 4096, 4096), (600, 4096, 8192), (5000, 512, 8192)])
def test_f8_products_under_a_limit_that_no_wait_keeps(m, n, k):
    """Whatever waits run out, the call ends, its status says so, and the next one is right."""
    L = _lib.load()
    p = f8_problem(m, n, k)
    want = ops.f8_matmul(*p, dtype=torch.float32)
    space = torch.zeros(L.up_sm100_f8_matmul_workspace_bytes(m, 1, n, k), dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    L.up_sm100_set_wait_limit_ns(1)
    try:
        got = ops.f8_matmul(*p, dtype=torch.float32, ws=space)
        status = ops.workspace_status(space)
    finally:
        L.up_sm100_set_wait_limit_ns(1_000_000_000)
    assert status == _lib.UP_ERR_DEVICE_TIMEOUT or (status == _lib.UP_OK and torch.equal(got, want))
    assert torch.equal(ops.f8_matmul(*p, dtype=torch.float32, ws=space), want) and ops.workspace_status(space) == _lib.UP_OK
