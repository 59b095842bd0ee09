"""Launches that begin before the ones ahead end, on buffers that are written again and again: each pass is what it is with a wait for the GPU
after every call."""
import pytest
import torch

from unpopped_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def twice(run):
    """run(wait) without waits, then with one after every call; the outputs have to be alike bit for bit."""
    torch.cuda.synchronize()
    got = run(lambda: None)
    torch.cuda.synchronize()
    want = run(torch.cuda.synchronize)
    assert len(got) == len(want) > 10
    for a, b in zip(got, want):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))  # NaNs too
    return got


def weights(seed, n, k):
    return ops.f8_quantise_weight(torch.randn(n, k, generator=gen(seed), device=DEV) / k ** 0.5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,k", [(1, 1024), (8, 2048), (200, 2048), (64, 400), (2000, 1024)])
def test_quantise_of_what_a_product_writes_anew(rows, k, dtype):
    first = torch.randn(rows, k, generator=gen(k), device=DEV).to(dtype)
    w = [weights(i, k, k) for i in range(3)]

    def run(wait):
        h, kept = first.clone(), []
        for i in range(40):
            q, s = ops.f8_quantise(h)
            wait()
            ops.f8_matmul(q, s, *w[i % 3], out=h)
            wait()
            kept += [q.view(torch.uint8), s]
        return kept + [h]

    twice(run)


@pytest.mark.parametrize("size", [1.0, 0.05])
@pytest.mark.parametrize("tokens,n", [(4, 2048), (64, 1024), (700, 512)])
def test_the_sum_and_the_gate_of_what_a_product_writes_anew(tokens, n, size):
    """With weights of full size the values grow until they are no numbers any more, with small ones they do not."""
    g, k = gen(n), 4
    x = torch.randn(tokens, n, generator=g, device=DEV).bfloat16()
    slots = torch.randperm(tokens * k, generator=g, device=DEV).int().view(tokens, k)
    rows = torch.randint(0, tokens, (tokens * k,), generator=g, device=DEV, dtype=torch.int32)
    share = size * torch.rand(tokens, k, generator=g, device=DEV)
    up, down = weights(1, 2 * n, n), weights(2, n, n)

    def run(wait):
        h = torch.zeros(tokens * k, 2 * n, device=DEV, dtype=torch.bfloat16)
        y, out, kept = torch.zeros(tokens * k, n, device=DEV, dtype=torch.bfloat16), x.clone(), []
        for _ in range(20):
            q, s = ops.f8_quantise(out, rows)
            wait()
            ops.f8_matmul(q, s, *up, out=h)
            wait()
            q, s = ops.f8_quantise(h, gate=True)
            wait()
            kept += [q.view(torch.uint8), s]
            ops.f8_matmul(q, s, *down, out=y)
            wait()
            ops.expert_combine(y, slots, share, x, out)
            wait()
        return kept + [out]

    assert bool(twice(run)[-1].isfinite().all()) or size == 1


@pytest.mark.parametrize("tokens", [3, 64, 300])
def test_routing_by_logits_that_a_product_writes_anew(tokens):
    """A layer whose router, routing and sum go round a few buffers; rows and slots are written anew each time too."""
    e, k, d = 16, 4, 512
    g = gen(tokens)
    x = torch.randn(tokens, d, generator=g, device=DEV).bfloat16()
    router, w = weights(3, e, d), ops.f8_quantise_weight(torch.randn(e, d, d, generator=g, device=DEV) / d ** 0.5)

    def run(wait):
        out, logits, kept = x.clone(), torch.zeros(tokens, e, device=DEV), []
        y = torch.zeros(tokens * k, d, device=DEV, dtype=torch.bfloat16)
        for _ in range(20):
            q, s = ops.f8_quantise(out)
            wait()
            ops.f8_matmul(q, s, *router, out=logits)
            wait()
            ids, share, rows, slots, offsets = ops.expert_route(logits, k)
            wait()
            q, s = ops.f8_quantise(out, rows)
            wait()
            ops.f8_expert_matmul(q, s, *w, offsets, out=y)
            wait()
            ops.expert_combine(y, slots, share, x, out)
            wait()
            kept += [ids, share, rows, slots, offsets]
            del ids, share, rows, slots, offsets, q, s  # their memory is the next pass's
        return kept + [out]

    twice(run)
