"""CUDA graphs of calls that take their workspace themselves."""
import pytest
import torch
from kv4_exact import cache_of, many_rows

from unpopped_b200 import ops

pytestmark = pytest.mark.gpu


def setup(batch, n, kv, dim, heads, nq, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(2, batch, n, kv, dim, generator=g, device="cuda")
    cache, table = cache_of(x, 16, 32, seed)
    q = torch.randn(batch * nq, heads, dim, generator=g, device="cuda").bfloat16()
    lens = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    cu = torch.arange(batch + 1, dtype=torch.int32, device="cuda") * nq
    return q, cache, table, lens, cu


def captured(q, cache, table, lens, cu):
    graph, out = torch.cuda.CUDAGraph(), torch.full_like(q, 7.0)
    with torch.cuda.graph(graph):
        ops.kv4_attention(q, cache, table, lens, cu_q=cu, out=out)
        ops.kv4_attention(q, cache, table, lens, cu_q=cu, out=out)
    return graph, out


@pytest.mark.parametrize("dim,heads,nq", [(64, 8, 1), (128, 16, 3), (128, 256, 45)])
def test_graphs_share_no_workspace(dim, heads, nq):
    """Two graphs of split tiles, the second replayed before the first; then a larger eager call, then both again. The last
    shape takes the tcgen05 kernel."""
    assert many_rows(2 * nq, 2, heads, 1, dim) == (heads == 256)
    ops._ws_cache.clear()
    sets = [setup(2, 3000, 1, dim, heads, nq, s) for s in (1, 2)]
    want = [ops.kv4_attention(*s[:4], cu_q=s[4]) for s in sets]
    ops._ws_cache.clear()
    junk = torch.full((64 << 20,), 0x5a, dtype=torch.uint8, device="cuda")  # what freed memory may hold
    del junk
    graphs = [captured(*s) for s in sets]
    assert not ops._ws_cache
    for i in (1, 0, 1, 1, 0):
        graphs[i][1].fill_(7.0)
        graphs[i][0].replay()
        assert torch.equal(graphs[i][1], want[i])
    big = setup(2, 3000, 1, 256, 64, 9, 3)
    ops.kv4_attention(*big[:4], cu_q=big[4])
    fresh = setup(2, 3000, 1, dim, heads, nq, 4)
    sets[0][0].copy_(fresh[0])
    graphs[0][0].replay()
    assert torch.equal(graphs[0][1], ops.kv4_attention(*sets[0][:4], cu_q=sets[0][4]))
    graphs[1][0].replay()
    assert torch.equal(graphs[1][1], want[1])


def test_a_stream_that_captures_and_runs_eagerly():
    """On one stream: a small eager call, a capture, a larger eager call (its workspace replaces the small one), replays."""
    ops._ws_cache.clear()
    a, b = setup(3, 2000, 1, 64, 4, 1, 5), setup(3, 2000, 1, 128, 16, 4, 6)
    want_a, want_b = ops.kv4_attention(*a[:4], cu_q=a[4]), ops.kv4_attention(*b[:4], cu_q=b[4])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert torch.equal(ops.kv4_attention(*a[:4], cu_q=a[4]), want_a)
        graph, out = torch.cuda.CUDAGraph(), torch.empty_like(a[0])
        with torch.cuda.graph(graph, stream=s):
            ops.kv4_attention(*a[:4], cu_q=a[4], out=out)
        for _ in range(3):
            got = ops.kv4_attention(*b[:4], cu_q=b[4])
            out.zero_()
            graph.replay()
            s.synchronize()
            assert torch.equal(got, want_b) and torch.equal(out, want_a)


def test_graphs_of_scans_and_w4a16_on_inputs_that_change():
    ops._ws_cache.clear()
    x = torch.randint(-50, 50, (3, 100001), device="cuda", dtype=torch.int32)
    w = torch.randint(0, 256, (512, 256), device="cuda", dtype=torch.uint8)
    scale = torch.rand(512, 4, device="cuda").half()
    act = torch.randn(4, 512, device="cuda").bfloat16()
    y, z = torch.empty_like(x), torch.empty(4, 512, device="cuda", dtype=torch.bfloat16)
    ops.scan(x), ops.w4a16(w, scale, act, 128)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.scan(x, out=y)
            ops.w4a16(w, scale, act, 128, out=z)
        graphs.append(graph)
    for i in (1, 0, 0, 1):
        x.copy_(torch.randint(-50, 50, x.shape, device="cuda", dtype=torch.int32))
        act.copy_(torch.randn(4, 512, device="cuda"))
        y.zero_(), z.zero_()
        graphs[i].replay()
        assert torch.equal(y, x.cumsum(1, dtype=torch.int32))
        assert torch.equal(z, ops.w4a16(w, scale, act, 128))
