"""The paged 4-bit key/value cache on the GPU: `ops.kv4_append` and `ops.kv4_attention` against plain implementations.

Append: every operation is defined as an f32 one rounded by itself, so packed values and scales equal a plain f32
restatement bit for bit; the stored values are held to half a step against 64 bits.

Attention, against 64 bits, for weights w (the softmax), logits s, values v:
  |out - exact| <= (u_p + 2 ds + 2^-20) sum w |v| + n 2^-22 max|v_scale| / l + u |exact|
u_p = 2^-11 (p * v_scale is rounded to f16), u the output type's half ulp, ds = 2^-18 max_j scale sum_d |q_d k_jd| (f32
sums of at most 256 exact products in pieces of 16, and the scales' products), 2^-20 the exponentials and the f32 sums
of probabilities; the middle term is the f16 range's lower end (2^-25 of the scaled probabilities, times a nibble of at
most 8), with l the sum of exp(s - max). |lse - exact| <= ds + 2^-19 + 2^-22 |exact|.

With 64 query rows a sequence and key/value head or more and heads of 64 or 128, nibble * scale is rounded to f16 before
the products: ds grows by 2^-11 max_j scale sum_d |q_d k_jd|, and v's rounding adds 2^-11 sum w |v|. Those are worst cases;
as roundings are independent with a mean square of a third of their bound, the whole output is also held to
||out - exact|| <= (u / sqrt(3) + 2^-10) ||exact|| for normally distributed inputs (logits and values of order 1)."""
import pytest
import torch

from unpopped_b200 import _lib, ops

pytestmark = pytest.mark.gpu
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def table_of(n, rot):
    f = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / max(rot, 1))
    a = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float().reshape(n, rot)


def values(packed, scale, dtype=torch.float64):
    b = packed.to(torch.int16)
    n = torch.stack([b & 15, b >> 4], -1).flatten(-2)
    n = torch.where(n > 7, n - 16, n).to(dtype)
    return n * scale.to(dtype).repeat_interleave(n.shape[-1] // scale.shape[-1], -1)


def quantised(x, group):
    """The append's formula, in f32: (packed, scale)."""
    x = x.float().unflatten(-1, (-1, group))
    amax = x.abs().amax(-1)
    scale = (amax * torch.tensor(1.0 / 7.0, dtype=torch.float32, device="cuda")).clamp(max=65504.0).half()
    scale = torch.where(torch.isfinite(amax), scale, torch.full_like(scale, float("nan")))
    f = scale.float()[..., None]
    n = torch.where(f > 0, (x * (1.0 / f)).round().clamp(-8, 7), torch.zeros_like(x)).to(torch.int16).flatten(-2)
    return ((n[..., 0::2] & 15) | ((n[..., 1::2] & 15) << 4)).to(torch.uint8), scale


def turned(x, pos, table, layout):
    """rope in f32, each product and sum rounded by itself."""
    rot = table.shape[1]
    y = x.float().clone()
    c, s = table[pos][:, None, :rot // 2], table[pos][:, None, rot // 2:]
    i = torch.arange(rot // 2, device="cuda")
    a, b = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
    x0, x1 = y[..., a], y[..., b]
    y[..., a], y[..., b] = x0 * c - x1 * s, x1 * c + x0 * s
    return y


def stale_cache(pages, kv, dim, page, group, seed=0):
    """A cache whose slots hold leftovers: any nibbles, NaN and infinite scales."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = ops.kv4_cache(pages, kv, dim, page, group)
    for t in c[:2]:
        t.copy_(torch.randint(0, 256, t.shape, generator=g, device="cuda"))
    for t in c[2:]:
        t.fill_(float("nan"))
        t.view(-1)[::3] = float("inf")
    return c


# ---- append ----
@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,kv,dim,rot,group,page", [
    (1, 1, 1, 32, 32, 32, 8), (1, 64, 8, 128, 128, 32, 16), (37, 6, 3, 96, 96, 96, 16), (50, 4, 4, 64, 20, 32, 8),
    (9, 5, 1, 256, 64, 256, 64), (130, 0, 2, 160, 0, 32, 32), (21, 7, 7, 192, 128, 64, 8), (3, 2, 1, 224, 30, 224, 4096)])
def test_append_equals_the_plain_restatement(kind, layout, tokens, heads, kv, dim, rot, group, page):
    g = torch.Generator(device="cuda").manual_seed(dim * 7 + tokens)
    qkv = torch.randn(tokens, heads + 2 * kv, dim, generator=g, device="cuda").to(kind)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    pages = -(-tokens // page) + 2
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    pos = torch.randint(0, 300, (tokens,), generator=g, device="cuda")
    table = table_of(300, rot)
    cache = stale_cache(pages, kv, dim, page, group)
    want = [t.clone() for t in cache]
    got_q = ops.kv4_append(k, v, cache, slots, pos, table, q=q if heads else None, layout=layout)
    if heads:
        assert torch.equal(got_q, turned(q, pos, table, layout).to(kind))
        assert torch.equal(got_q, ops.rope(q, pos, table, layout))
    new_k, new_v = quantised(turned(k, pos, table, layout), group), quantised(v, group)
    at = (slots // page, slice(None), slots % page)
    for t, rows in zip(want, (new_k[0], new_v[0], new_k[1], new_v[1])):
        t[at] = rows
    for got, t in zip(cache, want):  # written slots as restated, all others untouched
        assert torch.equal(got.view(torch.uint8), t.view(torch.uint8))
    # the values: within half a step (and f16's rounding of the step) of what went in
    step = cache[3][at].double().repeat_interleave(group, -1)
    assert bool(((values(cache[1], cache[3])[at] - v.double()).abs() <= step * (0.5 + 2.0 ** -8)).all())
    # int32 positions and slots, and no rotation
    again = stale_cache(pages, kv, dim, page, group)
    ops.kv4_append(k, v, again, slots.int(), pos.int(), table, layout=layout)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(again, cache))
    ops.kv4_append(k, v, again, slots)
    assert torch.equal(again[0][at], quantised(k, group)[0]) and torch.equal(again[2][at], quantised(k, group)[1])


def test_append_extremes_and_padding():
    """Zeros, values below f16's smallest step, above what its largest can span, infinities and NaN; slots and positions
    outside."""
    kv, dim, group, page = 2, 64, 32, 8
    x = torch.zeros(8, kv, dim, device="cuda")
    x[1] = 1e-9
    x[2] = torch.linspace(-3e-7, 3e-7, dim, device="cuda")
    x[3] = torch.linspace(-1e6, 1e6, dim, device="cuda")
    x[4, 0, 5], x[4, 1, 40] = float("inf"), float("nan")
    x[5] = 1.0
    x[6], x[7] = 2.0, 3.0
    x = x.to(torch.bfloat16)
    slots = torch.tensor([3, 0, 9, 15, 8, 1, -1, 16], device="cuda")
    cache = stale_cache(2, kv, dim, page, group)
    before = [t.clone() for t in cache]
    ops.kv4_append(x, x, cache, slots)
    keep = slots[:6]
    at = (keep // page, slice(None), keep % page)
    packed, scale = quantised(x[:6], group)
    for t, rows in zip(before, (packed, packed, scale, scale)):
        t[at] = rows
    for a, b in zip(cache, before):
        assert torch.equal(a.nan_to_num(nan=-1.0) if a.is_floating_point() else a,
                           b.nan_to_num(nan=-1.0) if b.is_floating_point() else b)
    read = values(cache[0], cache[2])[at]
    assert bool((read[0] == 0).all()) and bool((read[1] == 0).all())
    assert bool(read[4, 0, :32].isnan().all()) and bool((read[4, 0, 32:] == 0).all())
    assert bool((read[4, 1, :32] == 0).all()) and bool(read[4, 1, 32:].isnan().all())
    assert float(read[3].abs().max()) == 7 * 65504 or float(read[3].abs().max()) == 8 * 65504
    # a position outside the table: the key and the query are NaN, the value is not
    q = ops.kv4_append(x[5:6], x[5:6], cache, slots[5:6], torch.tensor([9], device="cuda"), table_of(9, 32), q=x[5:6])
    assert bool(q[..., :32].isnan().all()) and torch.equal(q[..., 32:], x[5:6, :, 32:])
    assert bool(values(cache[0], cache[2])[0, :, 1, :32].isnan().all())
    assert bool((values(cache[1], cache[3])[0, :, 1] - 1).abs().max() < 1e-3)


def test_append_strides_and_in_place_queries():
    kv, dim, group, page, t = 2, 96, 32, 8, 11
    table, pos = table_of(20, 96), torch.arange(11, device="cuda")
    k = torch.randn(t, kv, dim, device="cuda").half()
    q = torch.randn(t, 3, dim, device="cuda").half()
    slots = torch.arange(t, device="cuda")
    a, b = ops.kv4_cache(2, kv, dim, page, group), ops.kv4_cache(2, kv, dim, page, group)
    want = ops.kv4_append(k, k, a, slots, pos, table, q=q)
    odd = torch.empty(t, kv, dim + 3, device="cuda").half()[..., 1:dim + 1]  # rows that are not 16-byte aligned
    odd.copy_(k)
    heads_first = k.transpose(0, 1).contiguous().transpose(0, 1)
    got = ops.kv4_append(odd, heads_first, b, slots, pos, table, q=q, q_out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_dequant_reads_the_cache():
    kv, dim, group, page = 2, 64, 32, 8
    v = torch.randn(16, kv, dim, device="cuda").bfloat16()
    cache = ops.kv4_cache(2, kv, dim, page, group)
    ops.kv4_append(v, v, cache, torch.arange(16, device="cuda"))
    rows = 2 * kv * page
    got = ops.dequant_i4(cache[1].view(rows, -1), cache[3].view(rows, -1), group)
    assert torch.equal(got.double(), values(cache[1], cache[3]).view(rows, dim).bfloat16().double())


# ---- attention ----
def make(batch, kv, dim, group, page, lens, seed=0, spread=1.0, order=True):
    """A cache with `lens` tokens a sequence on shuffled pages; every slot past a sequence's end is a leftover."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = max(1, -(-max(lens) // page)) + 1
    pages = batch * width + 1
    cache = stale_cache(pages, kv, dim, page, group, seed)
    table = torch.randperm(pages, generator=g, device="cuda")[:batch * width].int().view(batch, width)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        x = torch.randn(2, n, kv, dim, generator=g, device="cuda") * spread
        j = torch.arange(n, device="cuda")
        slots = table[b, j // page].long() * page + j % page
        ops.kv4_append(x[0].bfloat16(), x[1].bfloat16(), cache, slots)
    return cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


def rounds_cache(q, cache, lens):
    """Whether nibble * scale is rounded to f16 (the kernel for many query rows)."""
    per = -(-q.shape[0] // len(lens)) * (q.shape[1] // cache[0].shape[1])
    return per >= 64 and q.shape[2] in (64, 128)


def reference(q, cache, table, lens, cu, causal, window, scale):
    """(out, lse, bound of out, bound of lse), in 64 bits."""
    f16 = 2.0 ** -11 if rounds_cache(q, cache, lens) else 0.0
    page, ratio = cache[0].shape[2], q.shape[1] // cache[0].shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    lse = torch.full(q.shape[:2], float("-inf"), dtype=torch.float64, device="cuda")
    tol_lse = torch.zeros_like(lse)
    for b, n in enumerate(lens.tolist()):
        q0, nq = (b, 1) if cu is None else (int(cu[b]), int(cu[b + 1]) - int(cu[b]))
        if n == 0 or nq == 0:
            continue
        ids = table[b, : -(-n // page)].long()
        rows = [values(cache[i][ids], cache[i + 2][ids]).transpose(1, 2).flatten(0, 1)[:n].repeat_interleave(ratio, 1)
                for i in (0, 1)]
        x = q[q0:q0 + nq].double()
        s = torch.einsum("qhd,khd->hqk", x, rows[0]) * scale
        mag = torch.einsum("qhd,khd->hqk", x.abs(), rows[0].abs()) * abs(scale)
        pos = n - nq + torch.arange(nq, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")
        see = (j <= pos) if causal else torch.ones(nq, n, dtype=torch.bool, device="cuda")
        if window:
            see = see & (j > pos - window)
        some = see.any(-1)
        s = s.masked_fill(~see, float("-inf"))
        m = s.amax(-1, keepdim=True)
        p = torch.where(see, torch.exp(s - torch.where(some[None, :, None], m, torch.zeros_like(m))), torch.zeros_like(s))
        l = p.sum(-1, keepdim=True)
        w = p / torch.where(l > 0, l, torch.ones_like(l))
        ds = (2.0 ** -18 + f16) * mag.masked_fill(~see, 0).amax(-1)
        vs = cache[3][ids].double().nan_to_num(0, 0, 0).abs().max()
        o = torch.einsum("hqk,khd->qhd", w, rows[1])
        near = torch.einsum("hqk,khd->qhd", w, rows[1].abs())
        seen = see.sum(-1)[:, None, None]
        tol[q0:q0 + nq] = ((2.0 ** -11 + f16 + 2.0 ** -20 + 2 * ds.T[..., None]) * near + o.abs() * U[q.dtype] +
                           seen * 2.0 ** -22 * vs / l.squeeze(-1).T[..., None].clamp(min=1.0) + 2.0 ** -24)
        out[q0:q0 + nq] = o
        z = (m.squeeze(-1) + l.squeeze(-1).log()).T
        lse[q0:q0 + nq] = torch.where(some[:, None], z, torch.full_like(z, float("-inf")))
        tol_lse[q0:q0 + nq] = (ds.T + 2.0 ** -19 + 2.0 ** -22 * z.abs()).nan_to_num(0, 0, 0)
    return out, lse, tol, tol_lse


def check(q, cache, table, lens, cu=None, causal=True, window=0, scale=None):
    out, lse = ops.kv4_attention(q, cache, table, lens, cu_q=cu, causal=causal, window=window, scale=scale, want_lse=True)
    want, want_lse, tol, tol_lse = reference(q, cache, table, lens, cu, causal, window,
                                             q.shape[2] ** -0.5 if scale is None else scale)
    off = (out.double() - want).abs()
    assert bool((off <= tol).all()), (float((off / tol).max()), int((~(off <= tol)).sum()))
    empty = want_lse == float("-inf")
    assert torch.equal(lse.double() == float("-inf"), empty) and bool((out[empty] == 0).all())
    if rounds_cache(q, cache, lens) and scale is None:
        assert float((out.double() - want).norm() / want.norm()) <= U[q.dtype] / 3 ** 0.5 + 2.0 ** -10
    off = (lse.double() - want_lse)[~empty].abs()
    assert bool((off <= tol_lse[~empty]).all()), float((off / tol_lse[~empty]).max())
    assert torch.equal(ops.kv4_attention(q, cache, table, lens, cu_q=cu, causal=causal, window=window, scale=scale), out)
    return out


@pytest.mark.parametrize("dim,group", [(32, 32), (64, 32), (64, 64), (96, 32), (96, 96), (128, 32), (128, 64), (128, 128),
                                       (160, 32), (160, 160), (192, 64), (192, 96), (224, 224), (256, 32), (256, 64),
                                       (256, 128), (256, 256)])
@pytest.mark.parametrize("ratio", [1, 3, 8, 11])
def test_one_token_a_sequence(dim, group, ratio):
    lens = [0, 1, 7, 8, 31, 32, 33, 127, 128, 129, 640, 1001]
    cache, table, n = make(len(lens), 2, dim, group, 16, lens, seed=dim)
    g = torch.Generator(device="cuda").manual_seed(ratio)
    for kind in (torch.bfloat16, torch.float16):
        check(torch.randn(len(lens), 2 * ratio, dim, generator=g, device="cuda").to(kind), cache, table, n)


@pytest.mark.parametrize("page", [8, 16, 64, 256, 4096])
def test_page_sizes(page):
    lens = [5, 300, 513]
    cache, table, n = make(3, 1, 64, 32, page, lens, seed=page)
    check(torch.randn(3, 4, 64, device="cuda").half(), cache, table, n)


@pytest.mark.parametrize("dim,group", [(64, 32), (128, 128), (128, 32), (96, 96), (256, 64)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [0, 1, 40, 300])
def test_several_tokens_a_sequence(dim, group, causal, window):
    """Ragged query counts, none among them; sequences shorter than their queries (rows that see nothing)."""
    lens, nq = [40, 9, 3, 0, 700, 255], [5, 1, 8, 2, 0, 130]
    cache, table, n = make(len(lens), 2, dim, group, 16, lens, seed=window)
    cu = torch.tensor([0] + nq, device="cuda").cumsum(0).int()
    q = torch.randn(sum(nq), 6, dim, device="cuda").bfloat16()
    check(q, cache, table, n, cu, causal, window)


@pytest.mark.parametrize("dim,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("ratio", [1, 4, 5])
def test_prompts(dim, group, ratio):
    lens, nq = [900, 513, 300, 0, 128, 129], [900, 250, 1, 3, 128, 200]
    cache, table, n = make(6, 2, dim, group, 32, lens, seed=5)
    cu = torch.tensor([0] + nq, device="cuda").cumsum(0).int()
    for kind, window, causal in ((torch.bfloat16, 0, True), (torch.float16, 200, True), (torch.float16, 0, False)):
        check(torch.randn(sum(nq), 2 * ratio, dim, device="cuda").to(kind), cache, table, n, cu, causal, window)


def test_prompts_over_a_longer_context_and_small_pages():
    cache, table, n = make(2, 1, 128, 128, 8, [3000, 2111], seed=15)
    cu = torch.tensor([0, 70, 333], device="cuda").int()
    check(torch.randn(333, 3, 128, device="cuda").bfloat16(), cache, table, n, cu)
    packed = torch.randn(333, 7, 128, device="cuda").half()
    out = torch.zeros(333, 7, 128, device="cuda").half()
    ops.kv4_attention(packed[:, 2:5], cache, table, n, cu_q=cu, out=out[:, 1:4])
    assert torch.equal(out[:, 1:4], check(packed[:, 2:5], cache, table, n, cu))
    assert bool((out[:, 0] == 0).all()) and bool((out[:, 4:] == 0).all())


def test_prompts_with_scales_far_apart():
    """Values whose scales fall and rise by 2^12 between tiles, a maximum that rises late: all rows, some of which see
    only the small ones. The values are not of order 1, so the element-wise bound alone holds (a scale of 1 / 8 given)."""
    cache, table, n = make(1, 1, 64, 32, 16, [700], seed=21, spread=4.0)
    j = torch.arange(700, device="cuda")
    page, at = table[0, j // 16].long(), j % 16
    cache[2][page, 0, at] *= (0.1 + j / 100)[:, None].half()
    cache[3][page, 0, at] *= (2.0 ** (12 * (j / 700 - 0.5).abs() - 8))[:, None].half()
    cu = torch.tensor([0, 700], device="cuda").int()
    check(torch.randn(700, 2, 64, device="cuda").bfloat16(), cache, table, n, cu, scale=0.125)
    check((torch.randn(700, 2, 64, device="cuda") * 1e30).bfloat16(), cache, table, n, cu, scale=1e-31)


def test_prompts_with_a_nan_and_pages_outside():
    """A NaN reaches the rows that see it only (where many rows share a tile, all of such a row)."""
    cache, table, n = make(1, 1, 128, 64, 16, [300], seed=4)
    j = 200
    cu = torch.tensor([0, 300], dtype=torch.int32, device="cuda")
    q = torch.randn(300, 2, 128, device="cuda").bfloat16()
    clean = ops.kv4_attention(q, cache, table, n, cu_q=cu)
    for which in (3, 2):
        keep = cache[which][int(table[0, j // 16]), 0, j % 16, 1].clone()
        for bad in (float("nan"), float("inf")):
            cache[which][int(table[0, j // 16]), 0, j % 16, 1] = bad
            out = ops.kv4_attention(q, cache, table, n, cu_q=cu)
            assert torch.equal(out[:j], clean[:j])
            assert not bool(torch.isfinite(out[j:, :, 64:]).any()) or which == 2
        cache[which][int(table[0, j // 16]), 0, j % 16, 1] = keep
    # pages outside the cache: as if those tokens were masked for every row
    bad = table.clone()
    bad[0, 3] = -1
    got = ops.kv4_attention(q, cache, bad, n, cu_q=cu)
    assert torch.equal(got[:48], clean[:48]) and bool(torch.isfinite(got).all())
    assert not torch.equal(got[64:], clean[64:])


@pytest.mark.parametrize("dim,group", [(64, 32), (64, 64), (96, 96), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("scale", [None, -0.2])
def test_prompts_keep_the_logits_of_32_bits(dim, group, scale):
    """The logsumexp has f32's precision: no nibble * scale is rounded to f16 on the way to a logit. A logit is at most 17
    sums of exact products (16 dimensions at a time, scales in two parts), each off by 2^-23 of what has been added so far
    at most, which is of the logits' size: 2^-19 with the sums of the softmax. A rounding to f16 is off by 2^-16 and more."""
    lens, nq = [900, 300], [700, 150]
    cache, table, n = make(2, 2, dim, group, 16, lens, seed=31)
    cu = torch.tensor([0] + nq, device="cuda").cumsum(0).int()
    g = torch.Generator(device="cuda").manual_seed(dim)
    q = torch.randn(sum(nq), 6, dim, generator=g, device="cuda").bfloat16()
    _, lse = ops.kv4_attention(q, cache, table, n, cu_q=cu, scale=scale, want_lse=True)
    _, want, _, _ = reference(q, cache, table, n, cu, True, 0, dim ** -0.5 if scale is None else scale)
    assert float((lse.double() - want).norm() / want.norm()) <= 2.0 ** -19


def test_prompts_with_a_nan_in_a_token_of_one_scale():
    cache, table, n = make(1, 1, 64, 64, 16, [300], seed=6)
    j = 200
    cu = torch.tensor([0, 300], dtype=torch.int32, device="cuda")
    q = torch.randn(300, 2, 64, device="cuda").bfloat16()
    clean = ops.kv4_attention(q, cache, table, n, cu_q=cu)
    for which in (3, 2):
        keep = cache[which][int(table[0, j // 16]), 0, j % 16, 0].clone()
        for bad in (float("nan"), float("inf")):
            cache[which][int(table[0, j // 16]), 0, j % 16, 0] = bad
            out = ops.kv4_attention(q, cache, table, n, cu_q=cu)
            assert torch.equal(out[:j], clean[:j]) and not bool(torch.isfinite(out[j:]).any())
        cache[which][int(table[0, j // 16]), 0, j % 16, 0] = keep


@pytest.mark.parametrize("dim,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("ratio", [12, 29])
def test_prompts_of_many_rows(dim, group, ratio):
    """Enough rows that they are shared by tiles of 256 at either head size."""
    lens, nq = [900, 513, 300, 0, 128, 129], [900, 250, 1, 3, 128, 200]
    cache, table, n = make(6, 2, dim, group, 32, lens, seed=5)
    cu = torch.tensor([0] + nq, device="cuda").cumsum(0).int()
    for kind, window, causal in ((torch.bfloat16, 0, True), (torch.float16, 200, True), (torch.float16, 0, False)):
        q = torch.randn(sum(nq), 2 * ratio, dim, device="cuda").to(kind)
        check(q, cache, table, n, cu, causal, window)
    packed = torch.randn(sum(nq), 2 * ratio + 3, dim, device="cuda").half()
    out = torch.zeros_like(packed)
    ops.kv4_attention(packed[:, 2:-1], cache, table, n, cu_q=cu, out=out[:, 1:-2])
    assert torch.equal(out[:, 1:-2], check(packed[:, 2:-1], cache, table, n, cu))
    assert bool((out[:, 0] == 0).all()) and bool((out[:, -2:] == 0).all())


@pytest.mark.parametrize("dim,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("scale", [None, -0.2])
def test_prompts_of_many_rows_keep_the_logits_of_32_bits(dim, group, scale):
    """As test_prompts_keep_the_logits_of_32_bits: the same sums, the same bound."""
    cache, table, n = make(1, 1, dim, group, 16, [500], seed=31)
    cu = torch.tensor([0, 400], device="cuda").int()
    g = torch.Generator(device="cuda").manual_seed(dim)
    q = torch.randn(400, 45, dim, generator=g, device="cuda").bfloat16()
    _, lse = ops.kv4_attention(q, cache, table, n, cu_q=cu, scale=scale, want_lse=True)
    _, want, _, _ = reference(q, cache, table, n, cu, True, 0, dim ** -0.5 if scale is None else scale)
    assert float((lse.double() - want).norm() / want.norm()) <= 2.0 ** -19


def test_prompts_of_many_rows_with_scales_far_apart():
    cache, table, n = make(1, 1, 64, 32, 16, [700], seed=21, spread=4.0)
    j = torch.arange(700, device="cuda")
    page, at = table[0, j // 16].long(), j % 16
    cache[2][page, 0, at] *= (0.1 + j / 100)[:, None].half()
    cache[3][page, 0, at] *= (2.0 ** (12 * (j / 700 - 0.5).abs() - 8))[:, None].half()
    cu = torch.tensor([0, 700], device="cuda").int()
    check(torch.randn(700, 24, 64, device="cuda").bfloat16(), cache, table, n, cu, scale=0.125)
    check((torch.randn(700, 24, 64, device="cuda") * 1e30).bfloat16(), cache, table, n, cu, scale=1e-31)
    check((torch.randn(700, 24, 64, device="cuda") * 1e-3).half(), cache, table, n, cu, scale=-90.0)
    check(torch.zeros(700, 24, 64, device="cuda").half(), cache, table, n, cu)


@pytest.mark.parametrize("dim,group", [(64, 64), (128, 64)])
def test_prompts_of_many_rows_with_a_nan_and_pages_outside(dim, group):
    cache, table, n = make(1, 1, dim, group, 16, [300], seed=4)
    j = 200
    cu = torch.tensor([0, 300], dtype=torch.int32, device="cuda")
    q = torch.randn(300, 60, dim, device="cuda").bfloat16()
    clean = ops.kv4_attention(q, cache, table, n, cu_q=cu)
    for which in (3, 2):
        keep = cache[which][int(table[0, j // 16]), 0, j % 16, -1].clone()
        for bad in (float("nan"), float("inf")):
            cache[which][int(table[0, j // 16]), 0, j % 16, -1] = bad
            out = ops.kv4_attention(q, cache, table, n, cu_q=cu)
            assert torch.equal(out[:j], clean[:j])
            assert not bool(torch.isfinite(out[j:, :, -group:]).any())
        cache[which][int(table[0, j // 16]), 0, j % 16, -1] = keep
    bad = table.clone()
    bad[0, 3] = -1
    got = ops.kv4_attention(q, cache, bad, n, cu_q=cu)
    assert torch.equal(got[:48], clean[:48]) and bool(torch.isfinite(got).all())
    assert not torch.equal(got[64:], clean[64:])


def test_a_long_sequence_is_split_over_the_gpu():
    lens = [70001]
    cache, table, n = make(1, 1, 128, 128, 64, lens, seed=9)
    check(torch.randn(1, 8, 128, device="cuda").bfloat16(), cache, table, n)


def test_logits_far_apart_and_scales_far_apart():
    """A maximum that rises late by hundreds, and values whose scales grow by 2^12 along the sequence."""
    lens = [1000]
    cache, table, n = make(1, 1, 64, 32, 16, lens, seed=2, spread=6.0)
    j = torch.arange(1000, device="cuda")
    page, at = table[0, j // 16].long(), j % 16
    cache[2][page, 0, at] *= (0.1 + j / 100)[:, None].half()
    cache[3][page, 0, at] *= (2.0 ** (12 * j / 1000 - 10))[:, None].half()
    check(torch.randn(1, 4, 64, device="cuda").half(), cache, table, n)
    # every logit very negative, and a negative scale
    check(torch.randn(1, 4, 64, device="cuda").bfloat16() * 50, cache, table, n, scale=-3.0)
    # tiny and huge queries
    check(torch.randn(1, 4, 64, device="cuda").bfloat16() * 1e-30, cache, table, n)
    check((torch.randn(1, 4, 64, device="cuda") * 1e30).bfloat16(), cache, table, n, scale=1e-31)
    check(torch.zeros(1, 4, 64, device="cuda").bfloat16(), cache, table, n)


def test_a_nan_in_the_cache_reaches_only_the_rows_that_see_it():
    cache, table, n = make(1, 1, 64, 32, 16, [50], seed=4)
    j = 47
    cache[3][int(table[0, j // 16]), 0, j % 16, 1] = float("nan")
    cu = torch.tensor([0, 5], dtype=torch.int32, device="cuda")
    q = torch.randn(5, 2, 64, device="cuda").bfloat16()
    out = ops.kv4_attention(q, cache, table, n, cu_q=cu)
    assert bool(out[2:, :, 32:].isnan().all()) and not bool(out[2:, :, :32].isnan().any())
    assert not bool(out[:2].isnan().any())
    cache[2][int(table[0, j // 16]), 0, j % 16, 1] = float("nan")
    out = ops.kv4_attention(q, cache, table, n, cu_q=cu)
    assert bool(out[2:].isnan().all()) and not bool(out[:2].isnan().any())


def test_pages_outside_the_cache_are_left_out():
    cache, table, n = make(1, 2, 64, 32, 16, [100], seed=6)
    q = torch.randn(1, 4, 64, device="cuda").half()
    bad = table.clone()
    bad[0, 2], bad[0, 4] = -1, cache[0].shape[0]
    got, lse = ops.kv4_attention(q, cache, bad, n, want_lse=True)
    # the same tokens without those pages, in order: no position matters to one query
    kept = table[:, [0, 1, 3, 5, 6]].contiguous()
    want, want_lse = ops.kv4_attention(q, cache, kept, n - 32, want_lse=True)
    assert float((got.float() - want.float()).abs().max()) <= 2.0 ** -8
    assert float((lse - want_lse).abs().max()) <= 2.0 ** -16
    # lengths beyond the table, below zero, and query offsets outside q
    wide = ops.kv4_attention(q, cache, table[:, :3], torch.tensor([999], dtype=torch.int32, device="cuda"))
    assert torch.equal(wide, ops.kv4_attention(q, cache, table, torch.tensor([48], dtype=torch.int32, device="cuda")))
    none = ops.kv4_attention(q, cache, table, torch.tensor([-5], dtype=torch.int32, device="cuda"))
    assert bool((none == 0).all())
    cu = torch.tensor([0, 7], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.kv4_attention(q, cache, table, n, cu_q=cu), ops.kv4_attention(q, cache, table, n))


def test_strides_streams_and_repeated_launches():
    """Views, another stream with its own workspace, and shapes in turn on one workspace: the same bits every time."""
    lens = [300, 2000, 17, 1024]
    cache, table, n = make(4, 2, 128, 64, 32, lens, seed=8)
    packed = torch.randn(4, 20, 128, device="cuda").bfloat16()
    q = packed[:, 2:18]
    want = check(q, cache, table, n)
    assert torch.equal(ops.kv4_attention(q.contiguous(), cache, table, n), want)
    out = torch.zeros(4, 20, 128, device="cuda").bfloat16()
    ops.kv4_attention(q, cache, table, n, out=out[:, 3:19])
    assert torch.equal(out[:, 3:19], want) and bool((out[:, :3] == 0).all()) and bool((out[:, 19:] == 0).all())
    wide = torch.full((4, table.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    assert torch.equal(ops.kv4_attention(q, cache, wide[:, :table.shape[1]], n), want)
    cu = torch.tensor([0, 30, 30, 31, 60], dtype=torch.int32, device="cuda")
    q2 = torch.randn(60, 4, 128, device="cuda").half()
    want2 = check(q2, cache, table, n, cu)
    for _ in range(5):
        assert torch.equal(ops.kv4_attention(q, cache, table, n), want)
        assert torch.equal(ops.kv4_attention(q2, cache, table, n, cu_q=cu), want2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.kv4_attention(q, cache, table, n)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


def test_many_short_sequences_and_captured_launches():
    g = torch.Generator(device="cuda").manual_seed(11)
    lens = torch.randint(0, 40, (700,), generator=g, device="cuda").tolist()
    cache, table, n = make(700, 1, 64, 64, 8, [max(lens)] * 1 + lens[1:], seed=11)
    q = torch.randn(700, 2, 64, device="cuda").half()
    want = check(q, cache, table, n)
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ws = torch.zeros(_lib.load().up_sm100_kv4_attention_workspace_bytes(700, 2, 700, 1, 64), dtype=torch.uint8,
                         device="cuda")
        ops.kv4_attention(q, cache, table, n, out=out, ws=ws)
    for _ in range(2):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)


@pytest.mark.parametrize("nq", [1, 40])
def test_a_captured_step_of_wide_heads(nq):
    """Heads of 128 need more shared memory than a launch has by default: setting it must not break a capture."""
    cache, table, n = make(3, 2, 128, 64, 16, [500, 64, 300], seed=13)
    cu = torch.arange(4, device="cuda", dtype=torch.int32) * nq
    q = torch.randn(3 * nq, 8, 128, device="cuda").bfloat16()
    want = check(q, cache, table, n, cu)
    out = torch.empty_like(q)
    ws = torch.zeros(_lib.load().up_sm100_kv4_attention_workspace_bytes(3 * nq, 8, 3, 2, 128), dtype=torch.uint8,
                     device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.kv4_attention(q, cache, table, n, cu_q=cu, out=out, ws=ws)
    out.zero_()
    graph.replay()
    assert torch.equal(out, want)


def test_a_cache_that_passes_32_bits():
    """Pages above 2^32 bytes into the arrays."""
    page, kv, dim, group = 4096, 8, 128, 128
    pages = 2100  # 4.4 GB of keys
    cache = ops.kv4_cache(pages, kv, dim, page, group)
    x = torch.randn(2, 300, kv, dim, device="cuda").bfloat16()
    slots = (pages - 1) * page + torch.arange(300, device="cuda")
    ops.kv4_append(x[0], x[1], cache, slots)
    table = torch.tensor([[pages - 1]], dtype=torch.int32, device="cuda")
    check(torch.randn(1, 16, dim, device="cuda").bfloat16(), cache, table,
          torch.tensor([300], dtype=torch.int32, device="cuda"))


def test_refusals():
    cache, table, n = make(2, 2, 64, 32, 16, [20, 30])
    q = torch.randn(2, 4, 64, device="cuda").half()
    for bad in (lambda: ops.kv4_attention(q.float(), cache, table, n), lambda: ops.kv4_attention(q[0], cache, table, n),
                lambda: ops.kv4_attention(q[:, :3], cache, table, n), lambda: ops.kv4_attention(q[..., :32], cache, table, n),
                lambda: ops.kv4_attention(q[:1], cache, table, n), lambda: ops.kv4_attention(q, cache, table.long(), n),
                lambda: ops.kv4_attention(q, cache, table, n.long()), lambda: ops.kv4_attention(q, cache, table[:1], n),
                lambda: ops.kv4_attention(q, cache, table, n, window=-1),
                lambda: ops.kv4_attention(q, cache, table, n, cu_q=torch.zeros(2, dtype=torch.int32, device="cuda")),
                lambda: ops.kv4_attention(q, cache, table.cpu(), n),
                lambda: ops.kv4_attention(q, cache, table, n, out=torch.empty_like(q).float()),
                lambda: ops.kv4_attention(q, (cache[0], cache[1], cache[2], cache[3][:1]), table, n),
                lambda: ops.kv4_attention(q, (cache[0].transpose(0, 1), cache[1], cache[2], cache[3]), table, n),
                lambda: ops.kv4_append(q, q, cache, n), lambda: ops.kv4_append(q[:, :2].float(), q[:, :2], cache, n),
                lambda: ops.kv4_append(q[:, :2], q[:, :2], cache, n[:1]),
                lambda: ops.kv4_append(q[:, :2], q[:, :2], cache, n, table=torch.zeros(4, 64, device="cuda")),
                lambda: ops.kv4_append(q[:, :2], q[:, :2], cache, n, q_out=q)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        ops.kv4_attention(q.cpu(), cache, table, n)
    odd = torch.empty(2, 4, 67, device="cuda").half()[..., 1:65]
    with pytest.raises(_lib.UpError):  # query rows that are not 16-byte aligned
        ops.kv4_attention(odd, cache, table, n)
    small = torch.zeros(256, dtype=torch.uint8, device="cuda")
    with pytest.raises(_lib.UpError):  # a workspace that is too small
        ops.kv4_attention(q, cache, table, n, ws=small)
    for pages, kv, dim, page, group in ((2, 2, 64, 12, 32), (2, 2, 64, 4, 32), (2, 2, 288, 16, 32), (2, 2, 48, 16, 48)):
        c = ops.kv4_cache(pages, kv, dim, page, group)
        x = torch.randn(2, 2, dim, device="cuda").half()
        with pytest.raises(_lib.UpError):
            ops.kv4_append(x, x, c, n)
        with pytest.raises(_lib.UpError):
            ops.kv4_attention(x, c, table, n)


@pytest.mark.parametrize("dim,group", [(64, 64), (128, 128), (96, 32), (256, 256)])
def test_an_infinite_key_scale_makes_its_logit_nan(dim, group):
    """A nibble of 0 times it is NaN, so the rows that see the token are, whatever the sign of the other products."""
    cache, table, n = make(1, 1, dim, group, 16, [200], seed=8)
    cu = torch.tensor([0, 4], device="cuda").int()
    q = torch.randn(4, 16, dim, device="cuda").bfloat16()
    cache[2][int(table[0, 198 // 16]), 0, 198 % 16, 0] = float("inf")
    out = ops.kv4_attention(q, cache, table, n, cu_q=cu)
    assert bool(out[2:].isnan().all()) and not bool(out[:2].isnan().any())


@pytest.mark.parametrize("dim,group", [(64, 32), (128, 128)])
def test_many_sequences_of_many_rows(dim, group):
    """More sequences than a warp looks through at once, empty ones among them; no wait inside the launch ran out."""
    g = torch.Generator().manual_seed(dim)
    lens = torch.randint(0, 300, (70,), generator=g).tolist()
    nq = torch.randint(0, 35, (70,), generator=g).tolist()
    lens[3] = nq[5] = nq[69] = 0
    cache, table, n = make(70, 1, dim, group, 16, lens, seed=12)
    cu = torch.tensor([0] + nq, device="cuda").cumsum(0).int()
    for kind in (torch.bfloat16, torch.float16):
        check(torch.randn(sum(nq), 16, dim, device="cuda").to(kind), cache, table, n, cu)
    ops.check_workspace("kv4", cache[0].device)
