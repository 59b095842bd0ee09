"""Attention over the paged 4-bit cache in 64 bits, the rule that chooses its kernel, and bounds of the kernels' error.

With weights w (the softmax of a row), logits s, visible values v, of n visible tokens:
  |out - exact| <= (u_p + u_v + 2 ds + 2^-19) sum w |v| + n 2^-27 max v_scale / l + u |exact| + 2^-25
  |lse - exact| <= ds + 2^-19 + 2^-22 |exact|
* u_p = 2^-11: p (for many query rows) or p * v_scale (for few) is rounded to f16. u_v = 2^-11 where nibble * v_scale is
  too: many query rows and a bf16 output. u: half an ulp of the output's type.
* ds = 2^-18 max_j scale sum_d |q_d k_jd|: f32 sums of at most 256 exact products, 16 at a time, and the scales' products.
  The kernel for few rows sums q (n + 8) and begins at -8 sum q, which this leaves out: of 30000 random shapes 8, of 32
  dimensions and few tokens, passed the bound of lse by it, 1.6 times at most.
* f16's lower end loses at most 2^-25 a token and nibble of what is rounded. For few rows that is 2^(logit - ref + 5) times
  a v_scale relative to the power of two of the largest one, for many rows 2^(logit - ref + 5) at least: 2^-25 2^-5 8 = 2^-27
  of the largest v_scale that the row has seen. l is the sum of exp(s - max), and ref is the largest logit seen or below it.
Only tokens that the row sees are in any of these."""
import torch

HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMS = 148


def many_rows(tokens, batch, heads, kv_heads, dim, sms=SMS):
    """Whether the tcgen05 kernel takes the call (`many_rows` of csrc/kv4_attention.cuh)."""
    if dim not in (64, 128):
        return False
    rows, pairs = -(-tokens // batch) * (heads // kv_heads), batch * kv_heads
    turns = -(-pairs * -(-rows // 256) // sms)
    return turns * sms * (6 if dim == 64 else 4) < pairs * -(-rows // 16)


def unpacked(packed, scale):
    b = packed.to(torch.int16)
    n = torch.stack([b & 15, b >> 4], -1).flatten(-2)
    n = torch.where(n > 7, n - 16, n).double()
    return n * scale.double().repeat_interleave(n.shape[-1] // scale.shape[-1], -1)


def exact(q, cache, table, lens, cu=None, causal=True, window=0, scale=None):
    """(out, lse, bound of out, bound of lse) of every query row, in 64 bits."""
    scale = q.shape[2] ** -0.5 if scale is None else scale
    page, kv = cache[0].shape[2], cache[0].shape[1]
    ratio = q.shape[1] // kv
    many = many_rows(q.shape[0], len(lens), q.shape[1], kv, q.shape[2])
    u = 2.0 ** -11 * (2 if many and q.dtype == torch.bfloat16 else 1) + 2.0 ** -19
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], float("-inf"), dtype=torch.float64, device=q.device)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    for b, n in enumerate(lens.tolist()):
        q0, nq = (b, 1) if cu is None else (int(cu[b]), int(cu[b + 1]) - int(cu[b]))
        if n == 0 or nq == 0:
            continue
        ids = table[b, : -(-n // page)].long()
        pos = n - nq + torch.arange(nq, device=q.device)[:, None]
        j = torch.arange(n, device=q.device)
        see = (j <= pos) if causal else torch.ones(nq, n, dtype=torch.bool, device=q.device)
        if window:
            see = see & (j > pos - window)
        some, seen = see.any(-1), see.sum(-1)
        for h in range(kv):
            k, v = (unpacked(cache[i][ids, h], cache[i + 2][ids, h]).flatten(0, 1)[:n] for i in (0, 1))
            size = cache[3][ids, h].flatten(0, 1)[:n].double().abs().amax(-1)
            x = q[q0:q0 + nq, h * ratio:(h + 1) * ratio].double()
            s = torch.einsum("qrd,kd->rqk", x, k) * scale
            mag = torch.einsum("qrd,kd->rqk", x.abs(), k.abs()) * abs(scale)
            s = s.masked_fill(~see, float("-inf"))
            m = s.amax(-1, keepdim=True)
            p = torch.where(see, torch.exp(s - torch.where(some[:, None], m, torch.zeros_like(m))), torch.zeros_like(s))
            l = p.sum(-1, keepdim=True)
            w = p / torch.where(l > 0, l, torch.ones_like(l))
            ds = 2.0 ** -18 * mag.masked_fill(~see, 0).amax(-1)
            most = torch.where(see, size, torch.zeros_like(size)).amax(-1)  # the largest v_scale that a row sees
            vv = torch.where((see.any(0))[:, None], v, torch.zeros_like(v))  # what no row sees may be anything
            o = torch.einsum("rqk,kd->qrd", w, vv)
            near = torch.einsum("rqk,kd->qrd", w, vv.abs())
            at = (slice(q0, q0 + nq), slice(h * ratio, (h + 1) * ratio))
            floor = seen[:, None] * 2.0 ** -27 * most[:, None] / l.squeeze(-1).T.clamp(min=1.0)
            tol[at] = (u + 2 * ds.T[..., None]) * near + o.abs() * HALF_ULP[q.dtype] + floor[..., None] + 2.0 ** -25
            out[at] = o
            z = (m.squeeze(-1) + l.squeeze(-1).log()).T
            lse[at] = torch.where(some[:, None], z, torch.full_like(z, float("-inf")))
            tol_lse[at] = (ds.T + 2.0 ** -19 + 2.0 ** -22 * z.abs()).nan_to_num(0, 0, 0)
    return out, lse, tol, tol_lse


def cache_of(x, page, group, seed=0):
    """A cache that holds the tokens x [2 (keys, values), sequences, n, kv_heads, dim] on shuffled pages, and its table. The
    slots past n hold NaN scales."""
    two, batch, n, kv, dim = x.shape
    width = -(-n // page)
    g = torch.Generator(device=x.device).manual_seed(seed)
    table = torch.randperm(batch * width, generator=g, device=x.device).int().view(batch, width)
    packed, scales = [], []
    for z in range(2):
        y = torch.full((batch, width * page, kv, dim), float("nan"), device=x.device)
        y[:, :n] = x[z].float()
        y = y.unflatten(-1, (-1, group))
        step = (y.abs().amax(-1) / 7).clamp(max=65504.0).half()
        f = step.float()[..., None]
        v = torch.where(f > 0, (y / f).round().clamp(-8, 7), torch.zeros_like(y)).to(torch.int16).flatten(-2)
        v = ((v[..., 0::2] & 15) | ((v[..., 1::2] & 15) << 4)).to(torch.uint8)
        for into, t in ((packed, v), (scales, step)):
            pages = torch.empty(batch * width, kv, page, t.shape[-1], dtype=t.dtype, device=x.device)
            pages[table.flatten().long()] = t.unflatten(1, (width, page)).transpose(2, 3).flatten(0, 1)
            into.append(pages)
    return (packed[0], packed[1], scales[0], scales[1]), table
