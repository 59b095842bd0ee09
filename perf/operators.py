"""Cases and measurement of the serving operators: rotary positions, the 4-bit paged key/value cache and the
attention that reads it.

With `own` false, `run` computes the plain form: elementary torch operations in 32 bits, rounded once at the end. With
`own` true it makes the calls of unpopped_b200.ops that a user's program makes. `exact` gives the same outputs from the
operators' definitions in 64 bits.

Formulas. Rotation by position p of the pairs (i, i + R/2) ("half") or (2i, 2i + 1) ("interleaved") of a head's first R
dimensions, with c = table[p, i] and s = table[p, R/2 + i]: y0 = x0 c - x1 s, y1 = x1 c + x0 s; its gradient is the
transposed map. A cache row keeps D values as int4 with one f16 scale a group: scale = f16(max|x| / 7), value =
round(x / scale). Attention of query token i of a sequence with nq query tokens and L cached ones sees the tokens
j <= L - nq + i, and of these the last `window` where a window is given.
"""
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
N_POS = 32768


# ---- cases ----
def listed():
    return [
        # one token of one sequence: 64 query heads of an 8192-wide model; the call's latency is what counts
        dict(name="rope_one_token", op="rope", tokens=1, heads=64, dim=128, rot=128, layout="half", type="bf16",
             backward=False),
        # a training step's queries, 4 sequences of 4096 tokens: forward, and the gradient back through the rotation
        dict(name="rope_train", op="rope", tokens=16384, heads=64, dim=128, rot=128, layout="half", type="bf16",
             backward=True),
        # part of a head rotated in neighbouring pairs, a head size and a token count that are no powers of two
        dict(name="rope_partial_interleaved", op="rope", tokens=1999, heads=24, dim=96, rot=32, layout="interleaved",
             type="f32", backward=True),
        # a decode step's one sequence: 64 query heads over 8 key/value heads
        dict(name="append_one", op="append", tokens=1, heads=64, kv=8, dim=128, rot=128, layout="half", type="bf16",
             group=32, page=16, prompt=False),
        # a decode step of a batch, each token on a page of its own; a few slots are padding
        dict(name="append_batch", op="append", tokens=96, heads=32, kv=8, dim=128, rot=128, layout="half",
             type="bf16", group=128, page=16, prompt=False),
        # prompts going in: whole pages, half of each head rotated
        dict(name="append_prompt", op="append", tokens=16001, heads=64, kv=8, dim=128, rot=64, layout="half",
             type="f16", group=64, page=64, prompt=True),
        # one short sequence, one token: latency
        dict(name="attend_one", op="attend", batch=1, heads=64, kv=8, dim=128, group=32, page=16, lo=777, hi=777,
             q_lo=1, q_hi=1, window=0, type="bf16"),
        # a batch of ordinary ragged lengths, an empty one among them
        dict(name="attend_batch", op="attend", batch=64, heads=32, kv=8, dim=128, group=128, page=16, lo=0, hi=4096,
             q_lo=1, q_hi=1, window=0, type="bf16"),
        # one long sequence: its length has to be split over the GPU
        dict(name="attend_long", op="attend", batch=1, heads=64, kv=8, dim=128, group=64, page=64, lo=131071,
             hi=131071, q_lo=1, q_hi=1, window=0, type="bf16"),
        # the largest decode step: 32 long contexts
        dict(name="attend_large", op="attend", batch=32, heads=64, kv=8, dim=128, group=128, page=32, lo=8000,
             hi=16384, q_lo=1, q_hi=1, window=0, type="bf16"),
        # several tokens a sequence checked at once, small heads, a sliding window
        dict(name="attend_verify", op="attend", batch=24, heads=24, kv=8, dim=64, group=32, page=16, lo=100, hi=6000,
             q_lo=1, q_hi=5, window=4096, type="f16"),
        # prompts: long runs of query tokens over a cache that holds an earlier part too
        dict(name="attend_prompt", op="attend", batch=3, heads=32, kv=8, dim=128, group=128, page=64, lo=2049,
             hi=4096, q_lo=1500, q_hi=2048, window=0, type="bf16"),
    ]


def _log_int(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]; odd, so never whole tiles, where it is large."""
    n = max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))
    return n if n < 1024 else (n - 1) | 1


def draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend"])
    kv = rng.choice([1, 2, 4, 8])
    ratio = rng.choice([1, 2, 3, 4, 8])
    kind = rng.choice(["bf16", "f16"])
    if op == "rope":
        dim = rng.choice([64, 80, 96, 128, 256])
        rot = rng.choice([dim, dim // 2, 32])
        return dict(op=op, tokens=_log_int(rng, 1, 16384), heads=rng.choice([1, 8, 12, 24, 32, 40]), dim=dim, rot=rot,
                    layout=rng.choice(["half", "interleaved"]), type=rng.choice(["bf16", "f16", "f32"]),
                    backward=rng.random() < 0.5)
    dim = rng.choice([64, 96, 128, 256])
    group = rng.choice([g for g in (32, 64, 128, dim) if dim % g == 0])
    page = rng.choice([8, 16, 32, 64, 128])
    if op == "append":
        prompt = rng.random() < 0.5
        return dict(op=op, tokens=_log_int(rng, 1, 16000 if prompt else 256), heads=kv * ratio, kv=kv, dim=dim,
                    rot=rng.choice([dim, dim // 2, 32]), layout=rng.choice(["half", "interleaved"]), type=kind,
                    group=group, page=page, prompt=prompt)
    way = rng.choice(["decode", "decode", "verify", "prompt"])
    case = dict(op=op, heads=kv * ratio, kv=kv, dim=dim, group=group, page=page, type=kind,
                window=rng.choice([0, 0, _log_int(rng, 16, 4096)]))
    if way == "prompt":
        hi = _log_int(rng, 64, min(2048, 2048 * 4096 // max(4096, kv * ratio * dim)))
        return dict(case, batch=rng.randint(1, 4), lo=hi // 2, hi=(hi + rng.randint(0, 1000)) | 1, q_lo=max(1, hi // 3),
                    q_hi=hi)
    batch = _log_int(rng, 1, 128)
    hi = _log_int(rng, 1, max(2, min(131072, 350000 // batch * 128 // dim)))
    q = 1 if way == "decode" else rng.randint(2, 8)
    return dict(case, batch=batch, lo=rng.choice([0, 1, hi // 2, hi]), hi=hi, q_lo=1, q_hi=q)


def _spread(n, lo, hi):
    """n whole numbers from lo to hi in even steps."""
    return [hi] if n == 1 else [lo + (i * (hi - lo)) // (n - 1) for i in range(n)]


def _lengths(case):
    """(cached tokens, query tokens) of every sequence, before their order is shuffled."""
    return _spread(case["batch"], case["lo"], case["hi"]), _spread(case["batch"], case["q_lo"], case["q_hi"])


def work(case):
    if case["op"] == "rope":
        one = case["tokens"] * case["heads"] * case["dim"] * SIZE[case["type"]]
        n = 2 if case["backward"] else 1
        rows = min(case["tokens"], N_POS) * (case["rot"] * 4 + 8)
        return {"bytes": n * (2 * one + rows), "flops": n * 3 * case["tokens"] * case["heads"] * case["rot"]}
    row = case["dim"] // 2 + 2 * (case["dim"] // case["group"])  # a cached row: its values and its scales
    if case["op"] == "append":
        t, h, kv, d = case["tokens"], case["heads"], case["kv"], case["dim"]
        slots = _pages(case) * case["page"]
        bytes_ = t * (h + 2 * kv) * d * 2 + t * h * d * 2 + 2 * t * kv * row + t * (case["rot"] * 4 + 16)
        # the outputs: the cache as the values that it stands for
        return {"bytes": bytes_ + 2 * slots * kv * (row + 2 * d), "flops": t * ((h + kv) * 3 * case["rot"] + 4 * kv * d)}
    lens, queries = _lengths(case)
    seen = cached = 0
    for n, q in zip(lens, queries):
        first = max(0, n - q + 1 - case["window"]) if case["window"] else 0
        cached += max(0, n - first)
        for i in range(q):
            last = n - q + i + 1
            seen += max(0, min(last, case["window"]) if case["window"] else last)
    t = sum(queries)
    return {"bytes": 2 * cached * case["kv"] * row + 2 * t * case["heads"] * case["dim"] * 2,
            "flops": 4 * seen * case["heads"] * case["dim"]}


# ---- inputs ----
def _table(rot):
    """cos and sin of N_POS positions, as a program makes them once."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    a = torch.arange(N_POS, device=DEV, dtype=torch.float64)[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float()


def _cache(g, pages, case, k_size=1.0):
    """A cache of normally distributed keys and values: (k, v, k_scale, v_scale)."""
    kv, page, dim, group = case["kv"], case["page"], case["dim"], case["group"]

    def packed():
        n = torch.randn(pages, kv, page, dim, generator=g, device=DEV, dtype=torch.float16)
        n = n.mul_(2.6).round_().clamp_(-8, 7).to(torch.int8)
        return ((n[..., 0::2] & 15) | (n[..., 1::2] << 4)).view(torch.uint8)

    def scales(size):
        u = torch.rand(pages, kv, page, dim // group, generator=g, device=DEV)
        return ((0.32 + 0.12 * u) * size).to(torch.float16)

    return packed(), packed(), scales(k_size), scales(1.0)


def _pages(case):
    need = -(-case["tokens"] // case["page"]) if case["prompt"] else case["tokens"]
    return need + 3


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    kind = TYPES[case["type"]]
    if case["op"] == "rope":
        shape = (case["tokens"], case["heads"], case["dim"])
        # queries lie beside keys and values in one projection's output
        x = torch.randn(shape[0], shape[1] + 2, shape[2], generator=g, device=DEV).to(kind)[:, :shape[1]]
        grad = torch.randn(shape, generator=g, device=DEV).to(kind) if case["backward"] else None
        pos = torch.randint(0, N_POS, (shape[0],), generator=g, device=DEV)
        return dict(case=case, x=x, grad=grad, pos=pos, table=_table(case["rot"]))
    if case["op"] == "append":
        t, h, kv, page = case["tokens"], case["heads"], case["kv"], case["page"]
        qkv = torch.randn(t, h + 2 * kv, case["dim"], generator=g, device=DEV).to(kind)
        order = torch.randperm(_pages(case), generator=g, device=DEV)
        at = torch.arange(t, device=DEV)
        if case["prompt"]:
            slots = order[at // page] * page + at % page
            pos = at % N_POS
        else:
            slots = order[at] * page + torch.randint(0, page, (t,), generator=g, device=DEV)
            pos = torch.randint(0, N_POS, (t,), generator=g, device=DEV)
        if t >= 16:
            slots[-(t // 16):] = -1  # a batch padded to a fixed size
        return dict(case=case, q=qkv[:, :h], k=qkv[:, h:h + kv], v=qkv[:, h + kv:], pos=pos, slots=slots,
                    table=_table(case["rot"]), cache=_cache(g, _pages(case), case))
    lens, queries = _lengths(case)
    b, page = case["batch"], case["page"]
    order = torch.randperm(b, generator=g, device=DEV)
    lens_t = torch.tensor(lens, device=DEV, dtype=torch.int32)[order]
    q_t = torch.tensor(queries, device=DEV, dtype=torch.int32)[order]
    width = max(1, -(-max(lens) // page))
    pages = b * width
    blocks = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).view(b, width)
    cu = None
    if case["q_hi"] > 1:
        cu = torch.zeros(b + 1, device=DEV, dtype=torch.int32)
        cu[1:] = q_t.cumsum(0)
    q = torch.randn(sum(queries), case["heads"], case["dim"], generator=g, device=DEV)
    q = (q * (0.5 + 2 * torch.rand(1, case["heads"], 1, generator=g, device=DEV))).to(kind)
    return dict(case=case, q=q, cache=_cache(g, pages, case), blocks=blocks, lens=lens_t, cu=cu)


# ---- the plain forms ----
def _rotated(x, pos, table, layout, rot, back=False):
    c, s = table[pos, None, :rot // 2], table[pos, None, rot // 2:]
    if back:
        s = -s
    x = x.float()
    if layout == "half":
        a, b, rest = x[..., :rot // 2], x[..., rot // 2:rot], x[..., rot:]
        return torch.cat([a * c - b * s, b * c + a * s, rest], -1)
    a, b, rest = x[..., 0:rot:2], x[..., 1:rot:2], x[..., rot:]
    return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), rest], -1)


def _values(packed, scale):
    """The 32-bit values of int4 rows [..., n/2] with scales [..., n/group]."""
    n = torch.stack([packed << 4, packed & 0xF0], -1).view(torch.int8) >> 4
    shape = scale.shape + (-1,)
    return (n.reshape(shape).float() * scale[..., None].float()).flatten(-2)


def _quantised(x, group):
    """(packed int4, f16 scales) of the rows of x."""
    x = x.unflatten(-1, (-1, group))
    scale = (x.abs().amax(-1) * (1.0 / 7.0)).clamp(max=65504.0).to(torch.float16)
    f = scale.float()[..., None]
    n = torch.where(f > 0, (x * (1.0 / f)).round().clamp(-8, 7), torch.zeros_like(x)).to(torch.int8).flatten(-2)
    return ((n[..., 0::2] & 15) | (n[..., 1::2] << 4)).view(torch.uint8), scale


def _plain_append(st):
    case = st["case"]
    q = _rotated(st["q"], st["pos"], st["table"], case["layout"], case["rot"]).to(st["q"].dtype)
    k = _rotated(st["k"], st["pos"], st["table"], case["layout"], case["rot"])
    new = _quantised(k, case["group"]) + _quantised(st["v"].float(), case["group"])
    slots, page = st["slots"], case["page"]
    # padding goes to a row of its own past the cache, which is dropped again
    at = torch.where(slots >= 0, slots, st["cache"][0].shape[0] * page)
    cache = []
    for old, rows in zip(st["cache"], (new[0], new[2], new[1], new[3])):
        flat = old.transpose(1, 2).flatten(0, 1)
        flat = torch.cat([flat, flat[:1]])
        flat[at] = rows
        cache.append(flat[:-1].unflatten(0, (-1, page)).transpose(1, 2))
    return {"q": q, "k": _values(cache[0], cache[2]).to(torch.bfloat16),
            "v": _values(cache[1], cache[3]).to(torch.bfloat16)}


def _plain_attend(st):
    case = st["case"]
    k4, v4, ks, vs = st["cache"]
    blocks, lens, cu, q = st["blocks"].long(), st["lens"].long(), st["cu"], st["q"]
    b, kv, dim, r = case["batch"], case["kv"], case["dim"], case["heads"] // case["kv"]
    n, nq = blocks.shape[1] * case["page"], case["q_hi"]

    def rows(packed, scale):  # [batch, kv heads, tokens, dim] in the sequences' order
        return _values(packed[blocks], scale[blocks]).transpose(1, 2).reshape(b, kv, n, dim)

    if cu is None:
        own_q = torch.ones_like(lens)
        first = torch.arange(b, device=DEV)
    else:
        own_q = (cu[1:] - cu[:-1]).long()
        first = cu[:-1].long()
    i = torch.arange(nq, device=DEV)
    take = (first[:, None] + i).clamp(max=q.shape[0] - 1)
    qp = q[take].float().unflatten(2, (kv, r)).permute(0, 2, 3, 1, 4).reshape(b, kv, r * nq, dim)
    s = torch.matmul(qp, rows(k4, ks).transpose(2, 3)).mul_(dim ** -0.5).view(b, kv, r, nq, n)
    last = (lens - own_q)[:, None, None] + i[:, None]  # the newest token that a query sees
    j = torch.arange(n, device=DEV)
    see = (j <= last) & (j < lens[:, None, None])
    if case["window"]:
        see &= j > last - case["window"]
    s.masked_fill_(~see[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, kv, r * nq, n), rows(v4, vs)).view(b, kv, r, nq, dim)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = m + total.log()
    t = torch.arange(q.shape[0], device=DEV)
    seq = torch.searchsorted(first.contiguous(), t, right=True) - 1
    at = t - first[seq]
    o = o.permute(0, 3, 1, 2, 4)[seq, at].flatten(1, 2).to(q.dtype)
    return {"out": o, "lse": lse[..., 0].permute(0, 3, 1, 2)[seq, at].flatten(1, 2)}


def run(state):
    case = state["case"]
    if not own:
        if case["op"] == "append":
            return _plain_append(state)
        if case["op"] == "attend":
            return _plain_attend(state)
        out = {"y": _rotated(state["x"], state["pos"], state["table"], case["layout"], case["rot"]).to(
            state["x"].dtype)}
        if case["backward"]:
            out["dx"] = _rotated(state["grad"], state["pos"], state["table"], case["layout"], case["rot"],
                                 True).to(state["x"].dtype)
        return out
    from unpopped_b200 import ops

    if case["op"] == "rope":
        out = {"y": ops.rope(state["x"], state["pos"], state["table"], case["layout"])}
        if case["backward"]:
            out["dx"] = ops.rope_backward(state["grad"], state["pos"], state["table"], case["layout"])
        return out
    if case["op"] == "append":
        q = ops.kv4_append(state["k"], state["v"], state["cache"], state["slots"], state["pos"], state["table"],
                           q=state["q"], layout=case["layout"])
        k4, v4, ks, vs = state["cache"]
        rows, groups = k4.numel() // k4.shape[-1], ks.shape[-1]
        shape = k4.shape[:-1] + (case["dim"],)
        return {"q": q,
                "k": ops.dequant_i4(k4.view(rows, -1), ks.view(rows, groups), case["group"]).view(shape),
                "v": ops.dequant_i4(v4.view(rows, -1), vs.view(rows, groups), case["group"]).view(shape)}
    o, lse = ops.kv4_attention(state["q"], state["cache"], state["blocks"], state["lens"], cu_q=state["cu"],
                               window=case["window"], want_lse=True)
    return {"out": o, "lse": lse}


# ---- the definitions in 64 bits ----
def _pairs(rot, layout):
    i = torch.arange(rot // 2, device=DEV)
    return (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)


def _turn(x, pos, table, layout, rot, sign=1.0):
    i0, i1 = _pairs(rot, layout)
    y = x.double().clone()
    angle = table.double()[pos]
    c, s = angle[:, None, : rot // 2], sign * angle[:, None, rot // 2:]
    x0, x1 = y[..., i0], y[..., i1]
    y[..., i0], y[..., i1] = x0 * c - x1 * s, x0 * s + x1 * c
    return y


def _unpacked(packed, scale):
    """64-bit values of whole cache arrays, from their bytes' two's complement nibbles."""
    b = packed.long()
    low, high = b % 16, b // 16
    n = torch.empty(b.shape[:-1] + (2 * b.shape[-1],), device=DEV, dtype=torch.float64)
    n[..., 0::2] = torch.where(low > 7, low - 16, low).double()
    n[..., 1::2] = torch.where(high > 7, high - 16, high).double()
    return n * scale.double().repeat_interleave(n.shape[-1] // scale.shape[-1], -1)


def _exact_append(st):
    case = st["case"]
    page, group = case["page"], case["group"]
    out = {"q": _turn(st["q"], st["pos"], st["table"], case["layout"], case["rot"])}
    new = {"k": _turn(st["k"], st["pos"], st["table"], case["layout"], case["rot"]), "v": st["v"].double()}
    for name, packed, scale in (("k", st["cache"][0], st["cache"][2]), ("v", st["cache"][1], st["cache"][3])):
        values = _unpacked(packed, scale)
        x = new[name].unflatten(-1, (-1, group))
        step = (x.abs().amax(-1, keepdim=True) / 7).clamp(max=65504.0).half().double()
        rows = torch.where(step > 0, (x / step).round().clamp(-8, 7) * step, torch.zeros_like(x)).flatten(-2)
        keep = st["slots"] >= 0
        slot = st["slots"][keep]
        values[slot // page, :, slot % page] = rows[keep]
        out[name] = values
    return out


def _exact_attend(st):
    case = st["case"]
    k4, v4, ks, vs = st["cache"]
    q, r, window = st["q"].double(), case["heads"] // case["kv"], case["window"]
    lens = st["lens"].tolist()
    cu = list(range(case["batch"] + 1)) if st["cu"] is None else st["cu"].tolist()
    out = torch.zeros(q.shape, device=DEV, dtype=torch.float64)
    lse = torch.full(q.shape[:2], float("-inf"), device=DEV, dtype=torch.float64)
    for b, n in enumerate(lens):
        nq = cu[b + 1] - cu[b]
        if n == 0 or nq == 0:
            continue
        pages = st["blocks"][b, : -(-n // case["page"])].long()
        for h in range(case["kv"]):
            k = _unpacked(k4[pages, h], ks[pages, h]).flatten(0, 1)[:n]
            v = _unpacked(v4[pages, h], vs[pages, h]).flatten(0, 1)[:n]
            at = torch.arange(n, device=DEV)
            newest = n - nq + torch.arange(nq, device=DEV)[:, None]
            see = at <= newest
            if window:
                see &= newest - at < window
            rows = q[cu[b]:cu[b + 1], h * r:(h + 1) * r]
            s = torch.einsum("qrd,kd->rqk", rows, k) / float(case["dim"]) ** 0.5
            s = torch.where(see, s, torch.full_like(s, float("-inf")))
            z = torch.logsumexp(s, -1)
            w = torch.where(see & (z > float("-inf"))[..., None], torch.exp(s - z[..., None]), torch.zeros_like(s))
            out[cu[b]:cu[b + 1], h * r:(h + 1) * r] = torch.einsum("rqk,kd->qrd", w, v)
            lse[cu[b]:cu[b + 1], h * r:(h + 1) * r] = z.T
    return {"out": out, "lse": lse}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rope":
        out = {"y": _turn(st["x"], st["pos"], st["table"], case["layout"], case["rot"])}
        if case["backward"]:
            out["dx"] = _turn(st["grad"], st["pos"], st["table"], case["layout"], case["rot"], -1.0)
        return out
    return _exact_append(st) if case["op"] == "append" else _exact_attend(st)
