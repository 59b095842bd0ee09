"""Cases and measurement of the operators of an 8-bit mixture-of-experts layer: routing, quantisation in blocks of 128, the
matrix product of 8-bit values (dense, and grouped by expert) and the weighted sum of the experts' rows.

With `own` false, `run` computes the plain form: elementary torch operations in 32 bits, rounded once at the end. With
`own` true it makes the calls of unpopped_b200.ops that a user's program makes. `exact` gives the same outputs from the
operators' definitions in 64 bits.

Formulas. Routing takes for each token the k largest logits (ties to the lowest expert; an expert whose logit is -inf is
never taken, and a token short of experts gets -1 with weight 0). Their weights are exp(l - max) / sum or 1 / (1 + exp(-l)),
divided by the chosen ones' sum where that is asked for. The pairs (token, expert) are then laid out by expert, in each by
token: rows[slot] is the slot's token, slots[token, j] the pair's place, offsets where the experts begin. Quantisation in groups of
128 values of a row (of 128 x 128 for weights): scale = max|y| / 448, value = e4m3(y / scale). The product is
out[m, n] = sum over blocks b of 128: x_scale[m, b] w_scale[n / 128, b] sum over k in b: x[m, k] w[n, k]; grouped, rows
offsets[e] to offsets[e + 1] take w[e]. The sum is out[t] = add[t] + sum over j: weights[t, j] y[slots[t, j]].
"""
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
F8 = torch.float8_e4m3fn
BLOCK = 128
SMALLEST = 2.0 ** -126  # a group whose scale would be below it is held as zeros


# ---- cases ----
def listed():
    return [
        # one token's routing: the call's latency is what counts
        dict(name="route_one", op="route", tokens=1, experts=128, k=8, type="f32", score="softmax", renormalise=True),
        # a prompt's tokens; some are padding, whose logits are all -inf
        dict(name="route_prompt", op="route", tokens=16384, experts=256, k=8, type="f32", score="sigmoid",
             renormalise=True),
        # one token's activations of an 8192-wide model
        dict(name="quantise_one", op="quantise", rows=1, size=8192, type="bf16", form="plain"),
        # between an expert's two products: gate and up projections of a prompt's pairs, multiplied and quantised
        dict(name="quantise_gate", op="quantise", rows=32768, size=2048, type="bf16", form="gate"),
        # one token through the largest projection of the benchmark's width: every weight is read once
        dict(name="f8_one_token", op="matmul", rows=1, n=28672, size=8192, type="bf16"),
        # a batch of odd sizes: no whole tile in any direction
        dict(name="f8_batch_odd", op="matmul", rows=61, n=4111, size=2064, type="bf16"),
        # a long prompt: the tensor cores' rate
        dict(name="f8_prompt", op="matmul", rows=8192, n=8192, size=8192, type="bf16"),
        # one token's eight experts: eight groups of one row
        dict(name="experts_one", op="experts", tokens=1, k=8, experts=128, n=4096, size=2048, type="bf16"),
        # a decode step of a batch: nearly every expert has a few rows, and all weights are read
        dict(name="experts_batch", op="experts", tokens=64, k=8, experts=128, n=4096, size=2048, type="bf16"),
        # a prompt: ragged groups of some hundred rows
        dict(name="experts_prompt", op="experts", tokens=8192, k=8, experts=128, n=4096, size=2048, type="bf16"),
        # a batch's eight rows a token back in one, with the residual added
        dict(name="combine_batch", op="combine", tokens=64, k=8, n=8192, type="bf16", add=True),
        # a prompt's
        dict(name="combine_prompt", op="combine", tokens=8192, k=8, n=4096, type="bf16", add=False),
    ]


def _log_int(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["route", "quantise", "matmul", "matmul", "experts", "experts", "combine"])
    if op == "route":
        experts = rng.choice([8, 16, 60, 64, 128, 160, 256])
        return dict(op=op, tokens=_log_int(rng, 1, 16384), experts=experts, k=rng.choice([1, 2, 4, 6, 8]),
                    type=rng.choice(["f32", "bf16", "f16"]), score=rng.choice(["softmax", "sigmoid"]),
                    renormalise=rng.random() < 0.5)
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "quantise":
        form = rng.choice(["plain", "rows", "gate", "weight"])
        size = 16 * _log_int(rng, 8, 512)
        return dict(op=op, rows=_log_int(rng, 1, min(32768, (1 << 26) // size)), size=size, type=kind, form=form)
    if op == "combine":
        n = 8 * _log_int(rng, 8, 1024)
        k = rng.choice([1, 2, 4, 6, 8])
        return dict(op=op, tokens=_log_int(rng, 1, min(8192, (1 << 28) // (n * k))), k=k, n=n, type=kind,
                    add=rng.random() < 0.5)
    size = 16 * _log_int(rng, 8, 512)
    if op == "matmul":
        n = _log_int(rng, 64, 28672)
        if rng.random() < 0.5:
            n = (n + 127) // 128 * 128
        return dict(op=op, rows=_log_int(rng, 1, min(8192, (1 << 39) // (n * size))), n=n, size=size, type=kind)
    experts = rng.choice([4, 8, 16, 60, 64, 128])
    n = 8 * _log_int(rng, 16, 512)
    return dict(op=op, tokens=_log_int(rng, 1, max(2, min(8192, (1 << 36) // (n * size)))), k=rng.choice([1, 2, 4]),
                experts=experts, n=n, size=size, type=kind)


def _blocks(n):
    return -(-n // BLOCK)


def work(case):
    op = case["op"]
    one = SIZE[case["type"]]
    if op == "route":
        t, e, k = case["tokens"], case["experts"], case["k"]
        return {"bytes": t * e * one + t * k * 16 + (e + 1) * 4, "flops": 4 * t * e}
    if op == "quantise":
        r, n = case["rows"], case["size"]
        per = 2 if case["form"] == "gate" else 1
        scales = _blocks(n) * (_blocks(r) if case["form"] == "weight" else r)
        read = (-(-r // 4) if case["form"] == "rows" else r) * n * per * one
        return {"bytes": read + r * n + 4 * scales + (4 * r if case["form"] == "rows" else 0),
                "flops": r * n * (8 if case["form"] == "gate" else 3)}
    if op == "combine":
        t, k, n = case["tokens"], case["k"], case["n"]
        return {"bytes": t * n * one * (k + 1 + case["add"]) + t * k * 8, "flops": 2 * t * k * n}
    n, size = case["n"], case["size"]
    rows = case["rows"] if op == "matmul" else case["tokens"] * case["k"]
    # experts that some token takes, as many as are expected where each is as likely
    used = 1 if op == "matmul" else case["experts"] * (1 - (1 - case["k"] / case["experts"]) ** case["tokens"])
    weights = used * (n * size + 4 * _blocks(n) * _blocks(size))
    return {"bytes": int(weights + rows * (size + 4 * _blocks(size)) + rows * n * one), "flops": 2 * rows * n * size}


# ---- inputs ----
def _codes(g, *shape):
    """8-bit values as quantisation leaves them: normally distributed, the group's largest near 448."""
    x = torch.randn(*shape, generator=g, device=DEV, dtype=torch.float16)
    return x.mul_(150).clamp_(-448, 448).to(F8)


def _scales(g, *shape, size=1.0):
    u = torch.rand(*shape, generator=g, device=DEV)
    return (0.5 + u) * size


def _chosen(g, tokens, experts, k):
    """[tokens, k] distinct experts of each token, some experts far more wanted than others."""
    want = 0.7 * torch.randn(experts, generator=g, device=DEV)
    u = torch.rand(tokens, experts, generator=g, device=DEV).clamp_(1e-7, 1 - 1e-7)
    return (want - (-u.log()).log()).topk(k, 1).indices


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    op, kind = case["op"], TYPES[case["type"]]
    if op == "route":
        t, e = case["tokens"], case["experts"]
        logits = torch.randn(t, e, generator=g, device=DEV) + 0.7 * torch.randn(e, generator=g, device=DEV)
        if t >= 16:
            logits[-(t // 16):] = float("-inf")  # a batch padded to a fixed size
        return dict(case=case, logits=logits.to(kind))
    if op == "quantise":
        r, n = case["rows"], case["size"]
        tokens = -(-r // 4) if case["form"] == "rows" else r
        x = torch.randn(tokens, n * (2 if case["form"] == "gate" else 1), generator=g, device=DEV)
        x *= torch.exp(torch.randn(tokens, 1, generator=g, device=DEV))
        x[:, :: max(1, n // 64)] *= 8  # a few columns are far larger than the others
        rows = torch.randint(0, tokens, (r,), generator=g, device=DEV, dtype=torch.int32)
        return dict(case=case, x=x.to(kind), rows=rows if case["form"] == "rows" else None)
    if op == "combine":
        t, k, n = case["tokens"], case["k"], case["n"]
        slots = torch.randperm(t * k, generator=g, device=DEV).to(torch.int32).view(t, k)
        weights = torch.rand(t, k, generator=g, device=DEV)
        if t >= 16:
            slots[-(t // 16):] = -1  # padding, and a few pairs that no expert took
            slots[0, -1] = -1
        return dict(case=case, y=torch.randn(t * k, n, generator=g, device=DEV).to(kind), slots=slots,
                    weights=weights / weights.sum(1, keepdim=True),
                    add=torch.randn(t, n, generator=g, device=DEV).to(kind) if case["add"] else None)
    n, size = case["n"], case["size"]
    nb, kb = _blocks(n), _blocks(size)
    if op == "matmul":
        m = case["rows"]
        # the scales lie as quantisation leaves them: a group of 128 after the other, each with all rows
        return dict(case=case, x=_codes(g, m, size), xs=_scales(g, kb, m, size=0.01).t(), w=_codes(g, n, size),
                    ws=_scales(g, nb, kb, size=1e-4))
    e, m = case["experts"], case["tokens"] * case["k"]
    sizes = torch.bincount(_chosen(g, case["tokens"], e, case["k"]).flatten(), minlength=e)
    offsets = torch.zeros(e + 1, dtype=torch.int32, device=DEV)
    offsets[1:] = sizes.cumsum(0)
    return dict(case=case, x=_codes(g, m, size), xs=_scales(g, kb, m, size=0.01).t(), w=_codes(g, e, n, size),
                ws=_scales(g, e, nb, kb, size=1e-4), offsets=offsets, most=int(sizes.max()))


# ---- the plain forms ----
def _plain_route(st):
    case, l = st["case"], st["logits"].float()
    t, e, k = case["tokens"], case["experts"], case["k"]
    top, ids = torch.sort(l, dim=1, descending=True, stable=True)
    top, ids = top[:, :k], ids[:, :k]
    there = top != float("-inf")
    if case["score"] == "softmax":
        m = l.amax(1, keepdim=True)
        m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
        w, total = (top - m).exp(), (l - m).exp().sum(1, keepdim=True)
    else:
        w, total = 1.0 / (1.0 + (-top).exp()), 1.0
    w = torch.where(there, w, torch.zeros_like(w))
    if case["renormalise"]:
        total = w.sum(1, keepdim=True)
    w = w / total
    w = torch.where(there, w, torch.zeros_like(w))
    # by expert, in each by token; pairs that are not there come last
    key = torch.where(there, ids, torch.full_like(ids, e)).flatten()
    order = torch.sort(key, stable=True).indices
    sizes = torch.zeros(e + 1, dtype=torch.int64, device=DEV).index_add_(0, key, torch.ones_like(key))[:e]
    offsets = torch.zeros(e + 1, dtype=torch.int32, device=DEV)
    offsets[1:] = sizes.cumsum(0)
    at = torch.arange(t * k, device=DEV)
    rows = torch.where(at < offsets[-1], order // k, torch.full_like(order, -1)).to(torch.int32)
    slots = torch.empty_like(at)
    slots[order] = at
    slots = torch.where(there.flatten(), slots, torch.full_like(slots, -1)).to(torch.int32).view(t, k)
    ids = torch.where(there, ids, torch.full_like(ids, -1)).to(torch.int32)
    return {"ids": ids, "weights": w, "rows": rows, "slots": slots, "offsets": offsets}


def _padded(y, dims):
    """y with zeros up to whole blocks of 128 in each of its dims."""
    pad = []
    for d in (-1, -2)[:dims]:
        pad += [0, -y.shape[d] % BLOCK]
    return torch.nn.functional.pad(y, pad)


def _quantised(y, group):
    """(values as e4m3, scales) of f32 groups, the dims `group` of y being one group."""
    a = y.abs()
    fine = a < float("inf")
    s = torch.where(fine, a, torch.zeros_like(a)).amax(group, keepdim=True) * (1.0 / 448.0)
    s = torch.where(s >= SMALLEST, s, torch.zeros_like(s))
    v = torch.where(s > 0, y * (1.0 / s), torch.zeros_like(y))
    return torch.where(fine, v, torch.full_like(v, float("nan"))), s


def _plain_quantise(st):
    case, x = st["case"], st["x"].float()
    n = case["size"]
    if case["form"] == "rows":
        x = x[st["rows"].long()]
    if case["form"] == "gate":
        x = x[:, :n] / (1.0 + (-x[:, :n]).exp()) * x[:, n:]
    if case["form"] == "weight":
        y = _padded(x, 2).unflatten(1, (-1, BLOCK)).unflatten(0, (-1, BLOCK))
        v, s = _quantised(y, (1, 3))
        return {"q": v.flatten(2).flatten(0, 1)[: x.shape[0], :n].contiguous().to(F8), "scale": s[:, 0, :, 0]}
    v, s = _quantised(_padded(x, 1).unflatten(1, (-1, BLOCK)), 2)
    return {"q": v.flatten(1)[:, :n].contiguous().to(F8), "scale": s[..., 0]}


def _spread(s, dim, n):
    return s.repeat_interleave(BLOCK, dim).narrow(dim, 0, n)


def _plain_matmul(st):
    case = st["case"]
    n, size, kind = case["n"], case["size"], TYPES[case["type"]]
    x = st["x"].float() * _spread(st["xs"], 1, size)
    w = st["w"].float() * _spread(_spread(st["ws"], -1, size), -2, n)
    if case["op"] == "matmul":
        return {"out": torch.matmul(x, w.t()).to(kind)}
    # every expert's rows, padded to as many as the largest group has
    at = torch.arange(x.shape[0], device=DEV)
    e = torch.searchsorted(st["offsets"][1:].contiguous(), at, right=True)
    place = at - st["offsets"].long()[e]
    rows = torch.zeros(case["experts"], st["most"], size, device=DEV)
    rows[e, place] = x
    return {"out": torch.matmul(rows, w.transpose(1, 2))[e, place].to(kind)}


def _plain_combine(st):
    case, slots = st["case"], st["slots"].long()
    w = torch.where(slots >= 0, st["weights"], torch.zeros_like(st["weights"]))
    rows = st["y"][slots.clamp(min=0)].float()
    out = (rows * w[..., None]).sum(1)
    if case["add"]:
        out = out + st["add"].float()
    return {"out": out.to(TYPES[case["type"]])}


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"route": _plain_route, "quantise": _plain_quantise, "matmul": _plain_matmul, "experts": _plain_matmul,
                "combine": _plain_combine}[op](state)
    from unpopped_b200 import ops

    kind = TYPES[case["type"]]
    if op == "route":
        ids, weights, rows, slots, offsets = ops.expert_route(state["logits"], case["k"], score=case["score"],
                                                              renormalise=case["renormalise"])
        return {"ids": ids, "weights": weights, "rows": rows, "slots": slots, "offsets": offsets}
    if op == "quantise":
        if case["form"] == "weight":
            q, scale = ops.f8_quantise_weight(state["x"])
        else:
            q, scale = ops.f8_quantise(state["x"], rows=state["rows"], gate=case["form"] == "gate")
        return {"q": q, "scale": scale}
    if op == "matmul":
        return {"out": ops.f8_matmul(state["x"], state["xs"], state["w"], state["ws"], dtype=kind)}
    if op == "experts":
        return {"out": ops.f8_expert_matmul(state["x"], state["xs"], state["w"], state["ws"], state["offsets"],
                                            dtype=kind)}
    return {"out": ops.expert_combine(state["y"], state["slots"], state["weights"], add=state["add"])}


# ---- the definitions in 64 bits ----
def _exact_route(st):
    case, l = st["case"], st["logits"].double()
    t, e, k = case["tokens"], case["experts"], case["k"]
    left = l.clone()
    ids = torch.full((t, k), -1, dtype=torch.int32, device=DEV)
    w = torch.zeros((t, k), dtype=torch.float64, device=DEV)
    index = torch.arange(e, device=DEV)
    score = torch.sigmoid(l) if case["score"] == "sigmoid" else torch.softmax(l, 1)
    for j in range(k):  # the largest one left, the first of equals
        best = left.amax(1, keepdim=True)
        i = torch.where(left == best, index, torch.full_like(index, e)).amin(1)
        got = best[:, 0] > float("-inf")
        ids[:, j] = torch.where(got, i, torch.full_like(i, -1)).to(torch.int32)
        w[:, j] = torch.where(got, score.gather(1, i.clamp(max=e - 1)[:, None])[:, 0], w[:, j])
        left.scatter_(1, i.clamp(max=e - 1)[:, None], float("-inf"))
    if case["renormalise"]:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, w)
    return {"ids": None, "weights": w, "rows": None, "slots": None, "offsets": None}


def _to_e4m3(v):
    """The nearest e4m3 value (ties to even), in 64 bits: 4 bits of precision down to 2^-6, steps of 2^-9 below."""
    e = torch.frexp(v.abs().clamp(min=2.0 ** -6)).exponent.double() - 1
    step = torch.exp2(e - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def _exact_quantise(st):
    case, x = st["case"], st["x"].double()
    n, form = case["size"], case["form"]
    if form == "rows":
        x = x.index_select(0, st["rows"].long())
    if form == "gate":
        x = x[:, :n] * torch.sigmoid(x[:, :n]) * x[:, n:]
    q = torch.empty_like(x)
    high = BLOCK if form == "weight" else 1
    scale = torch.empty(-(-x.shape[0] // high), _blocks(n), dtype=torch.float64, device=DEV)
    for b in range(_blocks(n)):
        part = x[:, b * BLOCK:(b + 1) * BLOCK]
        a = part.abs().amax(1)
        if form == "weight":
            a = torch.stack([c.amax() for c in a.split(BLOCK)])
        scale[:, b] = a / 448
        s = scale[:, b].repeat_interleave(high)[: x.shape[0], None]
        q[:, b * BLOCK:(b + 1) * BLOCK] = torch.where(s > 0, _to_e4m3(part / s), torch.zeros_like(part))
    return {"q": q, "scale": scale}


def _exact_product(x, xs, w, ws):
    """Block by block, the scales outside of each block's sum."""
    out = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device=DEV)
    column = torch.arange(w.shape[0], device=DEV) // BLOCK
    for b in range(_blocks(x.shape[1])):
        part = x[:, b * BLOCK:(b + 1) * BLOCK].double() @ w[:, b * BLOCK:(b + 1) * BLOCK].double().T
        out += part * xs[:, b, None].double() * ws[column, b].double()
    return out


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "route":
        return _exact_route(st)
    if op == "quantise":
        return _exact_quantise(st)
    if op == "matmul":
        return {"out": _exact_product(st["x"], st["xs"], st["w"], st["ws"])}
    if op == "experts":
        at = st["offsets"].tolist()
        parts = [_exact_product(st["x"][a:b], st["xs"][a:b], st["w"][e], st["ws"][e])
                 for e, (a, b) in enumerate(zip(at, at[1:])) if b > a]
        return {"out": torch.cat(parts)}
    out = st["add"].double() if case["add"] else torch.zeros(case["tokens"], case["n"], dtype=torch.float64, device=DEV)
    for j in range(case["k"]):
        slot = st["slots"][:, j].long()
        row = st["y"].index_select(0, slot.clamp(min=0)).double() * st["weights"][:, j, None].double()
        out = out + torch.where(slot[:, None] >= 0, row, torch.zeros_like(row))
    return {"out": out}
