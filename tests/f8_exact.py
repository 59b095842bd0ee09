"""The 8-bit operators and the experts' routing from their definitions, in 64 bits, on the CPU or the GPU."""
import torch

BLOCK = 128
F8 = torch.float8_e4m3fn
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # relative
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}  # of the subnormals


def blocks(n):
    return -(-n // BLOCK)


def product(x, xs, w, ws):
    """(exact product, sum of the terms' magnitudes) in f64 of x [m, k] and w [n, k] with their scales."""
    k, n = x.shape[1], w.shape[0]
    a = x.double() * xs.double().repeat_interleave(BLOCK, 1)[:, :k]
    b = w.double() * ws.double().repeat_interleave(BLOCK, 1)[:, :k].repeat_interleave(BLOCK, 0)[:n]
    return a @ b.T, a.abs() @ b.abs().T


def product_bound(exact, size, k, dtype):
    """How far a product may be from the exact one. Its 8-bit products are exact in f32 (4 bits by 4). A block's 128 are added
    by the tensor core in f32, in an order and with a rounding that are its own: at most a whole step (2^-23) of a partial sum
    each, and a partial sum is at most the sum of magnitudes. The block's sum times the product of two scales is added to the
    row's: three roundings of half a step for the block and one for each block after it. Then half a step of the output."""
    steps = BLOCK * 2.0 ** -23 + (3 + blocks(k)) * 2.0 ** -24
    return steps * size + HALF_STEP[dtype] * (exact.abs() + steps * size) + SMALLEST[dtype]


def by_expert(x, xs, w, ws, offsets):
    """The same by expert: rows offsets[e] to offsets[e + 1], each held to [0, m] and to its predecessors; None for the others."""
    m, n = x.shape[0], w.shape[1]
    out = torch.full((m, n), float("nan"), dtype=torch.float64, device=x.device)
    size = torch.zeros_like(out)
    at = 0
    bounds = []
    for o in offsets.tolist():
        at = max(at, min(max(o, 0), m))
        bounds.append(at)
    for e in range(w.shape[0]):
        lo, hi = bounds[e], bounds[e + 1]
        if hi > lo:
            out[lo:hi], size[lo:hi] = product(x[lo:hi], xs[lo:hi], w[e], ws[e])
    return out, size, bounds


def quantised(y, high=1):
    """(values, scales) of f32 rows y by the stated f32 operations; blocks of high x 128."""
    n, k = y.shape
    values = torch.empty_like(y)
    scale = torch.empty(-(-n // high), blocks(k), dtype=torch.float32, device=y.device)
    for i in range(scale.shape[0]):
        for b in range(scale.shape[1]):
            part = y[i * high:(i + 1) * high, b * BLOCK:(b + 1) * BLOCK]
            fine = part.isfinite()
            a = torch.where(fine, part.abs(), torch.zeros_like(part)).max()
            s = a * torch.tensor(1.0 / 448.0, dtype=torch.float32, device=y.device)
            s = s if float(s) >= 2.0 ** -126 else torch.zeros_like(s)
            v = part * (1.0 / s) if float(s) > 0 else torch.zeros_like(part)
            v = torch.where(fine, v, torch.full_like(v, float("nan")))
            values[i * high:(i + 1) * high, b * BLOCK:(b + 1) * BLOCK] = v
            scale[i, b] = s
    return values.to(F8), scale


def routed(logits, k, score, renormalise, gain=1.0):
    """(ids, weights in f64, rows, slots, offsets), token by token in plain Python."""
    t, e = logits.shape
    l = logits.double().cpu()
    ids = torch.full((t, k), -1, dtype=torch.int32)
    weights = torch.zeros(t, k, dtype=torch.float64)
    for i in range(t):
        row = l[i].tolist()
        order = [j for j in range(e) if row[j] != float("-inf")]
        order.sort(key=lambda j: (0 if row[j] != row[j] else 1, -row[j] if row[j] == row[j] else 0.0, j))
        order = order[:k]
        if not order:
            continue
        s = torch.sigmoid(l[i]) if score == "sigmoid" else torch.softmax(l[i], 0)
        got = s[order]
        if renormalise:
            if score == "softmax":
                got = torch.softmax(l[i][order], 0)  # the same, also where the others' sum has no number
            else:
                got = got / got.sum() if float(got.sum()) != 0 else torch.zeros_like(got)
        ids[i, :len(order)] = torch.tensor(order, dtype=torch.int32)
        weights[i, :len(order)] = got * gain
    rows = torch.full((t * k,), -1, dtype=torch.int32)
    slots = torch.full((t, k), -1, dtype=torch.int32)
    offsets = torch.zeros(e + 1, dtype=torch.int32)
    place = 0
    taken = [[] for _ in range(e)]
    for i in range(t):
        for j in range(k):
            if ids[i, j] >= 0:
                taken[int(ids[i, j])].append((i, j))
    for x in range(e):
        offsets[x] = place
        for i, j in taken[x]:
            rows[place] = i
            slots[i, j] = place
            place += 1
    offsets[e] = place
    return ids, weights, rows, slots, offsets
