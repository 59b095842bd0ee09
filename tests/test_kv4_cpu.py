"""The serving operators' host side on the CPU: refusals through the C ABI (nothing is launched), workspace sizes, the
interface artifacts, and the index rules of the kernels restated in Python."""
import ctypes
import os
import random

import pytest

from unpopped_b200 import _lib
from unpopped_b200._lib import EK, UP_ERR_INVALID, UP_ERR_UNSUPPORTED, UP_OK, UpKv4Cache
from unpopped_b200.interface import kernel_interface

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "unpopped_b200", "csrc")
P = 1 << 20  # an aligned address that is never read: every call here is refused, or has nothing to do


def cache(**kw):
    d = dict(k=P, v=P, k_scale=P, v_scale=P, pages=4, kv_heads=2, page=16, dim=64, group=32)
    d.update(kw)
    return UpKv4Cache(*d.values())


def rope(**kw):
    a = dict(x=P, dtype=EK["F16"], batch=0, seq=4, heads=2, dim=64, xb=512, xs=128, xh=64, pos=P, kind=EK["I64"], pb=0,
             table=P, n_pos=8, rot=64, layout=0, backward=0, out=P, ob=512, os=128, oh=64, stream=None)
    a.update(kw)
    return _lib.load().up_sm100_rope(*a.values())


def append(c=None, **kw):
    a = dict(q=P, k=P, v=P, dtype=EK["F16"], tokens=0, heads=2, qt=128, qh=64, kt=128, kh=64, vt=128, vh=64, pos=P,
             pos_kind=EK["I32"], table=P, n_pos=8, rot=64, layout=0, slots=P, slot_kind=EK["I32"], cache=c or cache(),
             out=P, ot=128, oh=64, stream=None)
    a.update(kw)
    a["cache"] = ctypes.byref(a["cache"])
    return _lib.load().up_sm100_kv4_append(*a.values())


def attention(c=None, **kw):
    a = dict(q=P, dtype=EK["F16"], tokens=0, heads=4, qt=256, qh=64, cache=c or cache(), table=P, ts=4, tw=4, lens=P, cu=P,
             batch=3, causal=1, window=0, scale=1.0, out=P, ot=256, oh=64, lse=None, lt=4, ws=P, wb=1 << 40, stream=None)
    a.update(kw)
    a["cache"] = ctypes.byref(a["cache"])
    return _lib.load().up_sm100_kv4_attention(*a.values())


def test_nothing_to_do_is_ok():
    assert rope() == UP_OK and append() == UP_OK and attention() == UP_OK
    assert rope(batch=2, heads=0) == UP_OK and attention(tokens=2, batch=0) == UP_OK
    assert _lib.load().up_sm100_rope_table(None, 0, 64, 10000.0, 0, 1.0, 0.0, 0.0, 0.0, 1.0, None) == UP_OK


@pytest.mark.parametrize("kw,want", [
    (dict(seq=-1), UP_ERR_INVALID), (dict(rot=65), UP_ERR_INVALID), (dict(rot=66), UP_ERR_INVALID),
    (dict(rot=-2), UP_ERR_INVALID), (dict(layout=2), UP_ERR_UNSUPPORTED), (dict(kind=EK["U32"]), UP_ERR_UNSUPPORTED),
    (dict(batch=1, x=None), UP_ERR_INVALID), (dict(batch=1, out=None), UP_ERR_INVALID),
    (dict(batch=1, table=None), UP_ERR_INVALID), (dict(batch=1, oh=63), UP_ERR_INVALID),
    (dict(batch=1, os=0), UP_ERR_INVALID), (dict(batch=1, xs=-1), UP_ERR_INVALID),
    (dict(batch=1, dtype=EK["I32"]), UP_ERR_UNSUPPORTED), (dict(batch=1, dtype=EK["F64"]), UP_ERR_UNSUPPORTED)])
def test_rope_refusals(kw, want):
    assert rope(**kw) == want


@pytest.mark.parametrize("kw,want", [
    (dict(dim=48), UP_ERR_UNSUPPORTED), (dict(dim=288), UP_ERR_UNSUPPORTED), (dict(dim=0), UP_ERR_UNSUPPORTED),
    (dict(group=16), UP_ERR_UNSUPPORTED), (dict(group=0), UP_ERR_UNSUPPORTED), (dict(dim=128, group=96), UP_ERR_UNSUPPORTED),
    (dict(page=4), UP_ERR_UNSUPPORTED), (dict(page=24), UP_ERR_UNSUPPORTED), (dict(page=8192), UP_ERR_UNSUPPORTED),
    (dict(pages=-1), UP_ERR_INVALID), (dict(kv_heads=0), UP_ERR_INVALID), (dict(k=None), UP_ERR_INVALID),
    (dict(v_scale=P + 8), UP_ERR_INVALID)])
def test_cache_refusals(kw, want):
    assert append(cache(**kw)) == want
    assert attention(cache(**kw)) == want


@pytest.mark.parametrize("kw,want", [
    (dict(tokens=-1), UP_ERR_INVALID), (dict(dtype=EK["F32"]), UP_ERR_UNSUPPORTED), (dict(layout=7), UP_ERR_UNSUPPORTED),
    (dict(slot_kind=EK["U32"]), UP_ERR_UNSUPPORTED), (dict(pos_kind=EK["F32"]), UP_ERR_UNSUPPORTED),
    (dict(rot=80), UP_ERR_INVALID), (dict(rot=7), UP_ERR_INVALID), (dict(tokens=1, k=None), UP_ERR_INVALID),
    (dict(tokens=1, slots=None), UP_ERR_INVALID), (dict(tokens=1, q=None), UP_ERR_INVALID),
    (dict(tokens=1, out=None), UP_ERR_INVALID), (dict(tokens=1, pos=None), UP_ERR_INVALID),
    (dict(tokens=1, oh=32), UP_ERR_INVALID), (dict(tokens=2, ot=8), UP_ERR_INVALID), (dict(kt=-1), UP_ERR_INVALID),
    (dict(tokens=1 << 31), UP_ERR_UNSUPPORTED)])
def test_append_refusals(kw, want):
    assert append(**kw) == want


@pytest.mark.parametrize("kw,want", [
    (dict(tokens=-1), UP_ERR_INVALID), (dict(window=-1), UP_ERR_INVALID), (dict(dtype=EK["F32"]), UP_ERR_UNSUPPORTED),
    (dict(heads=3), UP_ERR_UNSUPPORTED), (dict(cu=None, tokens=2), UP_ERR_INVALID), (dict(tokens=3, q=None), UP_ERR_INVALID),
    (dict(tokens=3, out=None), UP_ERR_INVALID), (dict(tokens=3, lens=None), UP_ERR_INVALID),
    (dict(tokens=3, table=None), UP_ERR_INVALID), (dict(tokens=3, ws=None), UP_ERR_INVALID),
    (dict(tokens=3, ws=P + 16), UP_ERR_INVALID), (dict(tokens=3, wb=4096), UP_ERR_INVALID),
    (dict(tokens=3, ts=3), UP_ERR_INVALID), (dict(tokens=3, oh=32), UP_ERR_INVALID), (dict(tokens=3, ot=32), UP_ERR_INVALID),
    (dict(tokens=3, lse=P, lt=3), UP_ERR_INVALID), (dict(tokens=3, q=P + 8), UP_ERR_UNSUPPORTED),
    (dict(tokens=3, qh=65), UP_ERR_UNSUPPORTED), (dict(tokens=3, out=P + 2), UP_ERR_UNSUPPORTED),
    (dict(tokens=3, oh=66), UP_ERR_UNSUPPORTED), (dict(tokens=(1 << 29) + 1), UP_ERR_UNSUPPORTED),
    (dict(tokens=3, tw=(1 << 26) + 1, ts=1 << 27), UP_ERR_UNSUPPORTED)])
def test_attention_refusals(kw, want):
    assert attention(**kw) == want


def test_table_refusals():
    t = _lib.load().up_sm100_rope_table
    for args, want in (((P, 8, 15, 1e4, 0, 1.0, 0.0, 0.0, 0.0), UP_ERR_INVALID), ((P, 8, 16, 1.0, 0, 1.0, 0.0, 0.0, 0.0), UP_ERR_INVALID),
                       ((P, 8, 16, 1e4, 5, 1.0, 0.0, 0.0, 0.0), UP_ERR_UNSUPPORTED), ((P, 8, 16, 1e4, 1, 0.0, 0.0, 0.0, 0.0), UP_ERR_INVALID),
                       ((P, 8, 16, 1e4, 3, 2.0, 4.0, 1.0, 64.0), UP_ERR_INVALID), ((None, 8, 16, 1e4, 0, 1.0, 0.0, 0.0, 0.0), UP_ERR_INVALID)):
        assert t(*args, 1.0, None) == want


def test_workspace_grows_with_the_rows_of_a_tile_only():
    w = _lib.load().up_sm100_kv4_attention_workspace_bytes
    assert w(0, 8, 4, 2, 128) == w(4, 8, 0, 2, 128) < w(4, 8, 4, 2, 64) < w(4, 8, 4, 2, 128)
    assert w(4, 8, 4, 2, 128) == w(4000, 8, 4000, 2, 128)       # 4 rows a sequence and key/value head
    assert w(4, 8, 4, 2, 128) < w(12, 8, 4, 2, 128)             # 12: a second column group


@pytest.mark.parametrize("kid,src", [(17, "rope.cu"), (18, "kv4_append.cu"), (19, "kv4_attention.cu")])
def test_interfaces(kid, src):
    assert kid in _lib.SERVING_KERNEL.values()
    ki = kernel_interface(kid)
    assert ki.entry_symbol == "up_sm100_" + src[:-3] and "sm_100a" in ki.requires
    assert all({"name", "role", "elem"} <= set(p) for p in ki.params)
    h = 0xCBF29CE484222325
    for b in open(os.path.join(CSRC, src), "rb").read():
        h = ((h ^ b) * 0x100000001B3) & 0xFFFFFFFFFFFFFFFF
    assert ki.revision_hash == h


def test_division_by_multiplication():
    """Divide32 of divide.cuh: exact for every dividend below 2^31, and no intermediate passes 32 bits."""
    rng = random.Random(1)
    for d in list(range(1, 2000)) + [rng.randrange(1, 2 ** 31) for _ in range(2000)] + [2 ** 30, 2 ** 30 + 1, 2 ** 31 - 1]:
        s = 0
        while (1 << s) < d:
            s += 1
        m = (((((1 << s) - d) << 32) // d) + 1) & 0xFFFFFFFF
        for x in [0, 1, d - 1, d, d + 1, 2 ** 31 - 1] + [rng.randrange(2 ** 31) for _ in range(10)]:
            if x < 2 ** 31:
                t = ((m * x) >> 32) + x
                assert t < 2 ** 32 and t >> s == x // d


@pytest.mark.parametrize("q,rows", [(24001, 8000), (0, 5), (5, 0), (7, 3), (3, 7), (1, 1), (5, 5), (100, 1), (1, 100)])
def test_the_append_blocks_alternate_over_every_block_once(q, rows):
    few_are_queries = q < rows
    few = q if few_are_queries else rows
    period = (q + rows) // few if few else 1
    got = {True: [], False: []}
    for block in range(q + rows):
        run = block // period
        rare = run < few and block - run * period == period - 1
        got[rare == few_are_queries].append(run if rare else block - min(run, few))
    assert sorted(got[True]) == list(range(q)) and sorted(got[False]) == list(range(rows))


def test_the_split_gives_every_unit_to_one_cta_and_every_part_its_counter():
    """The shares of kv4_split.cuh: each CTA's range in the space of tile costs and units, the parts that a split tile
    waits for, and the two part slots and three counters a CTA has."""
    cost, group = 2, 16
    rng = random.Random(2)
    for _ in range(300):
        tiles = [rng.choice([1, 1, 2, 3, 7, 40, 300]) for _ in range(rng.randrange(1, 40))]
        U, grid = sum(tiles) + cost * len(tiles), rng.choice([1, 5, 37, 592])
        P = min(grid, U)
        each, extra = U // P, U - U // P * P
        begin = lambda c: c * each + min(c, extra)  # noqa: E731
        cta_of = lambda u: u // (each + 1) if u < extra * (each + 1) else extra + (u - extra * (each + 1)) // each  # noqa: E731
        starts, at = [], 0
        for n in tiles:
            starts.append(at)
            at += n + cost
        seen, parts = [[] for _ in tiles], set()
        arrivals = {}
        for c in range(P):
            u, u1 = begin(c), begin(c + 1)
            assert u1 > u
            while u < u1:
                i = max(k for k in range(len(tiles)) if starts[k] <= u)
                pos, n = u - starts[i], tiles[i]
                take = min(n + cost - pos, u1 - u)
                first, count = max(pos - cost, 0), max(pos + take - cost, 0) - max(pos - cost, 0)
                u += take
                if count == 0:
                    continue
                seen[i] += range(first, first + count)
                if first == 0 and count == n:
                    continue
                c0, c1 = cta_of(starts[i] + cost), cta_of(starts[i] + cost + n - 1)
                assert c0 <= c <= c1 and (first == 0) == (c == c0)
                slot = (c, 0 if first > 0 else 1)
                assert slot not in parts
                parts.add(slot)
                mine = (c - c0) // group
                counter = (0 if mine == 0 else 1, c0 + mine * group)
                arrivals.setdefault(counter, []).append((i, min(group, c1 - c0 + 1 - mine * group)))
        assert all(s == list(range(n)) for s, n in zip(seen, tiles))
        for users in arrivals.values():  # one tile a counter, and it is met exactly as often as it is waited for
            assert len({i for i, _ in users}) == 1 and all(of == len(users) for _, of in users)


def test_the_calls_refuse_tensors_that_are_not_on_a_gpu():
    torch = pytest.importorskip("torch")
    from unpopped_b200 import ops

    x = torch.zeros(2, 2, 64)
    cache = tuple(torch.zeros(2, 2, 16, n, dtype=t) for n, t in ((32, torch.uint8), (32, torch.uint8), (2, torch.float16),
                                                                   (2, torch.float16)))
    lens = torch.zeros(2, dtype=torch.int32)
    for bad in (lambda: ops.rope(x, None, torch.zeros(4, 64)), lambda: ops.rope("x", None, torch.zeros(4, 64)),
                lambda: ops.rope_backward(x, None, torch.zeros(4, 64)), lambda: ops.kv4_append(x, x, cache, lens),
                lambda: ops.kv4_attention(x, cache, lens.view(2, 1), lens),
                lambda: ops.dequant_i4(cache[0].view(64, 32), cache[2].view(64, 2), 32)):
        with pytest.raises(TypeError):
            bad()
