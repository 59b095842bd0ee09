"""The schedule of the 8-bit products' tiles, the kernel's own code on the host: every group of every tile has one owner, the parts of a tile are
as many as its counter waits for, and no counter or place of a part is used twice."""
import random

import pytest

import f8_walk


def check(name, begin, n, k, sms, panel=1 << 30):
    """Returns (owners of each tile, tiles that each owner has parts of)."""
    f = f8_walk.FORMS.index(name)
    owners = max(1, sms // f8_walk.CTAS[f])
    groups = -(-(-(-k // 128)) // f8_walk.GROUP[f])
    tb = -(-n // f8_walk.WEIGHTS[f])
    seen, places, parts, counters = {}, set(), {}, {}
    joins = []
    for o in range(owners):
        first = last = 0
        mine = set()
        for t, g0, g1, e, w, m0, rows, c0, c1 in f8_walk.runs(name, begin, n, k, o, owners, panel).tolist():
            assert 0 <= g0 < g1 <= groups and 0 <= w < tb and 0 < rows <= f8_walk.TOKENS[f]
            assert begin[e] <= m0 and m0 + rows <= begin[e + 1]
            seen.setdefault(t, []).append((g0, g1))
            places.add((t, e, w, m0, rows))
            if g0 > 0 or g1 < groups:
                assert c0 <= o <= c1 < owners
                parts.setdefault(t, []).append((o, c0, c1))
                first, last = first + (c0 != o), last + (c0 == o)
                if c0 == o:
                    assert counters.setdefault(o, t) == t
                mine.add(t)
        assert first <= 1 and last <= 1  # an owner has two places for parts: of the tile that it begins, and of another
        joins.append(mine)
    tiles = sum(-(-(b - a) // f8_walk.TOKENS[f]) * tb for a, b in zip(begin, begin[1:]))
    assert sorted(seen) == list(range(tiles)) == sorted(t for t, *_ in places)
    for t, g in seen.items():
        g.sort()
        assert g[0][0] == 0 and g[-1][1] == groups and all(a[1] == b[0] for a, b in zip(g, g[1:]))
    for t, p in parts.items():
        assert len({(c0, c1) for _, c0, c1 in p}) == 1 and sorted(o for o, *_ in p) == list(range(p[0][1], p[0][2] + 1))
    # every output of every expert belongs to one tile
    area = {}
    for t, e, w, m0, rows in places:
        area.setdefault((e, w), []).append((m0, rows))
    for e, (a, b) in enumerate(zip(begin, begin[1:])):
        for w in range(tb if b > a else 0):
            at = a
            for m0, rows in sorted(area[(e, w)]):
                assert m0 == at
                at += rows
            assert at == b
    return {t: len(p) for t, p in parts.items()}, joins


def log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


@pytest.mark.parametrize("name", f8_walk.FORMS)
def test_one_matrix(name):
    rng = random.Random(1)
    f = f8_walk.FORMS.index(name)
    for _ in range(60):
        m, n, k = log_int(rng, 1, 12 * f8_walk.TOKENS[f]), log_int(rng, 1, 9000), 16 * log_int(rng, 1, 700)
        check(name, [0, m], n, k, rng.choice([2, 7, 100, 132, 148]), rng.choice([1 << 30, 1, 3 * f8_walk.TOKENS[f]]))


@pytest.mark.parametrize("name", f8_walk.FORMS)
def test_by_expert(name):
    rng = random.Random(2)
    f = f8_walk.FORMS.index(name)
    for _ in range(40):
        begin = [rng.choice([0, 5])]
        for _ in range(rng.choice([1, 3, 8, 40])):
            begin.append(begin[-1] + rng.choice([0, 0, 1, log_int(rng, 1, 5 * f8_walk.TOKENS[f])]))
        check(name, begin, log_int(rng, 1, 3000), 16 * log_int(rng, 1, 500), rng.choice([2, 37, 148]), rng.choice([1 << 30, 1, 300]))


@pytest.mark.parametrize("n,k", [(6144, 8192), (6144, 7168), (8192, 7680), (9216, 4608), (4736, 7168), (8192, 8192), (6144, 6144), (9088, 3584), (4736, 8192)])
def test_owners_of_one_number_of_them_a_tile_join_one_tile(n, k):
    """Where the last round's tiles are shared by fewer owners than there are, so that each tile has as many, none has parts of two tiles."""
    tiles, joins = check("narrow", [0, 1], n, k, 148)
    with_parts = [j for j in joins if j]
    if len(with_parts) < 148:
        assert len(set(tiles.values())) == 1 and all(len(j) == 1 for j in with_parts)
    assert tiles


def test_the_owners_of_64_tiles_of_16_groups_are_128():
    tiles, joins = check("narrow", [0, 1], 8192, 8192, 148)
    assert set(tiles.values()) == {2} and sum(1 for j in joins if j) == 128


def test_the_choice_of_a_form_is_one_of_them_for_every_size():
    rng = random.Random(3)
    seen = set()
    for _ in range(3000):
        seen.add(f8_walk.form(log_int(rng, 1, 1 << 20), log_int(rng, 1, 30000), 16 * log_int(rng, 1, 2000), rng.choice([1, 1, 8, 128, 1024]),
                              rng.choice([1, 2, 132, 148])))
    assert seen == set(f8_walk.FORMS)


def test_the_smoke_test_runs_every_form():
    import __graft_entry__ as entry

    assert [f8_walk.form(*shape) for shape in entry.F8_PRODUCTS] == ["narrow", "wide 128", "wide 256", "pair 256"]
