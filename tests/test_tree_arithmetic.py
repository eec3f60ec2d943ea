"""How the attention of drafted tokens is cut over the workgroups (csrc/tree_arith.h, compiled by the host compiler):
every unit in exactly one range, the pieces of a cut item found by the boundary that cuts it first, in slots of their
own, and every key that a token may see on an attended page."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def arith(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("arith") / "tree_arith.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC",
                    os.path.join(ROOT, "tests", "cpp", "tree_arith.cpp"), "-o", so], check=True)
    lib = ctypes.CDLL(so)
    L, I = ctypes.c_longlong, ctypes.c_int
    lib.t_ranges.argtypes, lib.t_start.argtypes, lib.t_of.argtypes = [L, I, I, I, I], [L, I, I, I, I, I], [L, I, I, I, I, L]
    lib.t_start.restype = lib.t_before.restype = L
    lib.t_group.argtypes = [ctypes.c_void_p, L]
    return lib


def _args(*args):
    return (ctypes.c_int * 10)(*args)


def _seq(lib, *args):
    out = (ctypes.c_int * 8)()
    lib.t_seq(_args(*args), out)
    return dict(zip(("len", "n", "ctx", "np", "s", "w0", "groups", "attended"), out))


@pytest.mark.parametrize("seed", range(30))
def test_ranges_cover_every_unit_once(arith, seed):
    rng = np.random.default_rng(seed)
    items = [(int(g), int(u)) for g, u in zip(rng.integers(0, 5, 40), rng.integers(1, rng.choice([3, 40, 900]), 40))]
    units = sum(g * u for g, u in items)
    if units == 0:
        return
    most, least = int(rng.choice([1, 2, 7, 64, 500])), int(rng.choice([4, 8]))
    early, late = [(1, 1), (9, 7), (5, 3), (8, 7)][int(rng.integers(0, 4))]
    cut = (units, most, least, early, late)
    R = arith.t_ranges(*cut)
    assert 1 <= R <= max(1, most) and (R == 1 or units >= R * least)
    starts = [arith.t_start(*cut, g) for g in range(R + 1)]
    assert starts[0] == 0 and starts[-1] == units and all(a < b for a, b in zip(starts, starts[1:]))
    if R == most and R > 1 and R % 2 == 0:
        assert abs(starts[R // 2] * late - (units - starts[R // 2]) * early) <= early + late
    for x in rng.integers(0, units, 50):
        g = arith.t_of(*cut, int(x))
        assert starts[g] <= x < starts[g + 1]
    # walk the ranges as the kernel does, and note who writes what of which item
    flat = [(i, j, u) for i, (g, u) in enumerate(items) for j in range(g)]
    firsts = np.concatenate([[0], np.cumsum([u for _, _, u in flat])])
    slots, cover, merges = {}, {k: [] for k in range(len(flat))}, {}
    for g in range(R):
        k = int(np.searchsorted(firsts, starts[g], side="right")) - 1
        skip, left = int(starts[g] - firsts[k]), starts[g + 1] - starts[g]
        g0, g1 = arith.t_of(*cut, int(firsts[k])), arith.t_of(*cut, int(firsts[k + 1]) - 1)
        if skip > 0:   # every cut of an item knows them all
            mine = [(g0 + i, 1 if i == 0 else 0) for i in range(g1 - g0 + 1)]
            assert g0 < g <= g1 and merges.setdefault(k, mine) == mine
        while left > 0:
            u = flat[k][2]
            take = min(left, u - skip)
            s = arith.t_slot(skip, take, u)
            cover[k].append((skip, skip + take))
            if s >= 0:
                assert (g, s) not in slots, "two pieces in one slot"
                slots[g, s] = k
            else:
                assert (skip, take) == (0, u)
            left, skip, k = left - take, 0, k + 1
    for k, (_, _, u) in enumerate(flat):
        c = cover[k]
        assert c[0][0] == 0 and c[-1][1] == u and all(a[1] == b[0] for a, b in zip(c, c[1:]))
        if len(c) > 1:   # merged from exactly its slots, in the order of its pieces
            assert [slots[x] for x in merges[k]] == [k] * len(c)
        else:
            assert k not in merges


def test_large_batches_stay_in_range(arith):
    cut = (9_000_000_000, 512, 8, 9, 7)
    starts = [arith.t_start(*cut, g) for g in range(513)]
    assert starts == [cut[0] * (9 * min(g, 256) + 7 * max(g - 256, 0)) // 4096 for g in range(513)]
    for g in range(512):
        assert arith.t_of(*cut, starts[g]) == g and arith.t_of(*cut, starts[g + 1] - 1) == g


@pytest.mark.parametrize("seed", range(40))
def test_attended_pages_hold_every_key_in_a_window(arith, seed):
    rng = np.random.default_rng(seed)
    length, n = int(rng.integers(1, 700)), int(rng.integers(1, 60))
    n = min(n, length)
    window, sink = int(rng.choice([0, 1, 5, 16, 40, 300])), int(rng.choice([0, 1, 16, 17, 64, 500]))
    np_, last = -(-length // 16), (length - 1) % 16 + 1
    args = (7, 7 + np_, last, 3, 3 + n, 100, int(rng.choice([2, 4, 16, 64])), window, sink, int(rng.integers(0, 2)))
    t = _seq(arith, *args)
    tpg, args = args[6], _args(*args)
    assert (t["len"], t["n"], t["ctx"], t["np"]) == (length, n, length - n, np_)
    assert t["groups"] == -(-n // tpg)
    pages = [arith.t_page(args, i) for i in range(t["attended"])]
    assert pages == sorted(set(pages)) and pages[-1] == np_ - 1
    for pos in range(n):   # any position a token may have: ctx + a depth of 0 or more
        seen = [k for k in range(length) if window == 0 or k >= t["ctx"] + pos - window + 1 or k < sink]
        assert {k // 16 for k in seen} <= set(pages)
    for page in range(np_ + 1):
        assert arith.t_below(args, page) == sum(x < page for x in pages)
    # the units of every group: enough for all the pages that its tokens may see, and found again from the sum
    start = 0
    for j in range(t["groups"]):
        u = arith.t_units(args, j)
        assert u >= 1 and arith.t_before(args, j) == start
        last_key = t["ctx"] + min(n, (j + 1) * tpg) - 1 if args[9] and 2 * n > t["ctx"] else length - 1
        assert u >= sum(p <= last_key // 16 for p in pages)
        for x in (start, start + u // 2, start + u - 1):
            assert arith.t_group(args, x) == j
        start += u
    assert arith.t_before(args, t["groups"]) == start
    if window and t["ctx"] > window + sink + 64:
        assert len(pages) < np_


@pytest.mark.parametrize("args,expect", [
    ((5, 5, 0, 0, 4, 10, 4, 0, 0), dict(len=0, n=4, ctx=-4, np=0, groups=1, attended=0)),
    ((5, 3, 9, 0, 4, 10, 4, 0, 0), dict(len=0, np=0)),                       # a page table that goes back
    ((0, 2, 99, 0, 4, 10, 4, 0, 0), dict(len=32)), ((0, 2, -3, 0, 4, 10, 4, 0, 0), dict(len=17)),
    ((0, 2, 5, 4, 2, 10, 4, 0, 0), dict(n=0, groups=0)),                     # and tokens that do
    ((0, 2, 5, -7, 3, 10, 4, 0, 0), dict(n=3)), ((0, 2, 5, 8, 99, 10, 4, 0, 0), dict(n=2)), ((0, 2, 5, 50, 99, 10, 4, 0, 0), dict(n=0)),
    ((0, 1, 3, 0, 9, 10, 4, 8, 2 ** 31 - 1), dict(len=3, n=9, ctx=-6, s=0, w0=0, attended=1)),
])
def test_tables_that_make_no_sense(arith, args, expect):
    for causal in (0, 1):
        t = _seq(arith, *args, causal)
        assert {k: t[k] for k in expect} == expect
        assert all(arith.t_units(_args(*args, causal), j) >= 1 for j in range(t["groups"]))


@pytest.mark.parametrize("step,width", [(8, 2), (4, 4)])
def test_order_of_blocks(arith, step, width):
    """Every block once, the plain ones first and all of them, whatever the pages that every row sees."""
    rng = np.random.default_rng(step)
    out, order = (ctypes.c_int * 2)(), (ctypes.c_int * 200)()
    plain_seen = 0
    for _ in range(4000):
        first, p1 = int(rng.integers(0, 40)), int(rng.integers(0, 120))
        a0, a1 = sorted(rng.integers(-5, 140, 2).tolist()) if rng.random() < 0.8 else rng.integers(-5, 140, 2).tolist()
        arith.t_order(first, step, width, p1, a0, a1, out, order)
        n, plain = out
        assert n == len(range(first, p1, step)) and sorted(order[:n]) == list(range(n)) and 0 <= plain <= n
        want = [i for i in range(n) if a0 <= first + step * i and first + step * i + width <= min(a1, p1)]
        assert sorted(order[:plain]) == want
        plain_seen += plain
    assert plain_seen > 1000


@pytest.mark.parametrize("tpg", [2, 4, 8, 16, 32, 128])
def test_units_of_a_long_chain(arith, tpg):
    """A chunk of a prefill: later groups see more pages, and the sum says so."""
    args = _args(0, 100, 16, 0, 1500, 1500, tpg, 0, 0, 1)   # 1600 cached, 100 of them before the chunk
    groups = -(-1500 // tpg)
    units = [arith.t_units(args, j) for j in range(groups)]
    need = [-(-(100 + min(1500, (j + 1) * tpg)) // 16) for j in range(groups)]
    assert all(n <= u <= n + max(1, tpg // 16) for n, u in zip(need, units))
    assert [arith.t_before(args, j) for j in range(groups + 1)] == np.concatenate([[0], np.cumsum(units)]).tolist()
    for x in range(0, sum(units), 7):
        assert arith.t_group(args, x) == int(np.searchsorted(np.cumsum(units), x, side="right"))


@pytest.mark.parametrize("seed", range(30))
@pytest.mark.parametrize("weight,extra", [(4, 0), (4, 32), (4, 3), (1, 8)])
def test_weighted_units(arith, seed, weight, extra):
    """A last group of at most half its rows counts three quarters, an item's start `extra`; cuts at any unit leave every page
    in exactly one piece, that of its first unit."""
    rng = np.random.default_rng(seed)
    n, tpg, causal = int(rng.integers(1, 300)), int(rng.choice([1, 2, 16, 32, 128])), int(rng.integers(0, 2))
    length = n + int(rng.choice([0, 3, 100, 4000]))
    np_ = -(-length // 16)
    args, out = _args(2, 2 + np_, (length - 1) % 16 + 1, 0, n, n, tpg, 0, 0, causal), (ctypes.c_int * 7)()

    def at(j, x=0):
        arith.t_weighted(args, weight, extra, j, x, out)
        return list(out)

    groups, start = -(-n // tpg), 0
    for j in range(groups):
        u, before, total, _, _, g, last = at(j)
        short = 2 * min(tpg, n - j * tpg) <= tpg
        pages, w = arith.t_units(args, j), weight - weight // 4 if short else weight
        assert g == groups and before == start and u == pages * w + extra and last == extra + (pages - 1) * w
        for x in (0, u // 2, u - 1):
            assert at(j, x)[3] == j
        cuts = sorted({0, u, *rng.integers(0, u + 1, 5).tolist()})
        edges = [at(j, c)[4] for c in cuts]
        assert edges[0] == 0 and edges[-1] == pages and edges == sorted(edges)
        for c, e in zip(cuts, edges):   # page e is the first whose first unit is c or later
            assert e == sum(extra + w * k < c for k in range(pages))
        start += u
    assert at(0)[2] == start


@pytest.mark.parametrize("seed", range(40))
def test_weighted_pieces_and_their_merges(arith, seed):
    """The walk of the ranges with starts that count: an item's pieces are whole, in slots of their own, and the merge's
    arithmetic finds exactly them."""
    rng = np.random.default_rng(seed)
    items = [(int(w), int(p)) for w, p in zip(rng.choice([3, 4], 40), rng.integers(1, rng.choice([3, 40, 900]), 40))]
    extra = int(rng.choice([0, 3, 32, 64]))
    size = [extra + w * p for w, p in items]
    firsts = np.concatenate([[0], np.cumsum(size)])
    cut = (int(firsts[-1]), int(rng.choice([1, 2, 7, 64, 500])), 32, *[(1, 1), (9, 8)][int(rng.integers(0, 2))])
    R = arith.t_ranges(*cut)
    starts = [arith.t_start(*cut, g) for g in range(R + 1)]
    page = lambda k, x: min(max(0, -(-(x - extra) // items[k][0])), items[k][1])  # noqa: E731
    slots, cover, merges = {}, {k: [] for k in range(len(items))}, {}
    for g in range(R):
        k = int(np.searchsorted(firsts, starts[g], side="right")) - 1
        skip, left = int(starts[g] - firsts[k]), starts[g + 1] - starts[g]
        w, p = items[k]
        g0, g1 = arith.t_of(*cut, int(firsts[k]) + extra), arith.t_of(*cut, int(firsts[k]) + extra + w * (p - 1))
        if g0 < g <= g1:
            mine = [(g0 + i, 1 if i == 0 else 0) for i in range(g1 - g0 + 1)]
            assert merges.setdefault(k, mine) == mine
        while left > 0:
            take = min(left, size[k] - skip)
            f0, f1 = page(k, skip), page(k, skip + take)
            if f0 < f1:
                s = arith.t_slot(f0, f1, items[k][1])
                cover[k].append((f0, f1))
                if s >= 0:
                    assert (g, s) not in slots, "two pieces in one slot"
                    slots[g, s] = k
            left, skip, k = left - take, 0, k + 1
    for k, (_, p) in enumerate(items):
        c = cover[k]
        assert c[0][0] == 0 and c[-1][1] == p and all(a[1] == b[0] for a, b in zip(c, c[1:]))
        if len(c) > 1:
            assert [slots[x] for x in merges[k]] == [k] * len(c)
        else:
            assert k not in merges
