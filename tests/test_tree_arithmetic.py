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
    lib.t_start.restype = ctypes.c_longlong
    lib.t_start.argtypes = [ctypes.c_longlong, ctypes.c_int, ctypes.c_int]
    lib.t_ranges.argtypes = [ctypes.c_longlong, ctypes.c_int, ctypes.c_int]
    lib.t_of.argtypes = [ctypes.c_longlong, ctypes.c_int, ctypes.c_longlong]
    return lib


def _seq(lib, *args):
    out = (ctypes.c_int * 9)()
    lib.t_seq(*args, out)
    return dict(zip(("len", "n", "ctx", "np", "s", "w0", "groups", "attended", "units"), out))


@pytest.mark.parametrize("seed", range(30))
def test_ranges_cover_every_unit_once(arith, seed):
    rng = np.random.default_rng(seed)
    items = [(int(g), int(u)) for g, u in zip(rng.integers(0, 5, 40), rng.integers(1, rng.choice([3, 40, 900]), 40))]
    units = sum(g * u for g, u in items)
    if units == 0:
        return
    most, least = int(rng.choice([1, 2, 7, 64, 500])), int(rng.choice([1, 4, 8]))
    R = arith.t_ranges(units, most, least)
    assert 1 <= R <= max(1, most) and (R == 1 or units >= R * least)
    starts = [arith.t_start(units, R, g) for g in range(R + 1)]
    assert starts[0] == 0 and starts[-1] == units and all(a < b for a, b in zip(starts, starts[1:]))
    for x in rng.integers(0, units, 50):
        g = arith.t_of(units, R, int(x))
        assert starts[g] <= x < starts[g + 1]
    # walk the ranges as the kernel does, and note who writes what of which item
    flat = [(i, j, u) for i, (g, u) in enumerate(items) for j in range(g)]
    firsts = np.concatenate([[0], np.cumsum([u for _, _, u in flat])])
    slots, cover, merges = {}, {k: [] for k in range(len(flat))}, {}
    for g in range(R):
        k = int(np.searchsorted(firsts, starts[g], side="right")) - 1
        skip, left = int(starts[g] - firsts[k]), starts[g + 1] - starts[g]
        g0, g1 = arith.t_of(units, R, int(firsts[k])), arith.t_of(units, R, int(firsts[k + 1]) - 1)
        if skip > 0 and g0 == g - 1:
            assert k not in merges
            merges[k] = [(g0 + i, 1 if i == 0 else 0) for i in range(g1 - g0 + 1)]
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
    units, R = 9_000_000_000, 512
    assert arith.t_start(units, R, 511) == units * 511 // 512 and arith.t_of(units, R, units - 1) == 511


@pytest.mark.parametrize("seed", range(40))
def test_attended_pages_hold_every_key_in_a_window(arith, seed):
    rng = np.random.default_rng(seed)
    length, n = int(rng.integers(1, 700)), int(rng.integers(1, 60))
    n = min(n, length)
    window, sink = int(rng.choice([0, 1, 5, 16, 40, 300])), int(rng.choice([0, 1, 16, 17, 64, 500]))
    np_, last = -(-length // 16), (length - 1) % 16 + 1
    args = (7, 7 + np_, last, 3, 3 + n, 100, int(rng.choice([2, 4, 16])), window, sink)
    t = _seq(arith, *args)
    assert (t["len"], t["n"], t["ctx"], t["np"]) == (length, n, length - n, np_)
    assert t["groups"] == -(-n // args[6])
    pages = [arith.t_page(*args, i) for i in range(t["attended"])]
    assert pages == sorted(set(pages)) and pages[-1] == np_ - 1
    for pos in range(n):   # any position a token may have: ctx + a depth of 0 or more
        seen = [k for k in range(length) if window == 0 or k >= t["ctx"] + pos - window + 1 or k < sink]
        assert {k // 16 for k in seen} <= set(pages)
    for page in range(np_ + 1):
        assert arith.t_below(*args, page) == sum(x < page for x in pages)
    if window and t["ctx"] > window + sink + 64:
        assert len(pages) < np_


@pytest.mark.parametrize("args,expect", [
    ((5, 5, 0, 0, 4, 10, 4, 0, 0), dict(len=0, n=4, ctx=-4, np=0, groups=1, attended=0, units=1)),
    ((5, 3, 9, 0, 4, 10, 4, 0, 0), dict(len=0, np=0)),                       # a page table that goes back
    ((0, 2, 99, 0, 4, 10, 4, 0, 0), dict(len=32)), ((0, 2, -3, 0, 4, 10, 4, 0, 0), dict(len=17)),
    ((0, 2, 5, 4, 2, 10, 4, 0, 0), dict(n=0, groups=0)),                     # and tokens that do
    ((0, 2, 5, -7, 3, 10, 4, 0, 0), dict(n=3)), ((0, 2, 5, 8, 99, 10, 4, 0, 0), dict(n=2)), ((0, 2, 5, 50, 99, 10, 4, 0, 0), dict(n=0)),
    ((0, 1, 3, 0, 9, 10, 4, 8, 2 ** 31 - 1), dict(len=3, n=9, ctx=-6, s=0, w0=0, attended=1)),
])
def test_tables_that_make_no_sense(arith, args, expect):
    t = _seq(arith, *args)
    assert {k: t[k] for k in expect} == expect


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
