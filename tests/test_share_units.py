"""How the units of two products of one launch are shared out to the CTA pairs: every unit once, no gaps in a pair's list, and no pair with more to do than it has to."""

import ctypes
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "lumen_b200", "csrc")

SOURCE = """
#include "share_units.h"
extern "C" int share(const long long* tiles, const long long* blocks, int pairs, uint16_t* table, int* slots, double* us) {
    return lb::share_units(tiles, blocks, pairs, table, *slots, *us);
}
"""
LISTED, NONE = 8192, 0xFFFF


@pytest.fixture(scope="module")
def share(tmp_path_factory):
    at = tmp_path_factory.mktemp("share")
    (at / "main.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-w", "-fPIC", "-shared", "-I", CSRC, "-o", str(at / "s.so"), str(at / "main.cpp")], check=True)
    lib = ctypes.CDLL(str(at / "s.so"))

    def call(tiles, blocks, pairs, lists=True):
        """The pairs' lists (None where the table does not hold them) and the time that the model gives."""
        table = (ctypes.c_uint16 * LISTED)(*([NONE] * LISTED)) if lists else None
        slots, us = ctypes.c_int(), ctypes.c_double()
        fits = lib.share((ctypes.c_longlong * 2)(*tiles), (ctypes.c_longlong * 2)(*blocks), pairs, table, ctypes.byref(slots), ctypes.byref(us))
        if not fits or not lists:
            return bool(fits), us.value
        return [[table[s * pairs + p] for s in range(slots.value)] for p in range(pairs)], us.value

    return call


def cost(unit, tiles, blocks):
    return 0.3 * blocks[unit >= tiles[0]] + 2.0


def test_known(share):
    lists, _ = share((3, 3), (20, 10), 2)
    assert lists == [[0, 2, 5], [1, 3, 4]]  # 8 + 8 + 5 and 8 + 5 + 5
    lists, _ = share((128, 256), (256, 128), 74)  # a piece of 16384 x 8192 x 1024
    assert max(sum(256 if u < 128 else 128 for u in pair if u != NONE) for pair in lists) == 896
    assert share((8000, 300), (4, 4), 74) == (False, share((8000, 300), (4, 4), 74)[1])


def test_random(share):
    r = random.Random(5)
    for _ in range(300):
        tiles, blocks, pairs = (r.randint(1, 400), r.randint(1, 400)), (r.randint(1, 300), r.randint(1, 300)), r.randint(1, 74)
        lists, us = share(tiles, blocks, pairs)
        assert (True, us) == share(tiles, blocks, pairs, lists=False)
        units = [u for pair in lists for u in pair if u != NONE]
        assert sorted(units) == list(range(sum(tiles)))
        loads = []
        for pair in lists:
            there = [u for u in pair if u != NONE]
            assert pair[: len(there)] == there
            loads.append(sum(cost(u, tiles, blocks) for u in there))
        total = sum(cost(u, tiles, blocks) for u in units)
        assert us == pytest.approx(max(loads) + 3.0 + 0.1 * sum(t * b for t, b in zip(tiles, blocks)) / pairs)
        # each to the pair with the least: the fullest has at most a unit more than the mean
        assert max(loads) <= total / pairs + max(cost(0, tiles, blocks), cost(tiles[0], tiles, blocks)) + 1e-9


def test_fewer_units_or_pairs_may_need_more_places(share):
    """Whether a table holds two products says nothing about fewer of their units, or about fewer pairs: a launch is asked about as it is."""
    assert share((1541, 5829), (347, 92), 74, lists=False)[0] and not share((67, 5829), (347, 1), 74, lists=False)[0]
    assert share((1572, 6420), (1756, 421), 74, lists=False)[0] and not share((1572, 6420), (1756, 421), 72, lists=False)[0]
