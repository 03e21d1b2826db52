"""Whether strided tensors share memory, as the entries that refuse such calls ask it: against all elements' bytes, one by one."""

import ctypes
import itertools
import os
import random
import subprocess

import pytest

from lumen_b200._lib import LbTensor

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "lumen_b200", "csrc")
SIZES = {5: 1, 9: 2, 11: 4, 4: 8}  # uint8, float16, float32, int64

SOURCE = """
#include "overlap.h"
extern "C" int shared(const lb_tensor* a, const lb_tensor* b) { return lb::share_memory(*a, *b); }
extern "C" int itself(const lb_tensor* a) { return lb::overlaps_itself(*a); }
extern "C" int same(const lb_tensor* a, const lb_tensor* b) { return lb::same_places(*a, *b); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    at = tmp_path_factory.mktemp("overlap")
    (at / "main.cpp").write_text(SOURCE)
    sources = [str(at / "main.cpp"), os.path.join(CSRC, "overlap.cpp"), os.path.join(CSRC, "common.cpp")]
    subprocess.run(["g++", "-O1", "-std=c++17", "-w", "-fPIC", "-shared", "-I", CSRC, "-o", str(at / "o.so"), *sources], check=True)
    return ctypes.CDLL(str(at / "o.so"))


def tensor(at, shape, strides, dtype):
    t = LbTensor()
    t.ptr, t.dtype, t.rank = at, dtype, len(shape)
    for d, (n, s) in enumerate(zip(shape, strides)):
        t.shape[d], t.stride[d] = n, s
    return t


def elements(at, shape, strides, dtype):
    size = SIZES[dtype]
    return [at + size * sum(i * s for i, s in zip(index, strides)) for index in itertools.product(*map(range, shape))]


def bytes_of(starts, dtype):
    return {a + p for a in starts for p in range(SIZES[dtype])}


def test_random_layouts(lib):
    r = random.Random(5)
    seen = [0, 0, 0, 0]
    for _ in range(6000):
        sides = []
        for _ in range(2):
            dtype = r.choice(list(SIZES))
            rank = r.randint(0, 4)
            shape = [r.choice([0, 1, 1, 2, 3, 4]) if r.random() < 0.3 else r.randint(1, 4) for _ in range(rank)]
            if r.random() < 0.5:  # views of a dense buffer
                room = [n + r.randint(0, 3) for n in shape]
                strides, step = [0] * rank, 1
                for d in r.sample(range(rank), rank):
                    strides[d], step = step, step * max(room[d], 1)
            else:
                strides = [r.randint(-12, 12) for _ in range(rank)]
            sides.append((4096 + SIZES[dtype] * r.randint(-30, 30), shape, strides, dtype))
        a, b = sides
        at_a, at_b = bytes_of(elements(*a), a[3]), bytes_of(elements(*b), b[3])
        shared = bool(at_a & at_b)
        assert bool(lib.shared(ctypes.byref(tensor(*a)), ctypes.byref(tensor(*b)))) == shared, (a, b)
        itself = len(at_a) < len(elements(*a)) * SIZES[a[3]]
        assert bool(lib.itself(ctypes.byref(tensor(*a)))) == itself, a
        seen[shared] += 1
        seen[2 + itself] += 1
    assert min(seen) > 500


def test_large_views(lib):
    """Sizes that nobody could walk: heads of a packed projection, halves of rows, sequences of a cache; a row apart and not quite."""

    def shared(*sides):
        return bool(lib.shared(*(ctypes.byref(tensor(*s)) for s in sides)))

    b, s, n, nk, h = 8, 32768, 32, 8, 128
    row = (n + 2 * nk) * h
    packed = [s * row, row, h, 1]
    q, k = (0, [b, s, n, h], packed, 9), (2 * n * h, [b, s, nk, h], packed, 9)
    assert not shared(q, k) and shared(q, (2 * n * h - 2, [b, s, nk, h], packed, 9)) and shared((0, [b, s, n + 1, h], packed, 9), k)
    left, right = (0, [b, s, n, 64], [s * n * 128, n * 128, 128, 1], 9), (128, [b, s, n, 64], [s * n * 128, n * 128, 128, 1], 9)
    assert not shared(left, right) and shared(left, (126, *right[1:]))
    outer = [n * s * h, h, s * h, 1]  # heads outermost
    assert not shared((0, [b, s, 3, h], outer, 9), (2 * 3 * s * h, [b, s, n - 3, h], outer, 9)) and shared((0, [b, s, 4, h], outer, 9), (2 * 3 * s * h, [b, s, n - 3, h], outer, 9))
    assert not shared((0, [b, s // 2, 1, h], [s * h, h, h, 1], 9), (s // 2 * h * 2, [b, s // 2, 1, h], [s * h, h, h, 1], 9))
    assert not shared((0, [1 << 40], [1 << 20], 9), (2, [1 << 40], [1 << 20], 9)) and shared((0, [1 << 40], [1 << 20], 9), (2 << 50, [5], [7], 9))
    assert not lib.itself(ctypes.byref(tensor(*q))) and lib.itself(ctypes.byref(tensor(0, [b, s, n, h], [s * row, row, h - 1, 1], 9)))
    assert lib.itself(ctypes.byref(tensor(0, [3, 2], [0, 1], 9))) and not lib.itself(ctypes.byref(tensor(0, [3, 2], [2, 3], 9)))


def test_the_same_places(lib):
    a = tensor(4096, [2, 1, 4], [8, 99, 1], 9)
    assert lib.same(ctypes.byref(a), ctypes.byref(tensor(4096, [2, 1, 4], [8, 5, 1], 9)))
    for other in ((4098, [2, 1, 4], [8, 5, 1], 9), (4096, [2, 1, 4], [4, 5, 1], 9), (4096, [2, 1, 4], [8, 5, 1], 10), (4096, [2, 4], [8, 1], 9), (4096, [1, 1, 4], [8, 5, 1], 9)):
        assert not lib.same(ctypes.byref(a), ctypes.byref(tensor(*other)))
