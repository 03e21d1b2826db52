"""How the tensors of a clipping call are shared out over launches, and which chunks are left in the L2: as many as one call may keep, at its end."""

import ctypes
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "lumen_b200", "csrc")

SOURCE = """
#include "grad_norm.h"
extern "C" int passes(const long long* chunks, int n, int most, int keep, long long* out) {
    const auto all = lb::norm_passes(std::vector<long long>(chunks, chunks + n), most, keep);
    for (size_t k = 0; k < all.size(); k++) out[4 * k] = all[k].from, out[4 * k + 1] = all[k].to, out[4 * k + 2] = all[k].chunks, out[4 * k + 3] = all[k].keep;
    return (int)all.size();
}
"""


@pytest.fixture(scope="module")
def passes(tmp_path_factory):
    at = tmp_path_factory.mktemp("passes")
    (at / "main.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-w", "-fPIC", "-shared", "-I", CSRC, "-o", str(at / "p.so"), str(at / "main.cpp")], check=True)
    lib = ctypes.CDLL(str(at / "p.so"))

    def call(chunks, most, keep):
        out = (ctypes.c_longlong * (4 * len(chunks) + 4))()
        n = lib.passes((ctypes.c_longlong * max(len(chunks), 1))(*chunks), len(chunks), most, keep, out)
        return [tuple(out[4 * k : 4 * k + 4]) for k in range(n)]

    return call


def test_known(passes):
    assert passes([], 240, 2048) == []
    assert passes([5], 240, 2048) == [(0, 1, 5, 5)]
    assert passes([1000] * 300, 240, 2048) == [(0, 240, 240000, 0), (240, 300, 60000, 2048)]  # a model of many layers
    assert passes([10] * 300, 240, 2048) == [(0, 240, 2400, 1448), (240, 300, 600, 600)]
    assert passes([0, 3, 0, 0, 4, 5, 0], 2, 6) == [(0, 5, 7, 1), (5, 7, 5, 5)]
    assert passes([7, 7], 1, 0) == [(0, 1, 7, 0), (1, 2, 7, 0)]


def test_random(passes):
    r = random.Random(3)
    for _ in range(500):
        chunks = [r.choice([0, 1, r.randint(1, 40)]) for _ in range(r.randint(0, 60))]
        most, keep = r.randint(1, 12), r.randint(0, 200)
        all_ = passes(chunks, most, keep)
        assert [p[0] for p in all_] == [0, *(p[1] for p in all_)][: len(all_)] and (not chunks or all_[-1][1] == len(chunks))
        assert all(p[2] == sum(chunks[p[0] : p[1]]) and sum(c > 0 for c in chunks[p[0] : p[1]]) <= most for p in all_)
        assert sum(p[3] for p in all_) == min(keep, sum(chunks))
        left = keep
        for p in reversed(all_):
            assert p[3] == min(left, p[2])
            left -= p[3]
