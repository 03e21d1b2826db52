"""Set-up once per device and kernel, from several threads: who returns finds it done."""

import ctypes
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "lumen_b200", "csrc")

SOURCE = """
#include "first_use.h"
#include <atomic>
#include <chrono>
#include <stdexcept>
#include <thread>
#include <vector>

// How many of `threads` calls at once, half of them on another device, return before their device's set-up is done; *runs: set-ups.
extern "C" int early(int threads, int* runs) {
    lb::FirstUse uses;
    std::atomic<int> done[2] = {}, count{0}, bad{0}, at{0};
    static int key;
    std::vector<std::thread> all;
    for (int k = 0; k < threads; k++)
        all.emplace_back([&, k] {
            at++;
            while (at < threads) std::this_thread::yield();
            uses.run(k % 2, &key, [&] {
                count++;
                std::this_thread::sleep_for(std::chrono::milliseconds(20));
                done[k % 2] = 1;
            });
            bad += !done[k % 2];
        });
    for (auto& t : all) t.join();
    *runs = count;
    return bad;
}
// Set-ups that a key takes whose first one throws, and a second key's.
extern "C" int again() {
    lb::FirstUse uses;
    int runs = 0, keys[2];
    try {
        uses.run(0, keys, [&] { runs++; throw std::runtime_error("no"); });
        return -1;
    } catch (const std::runtime_error&) {
    }
    for (int k = 0; k < 3; k++) uses.run(0, keys, [&] { runs++; });
    for (int k = 0; k < 3; k++) uses.run(0, keys + 1, [&] { runs += 10; });
    return runs;
}
"""


def test_who_returns_finds_it_done(tmp_path):
    (tmp_path / "main.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O1", "-std=c++17", "-w", "-fPIC", "-shared", "-pthread", "-I", CSRC, "-o", str(tmp_path / "f.so"), str(tmp_path / "main.cpp")], check=True)
    lib, runs = ctypes.CDLL(str(tmp_path / "f.so")), ctypes.c_int()
    for _ in range(5):
        assert lib.early(8, ctypes.byref(runs)) == 0 and runs.value == 2
    assert lib.again() == 12


def test_every_set_up_runs_inside_it():
    """No kernel's attributes are set behind an answer that another thread may already have had."""
    for name in sorted(os.listdir(CSRC)):
        if name.endswith((".cu", ".cpp", ".cuh", ".h")):
            text = open(os.path.join(CSRC, name)).read()
            assert "if (first_use_on_device(" not in text and "&& first_use_on_device(" not in text, name


def test_pairs_are_counted_behind_their_kernels_set_up():
    """The first launch of CTA pairs may be another mode's: what the runtime is asked about has its limit of shared memory by then."""
    text = open(os.path.join(CSRC, "gemm.cu")).read()
    body = text[text.index("static int resident_pairs(") :]
    body = body[: body.index("\n}\n")]
    assert 0 < body.index("cudaFuncSetAttribute(gemm_tcgen05_pair<PlainArgs>") < body.index("cudaOccupancyMaxActiveClusters")
