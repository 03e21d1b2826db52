"""The first calls of a process, from several threads at once, each on its own stream: kernels that are set up on first use are set up by then."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import threading
import torch
from lumen_b200.runtime import device_status, gated_mlp_backward, gated_mlp_forward, gemm, qk_norm_rope, qk_norm_rope_backward

g = torch.Generator(device="cuda").manual_seed(0)
def normal(*shape, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(torch.bfloat16)
x, wgu, wd = normal(2600, 840), normal(4112, 840, scale=0.03), normal(840, 2056, scale=0.02)
few, packed = x[:200], normal(2, 1500, 12, 128)
cos, sin = torch.ones(1500, 64, device="cuda"), torch.zeros(1500, 64, device="cuda")
weight = torch.ones(128, device="cuda", dtype=torch.bfloat16)

def calls():
    out = []
    for t in (x, few):
        y, gate_up, h = gated_mlp_forward(t, wgu, wd)
        out += [y, gate_up, h, *gated_mlp_backward(y, t, wgu, wd, gate_up, h)]
    q, k = packed[:, :, :8], packed[:, :, 8:]
    out += [*qk_norm_rope(q, k, cos, sin, q_weight=weight, k_weight=weight)]
    out += [*qk_norm_rope_backward(q, k, q, k, cos, sin, q_weight=weight, k_weight=weight)]
    out.append(gemm(x, wgu.t(), torch.empty(2600, 4112, device="cuda", dtype=torch.bfloat16)))
    return out

torch.cuda.synchronize()
results, errors, start = [None] * 8, [], threading.Barrier(8)
def work(k):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait(30)
            results[k] = calls()
            torch.cuda.current_stream().synchronize()
    except Exception as e:
        errors.append(e)
threads = [threading.Thread(target=work, args=(k,)) for k in range(8)]
for t in threads: t.start()
for t in threads: t.join()
assert not errors, errors
device_status()
want = calls()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for r in results for a, b in zip(r, want))
print("the same")
"""


def test_eight_threads(cuda):
    done = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "the same" in done.stdout, done.stdout + done.stderr
