"""Norms of queries and keys with the position rotation on more rows than a grid has threads, in every form that the kernel for many rows has: the whole
result of both passes against the formula in 64 bits."""

import pytest
import torch

from lumen_b200.runtime import device_status, qk_norm_rope, qk_norm_rope_backward
from tests.test_qk_norm_rope_gpu import backward64, case, close, forward64, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n, nk, h, pairs, interleaved, pad", [
    (7, 5, 72, 36, False, 0),  # pieces of four elements: a head dim that sixteen does not divide
    (6, 3, 72, 36, True, 0),
    (9, 2, 88, 12, False, 0),  # a rotated part that sixteen does not divide
    (5, 5, 128, 64, False, 4),  # rows that begin on 8 bytes and not on 16
    (5, 1, 128, 64, True, 4),
    (13, 3, 64, 32, True, 0),  # neighbours, pieces of eight
    (6, 2, 128, 64, True, 8),
    (5, 1, 256, 64, True, 0),
    (3, 2, 96, 48, False, 0),
    (1, 1, 16, 8, False, 0),
])  # fmt: skip
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_whole_results(cuda, n, nk, h, pairs, interleaved, pad, dtype):
    b, s = 3, 2501 if n > 1 else 20011
    q, k, dq, dk, g = case(cuda, b, s, n, nk, h, dtype, seed=h + pad, pad=pad)
    cos, sin = tables(s, pairs, cuda)
    rows = torch.randint(0, s, (b, s), generator=g, device=cuda)
    wq = (1 + 0.3 * torch.randn(h, generator=g, device=cuda)).to(dtype)
    wk = 1 + 0.3 * torch.randn(h, generator=g, device=cuda)
    out = qk_norm_rope(q, k, cos, sin, positions=rows, q_weight=wq, k_weight=wk, interleaved=interleaved)
    back = qk_norm_rope_backward(dq, dk, q, k, cos, sin, positions=rows, q_weight=wq, k_weight=wk, interleaved=interleaved)
    device_status()
    for x, w, y, dy, dx, dw in ((q, wq, out[0], dq, back[0], back[2]), (k, wk, out[1], dk, back[1], back[3])):
        close(y, *forward64(x, w, cos, sin, rows, interleaved))
        (want_dx, dx_size), (want_dw, dw_size) = backward64(dy, x, w, cos, sin, rows, interleaved)
        close(dx, want_dx, dx_size)
        close(dw, want_dw, dw_size, chain=5.0)  # chains of at most 16 rows, 256 groups of lanes and 14 + 32 sums of blocks
    # in the operands' place, and twice the same
    again = qk_norm_rope_backward(dq, dk, q, k, cos, sin, positions=rows, q_weight=wq, k_weight=wk, interleaved=interleaved, out=(dq, dk))
    assert all(torch.equal(a, c) for a, c in zip(again, back))
    again = qk_norm_rope(q, k, cos, sin, positions=rows, q_weight=wq, k_weight=wk, interleaved=interleaved, out=(q, k))
    assert all(torch.equal(a, c) for a, c in zip(again, out))
