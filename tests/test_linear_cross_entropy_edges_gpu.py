"""Softmax cross entropy of a projection where its ways through the kernels end: pieces of the vocabulary with a single class."""

import pytest
import torch

from lumen_b200.runtime import device_status, linear_cross_entropy, linear_cross_entropy_backward
from tests.test_linear_cross_entropy_gpu import check_backward, check_forward, operands

pytestmark = pytest.mark.gpu


# 16 bits: a piece is 32768 classes of 4096 rows; float32 in parts: 10752 of them
@pytest.mark.parametrize("dtype, shape", [(torch.bfloat16, (4096, 64, 32769)), (torch.float16, (4096, 40, 65537)), (torch.float32, (4096, 64, 10753)), (torch.float32, (4096, 72, 21505)),
                                          (torch.float32, (40000, 800, 1)), (torch.float32, (40000, 801, 1))], ids=lambda s: "x".join(map(str, s)) if isinstance(s, tuple) else None)  # fmt: skip
def test_a_last_piece_of_one_class(cuda, dtype, shape):
    x, w, targets = operands(cuda, *shape, dtype, ignored=0.1)
    targets[0], targets[1], targets[2] = shape[2] - 1, 0, max(0, shape[2] - 2)
    loss, lse = linear_cross_entropy(x, w, targets)
    check_forward(x, w, targets, "mean", loss, lse)
    check_backward(x, w, targets, lse, "mean", None, *linear_cross_entropy_backward(None, x, w, targets, lse))
    device_status()


def test_a_last_piece_of_one_class_in_other_layouts(cuda):
    t, d, v = 4096, 44, 32769
    x, w, targets = operands(cuda, t, d, v, torch.bfloat16)
    targets[0] = v - 1
    padded = torch.zeros(v, 48, dtype=w.dtype, device=cuda)[:, :d]  # rows of whole 16 bytes, of which the width is none
    across = torch.zeros(d, 32776, dtype=w.dtype, device=cuda)[:, :v].t()  # classes one behind the other
    wide = torch.zeros(t, 48, dtype=x.dtype, device=cuda)[:, :d]
    wide.copy_(x)
    for layout in (padded, across):
        layout.copy_(w)
        loss, lse = linear_cross_entropy(wide, layout, targets)
        check_forward(x, w, targets, "mean", loss, lse)
        check_backward(x, w, targets, lse, "mean", None, *linear_cross_entropy_backward(None, wide, layout, targets, lse))
    device_status()
