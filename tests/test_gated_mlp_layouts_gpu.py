"""The gated feed-forward block on batches and layouts that its kernels meet less often, against the formula in 64 bits."""

import pytest
import torch

from lumen_b200.runtime import device_status, gated_mlp_backward, gated_mlp_forward
from tests.test_gated_mlp_gpu import check_backward, check_forward, operands

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lead", [(3, 0), (0, 3), (5, 0, 2), (1, 0)])
def test_batches_without_tokens(cuda, lead):
    _, wgu, wd, _ = operands(cuda, 1, 64, 72, torch.bfloat16)
    x = torch.empty(*lead, 64, dtype=torch.bfloat16, device=cuda)
    y, gate_up, h = gated_mlp_forward(x, wgu, wd)
    assert y.shape == (*lead, 64) and gate_up.shape == (*lead, 144) and h.shape == (*lead, 72)
    dx, dwgu, dwd = gated_mlp_backward(torch.empty_like(y), x, wgu, wd, gate_up, h)
    device_status()
    assert dx.shape == x.shape and bool((dwgu == 0).all()) and bool((dwd == 0).all())  # empty sums


@pytest.mark.parametrize("m, d, f", [(1500, 840, 2056), (200, 512, 1024), (40, 256, 520)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weights_that_lie_the_other_way_round(cuda, m, d, f, dtype):
    """On tiles of CTA pairs and on narrow ones, with both projections' columns across and along the weights' rows."""
    x, wgu, wd, dy = operands(cuda, m, d, f, dtype)
    for a, b in ((wgu.t().contiguous().t(), wd.t().contiguous().t()), (wgu, wd.t().contiguous().t()), (wgu.t().contiguous().t(), wd)):
        y, gate_up, h = gated_mlp_forward(x, a, b, activation="gelu")
        check_forward(x, a, b, "gelu", y, gate_up, h)
        grads = gated_mlp_backward(dy, x, a, b, gate_up, h, activation="gelu")
        device_status()
        check_backward(dy, x, a, b, gate_up, h, "gelu", *grads)


@pytest.mark.parametrize("m", [40, 300, 1500])
def test_what_was_kept_in_rows_that_are_not_one_behind_the_other(cuda, m):
    """One token repeated: its projections and their gated product as rows that share memory."""
    x, wgu, wd, dy = operands(cuda, m, 840, 2056, torch.bfloat16)
    x = x[:1].expand(m, 840)
    y, gate_up, h = (t.expand(m, -1) for t in gated_mlp_forward(x[:1], wgu, wd))
    grads = gated_mlp_backward(dy, x, wgu, wd, gate_up, h)
    device_status()
    check_backward(dy, x, wgu, wd, gate_up, h, "silu", *grads)
