"""The AdamW step of gradients so small that their squares are subnormal: the weights' step and what the moments hold are those of any other size."""

import pytest
import torch

from lumen_b200.runtime import adamw_state, adamw_step, device_status
from tests.test_adamw_gpu import rounds_to

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [1e-17, 1e-18, 1e-19, 4e-20])
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("n, offset", [(8 * 256, 0), (256 * 5 + 37, 0), (700, 3)])
def test_subnormal_second_moments(cuda, size, bits, n, offset):
    g = torch.Generator(device=cuda).manual_seed(1)

    def off(x):  # memory that vectors do not fit
        out = torch.empty(n + offset, dtype=x.dtype, device=cuda)[offset:]
        return out.copy_(x)

    w = off(torch.randn(n, generator=g, device=cuda))
    grad = off((1 + 3 * torch.rand(n, generator=g, device=cuda)) * (torch.randint(0, 2, (n,), generator=g, device=cuda) * 2 - 1) * size)
    m, v, ms, vs = adamw_state([w], bits)
    m, v = [off(m[0])], [off(v[0])]
    before = w.clone()
    b1, b2, lr = 0.9, 0.999, 1e-3
    adamw_step([w], [grad], m, v, 1, lr=lr, betas=(b1, b2), eps=0.0, weight_decay=0.0, exp_avg_scale=ms, exp_avg_sq_scale=vs)
    m32, v32 = grad * (1 - b1), grad * grad * (1 - b2)
    assert bool((v32 > 0).all())
    step = lr / (1 - b1) * m32.double() / (v32.double() / (1 - b2)).sqrt()
    # the root and the quotient are off by a few units in the last place, and the weight is rounded once
    assert bool(((w.double() - (before.double() - step)).abs() <= 2.0**-20 * step.abs() + 2.0**-24 * (1 + 2.0**-8) * w.double().abs()).all())
    if bits == 32:
        assert torch.equal(m[0], m32) and torch.equal(v[0], v32)
    else:
        for got, scale, want, lowest in ((m[0], ms[0], m32.double(), False), (v[0], vs[0], v32.double().sqrt(), True)):
            rounds_to(got, scale, want, 2.0**-21 * want.abs(), lowest, "moments")
    device_status()


@pytest.mark.parametrize("size", [1e-18, 1e-19])
def test_small_gradients_beside_others_and_zeros(cuda, size):
    """A block that holds zeros, small gradients and ones of a usual size; a small one with zeros alone."""
    g = torch.Generator(device=cuda).manual_seed(2)
    grad = torch.randn(512, generator=g, device=cuda)
    grad[::3] = size
    grad[1::3] = 0.0
    grad[256:] = torch.where(torch.arange(256, device=cuda) % 5 == 0, size, 0.0)
    w = torch.ones(512, device=cuda)
    m, v, ms, vs = adamw_state([w], 8)
    adamw_step([w], [grad], m, v, 1, eps=1e-30, weight_decay=0.0, exp_avg_scale=ms, exp_avg_sq_scale=vs)
    m32, v32 = grad * (1 - 0.9), grad * grad * (1 - 0.999)
    step = 1e-2 * m32.double() / ((v32.double() / (1 - 0.999)).sqrt() + 1e-30)
    assert bool(((w.double() - (1 - step)).abs() <= 2.0**-20 * step.abs() + 2.0**-24 * (1 + 2.0**-8) * w.double().abs()).all())
    for got, scale, want, lowest in ((m[0], ms[0], m32.double(), False), (v[0], vs[0], v32.double().sqrt(), True)):
        rounds_to(got, scale, want, 2.0**-21 * want.abs(), lowest, "moments")
