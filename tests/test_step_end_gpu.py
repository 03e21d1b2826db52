"""The end of a training step from the package's kernels alone - a head's cross entropy, its backward pass, the gated block's behind it, the norm of all
gradients and the AdamW step that clips by it - against the same steps differentiated in 64 bits; eager over several steps, and replayed from a captured
graph while an eager graph of the same leaves lives."""

import math

import pytest
import torch

from lumen_b200.runtime import (
    adamw_state,
    adamw_step,
    device_status,
    gated_mlp_backward,
    gated_mlp_forward,
    grad_norm,
    linear_cross_entropy,
    linear_cross_entropy_backward,
)

pytestmark = pytest.mark.gpu

LR, DECAY, BETAS, EPS = 0.01, 0.05, (0.9, 0.99), 1e-8


def problem(cuda, tokens, width, hidden, vocab, dtype):
    g = torch.Generator(device=cuda).manual_seed(0)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=cuda) * scale).to(dtype)

    weights = [normal(2 * hidden, width, scale=width**-0.5), normal(width, hidden, scale=hidden**-0.5), normal(vocab, width, scale=width**-0.5)]
    targets = torch.randint(0, vocab, (tokens,), generator=g, device=cuda)
    targets[::5] = -100
    return normal(tokens, width), targets, weights


def step(x, targets, weights, state, count, max_norm, scale=None, lr=LR):
    wgu, wd, head = weights
    y, gate_up, h = gated_mlp_forward(x, wgu, wd)
    loss, lse = linear_cross_entropy(y, head, targets)
    d_y, d_head = linear_cross_entropy_backward(scale, y, head, targets, lse)
    d_x, d_wgu, d_wd = gated_mlp_backward(d_y, x, wgu, wd, gate_up, h)
    grads = [d_wgu, d_wd, d_head]
    norm = grad_norm(grads)
    adamw_step(weights, grads, state[0], state[1], count, lr=lr, betas=BETAS, eps=EPS, weight_decay=DECAY, exp_avg_scale=state[2], exp_avg_sq_scale=state[3], norm=norm,
               max_norm=max_norm)  # fmt: skip
    return loss, norm, d_x


def reference(x, targets, weights):
    x, (wgu, wd, head) = x.double().requires_grad_(), [w.double().requires_grad_() for w in weights]
    gate, up = (x @ wgu.t()).chunk(2, -1)
    z = ((torch.nn.functional.silu(gate) * up) @ wd.t()) @ head.t()
    counts = targets >= 0
    loss = (torch.logsumexp(z, -1) - z.gather(-1, targets.clamp(min=0)[:, None])[:, 0])[counts].mean()
    grads = torch.autograd.grad(loss, (x, wgu, wd, head))
    return float(loss.detach()), grads


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("shape, dtype", [((7, 64, 96, 300), torch.bfloat16), ((300, 136, 264, 1001), torch.bfloat16), ((90, 72, 104, 257), torch.float32)])
def test_steps(cuda, shape, dtype, bits):
    x, targets, weights = problem(cuda, *shape, dtype)
    state = adamw_state(weights, bits)
    m, v = [torch.zeros(w.shape, dtype=torch.float64, device=cuda) for w in weights], [torch.zeros(w.shape, dtype=torch.float64, device=cuda) for w in weights]
    # some eight roundings lie between inputs and gradients, each at most half a step of its value, and are passed on at most four times as large; in
    # float32 sums of up to a thousand products take a rounding's place
    allowed = 8 * 4 * torch.finfo(dtype).eps / 2 * (1 if dtype == torch.bfloat16 else 64)
    for k in (1, 2, 3):
        want_loss, want = reference(x, targets, weights)
        total = math.sqrt(sum(float(t.square().sum()) for t in want[1:]))
        before = [w.clone() for w in weights]
        loss, norm, d_x = step(x, targets, weights, state, k, 0.5 * total)
        device_status()
        assert abs(float(loss) - want_loss) <= allowed * want_loss and abs(float(norm) - total) <= allowed * total
        assert float((d_x.double() - want[0]).norm()) <= 2 * allowed * float(want[0].norm())
        for i, (w, start) in enumerate(zip(weights, before)):
            g = 0.5 * want[1 + i]
            m[i], v[i] = BETAS[0] * m[i] + (1 - BETAS[0]) * g, BETAS[1] * v[i] + (1 - BETAS[1]) * g * g
            up = LR * (m[i] / (1 - BETAS[0] ** k)) / (torch.sqrt(v[i] / (1 - BETAS[1] ** k)) + EPS)
            moved = w.double() - start.double() * (1 - LR * DECAY)
            # A step is lr times a quotient that moves with the gradient's relative error where both moments have the same; an element whose gradient is small beside
            # its tensor's errors may have any quotient of up to about one, so that the whole is compared: its share of the squares is that of elements below `allowed`
            # of the tensor's size, about `allowed` of them for a normal distribution. Weights add half a step of theirs, moments in 8 bits a sixteenth each.
            off = 4 * math.sqrt(allowed) + (0.0 if bits == 32 or k == 1 else 0.125)
            rounding = float((w.double() * torch.finfo(dtype).eps / 2).norm())
            assert float((moved + up).norm()) <= off * float(up.norm()) + rounding, (k, i)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_beside_eager_ones(cuda, bits):
    shape = (130, 64, 96, 700)
    x, targets, weights = problem(cuda, *shape, torch.bfloat16)
    weights = [w.requires_grad_() for w in weights]
    alive = sum((w.float() ** 2).sum() for w in (w.clone() for w in weights))  # an eager graph of the same leaves
    other = [w.detach().clone() for w in weights]
    state, other_state = adamw_state(weights, bits), adamw_state(other, bits)
    count, scale = torch.ones((), dtype=torch.int64, device=cuda), torch.full((), 3.0, device=cuda)
    with torch.no_grad():
        warm = [w.detach().clone() for w in weights]
        step(x, targets, warm, adamw_state(warm, bits), 1, 1.0, scale)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(x, targets, weights, state, count, 1.0, scale)
        for k in (1, 2, 3):
            count.fill_(k)
            graph.replay()
            want = step(x, targets, other, other_state, k, 1.0, scale)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), k
            assert all(torch.equal(a, b) for a, b in zip(weights, other)), k
            assert all(torch.equal(a, b) for s, t in zip(state, other_state) if s for a, b in zip(s, t)), k
    alive.backward()
    torch.cuda.synchronize()
    assert all(bool(torch.isfinite(w.grad).all()) for w in weights)
