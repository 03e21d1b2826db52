"""The gated feed-forward block and its backward pass against the formula in 64 bits: one token to many, sizes around the tiles, every activation
and type, layouts that the tensor cores take and others, and the gradients against differences."""

import math

import numpy as np
import pytest
import torch

from lumen_b200 import device as D
from lumen_b200.runtime import device_status, gated_mlp_backward, gated_mlp_forward, gemm

pytestmark = pytest.mark.gpu

# A float32 sum of K products on the tensor cores drops at most 2^-23 of the running sum's magnitude a step; the activation's exponential and
# reciprocal are within 2^-17 of its value for arguments up to 30 in 16-bit types, 2^-20 in float32.
STEP = 2.0**-23


def half(dtype):
    return torch.finfo(dtype).eps / 2 * (1 + 2.0**-8)


def tiny(dtype):
    # half a step of float16's subnormals; else where float32 ends: a sigmoid below 2^-126 may be 0, which a gate of 1000, its cube's slope and a sum of
    # a hundred such terms make 1e-38 x 1e3 x 1e6 x 1e2 at most
    return 2.0**-25 if dtype == torch.float16 else 1e-26


def unit(a, kind):
    if kind == "silu":
        return a * torch.sigmoid(a)
    if kind == "relu":
        return torch.where(a > 0, a, 0.0)
    # 0.5 a (1 + tanh(t)) is a sigmoid(2 t); far out 1 + tanh(t) itself has 2^-53 of error in 64 bits and nothing else
    return a * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (a + 0.044715 * a**3))


def slope(a, kind):
    a = a.clone().requires_grad_()
    return torch.autograd.grad(unit(a, kind).sum(), a)[0]


def within(got, want, tol, what):
    off = (got.double() - want).abs() - tol
    assert bool((off <= 0).all()), f"{what}: off by up to {off.max().item():.3g} more than allowed"


def operands(cuda, m, d, f, dtype, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=cuda) * scale).to(dtype)

    return normal(m, d), normal(2 * f, d, scale=1.5 * d**-0.5), normal(d, f, scale=f**-0.5), normal(m, d, scale=0.5)


def check_forward(x, wgu, wd, kind, y, gate_up, h, residual=None):
    dtype, d, f = x.dtype, x.shape[-1], wd.shape[1]
    fast = 2.0**-17 if dtype != torch.float32 else 2.0**-20
    x2, w2 = x.double().reshape(-1, d), wgu.double()
    pre, size = x2 @ w2.t(), x2.abs() @ w2.abs().t()
    sums = (d + 8) * STEP * size
    if gate_up is not None:
        within(gate_up.reshape(pre.shape), pre, half(dtype) * pre.abs() + sums + tiny(dtype), "gate_up")
    a, b = pre.split(f, -1)
    da, db = sums.split(f, -1)
    want = unit(a, kind) * b
    # |f'| is at most 1.13
    within(h.reshape(want.shape), want, half(dtype) * want.abs() + 1.13 * da * (b.abs() + db) + unit(a, kind).abs() * db + fast * want.abs() + tiny(dtype) + 1e-36, "h")
    h2, wd2 = h.double().reshape(-1, f), wd.double()
    want, size = h2 @ wd2.t(), h2.abs() @ wd2.abs().t()
    tol = half(dtype) * want.abs() + (f + 8) * STEP * size + tiny(dtype)
    if residual is not None:  # the product rounded, the sum rounded
        r = residual.double().reshape(want.shape)
        want, tol = want + r, tol * (1 + half(dtype)) + half(dtype) * (want + r).abs() + tiny(dtype)
    within(y.reshape(want.shape), want, tol, "y")


def check_backward(dy, x, wgu, wd, gate_up, h, kind, dx, dwgu, dwd):
    dtype, d, f = x.dtype, x.shape[-1], wd.shape[1]
    fast = 2.0**-16 if dtype != torch.float32 else 2.0**-19
    dy, x2, h2, pre = (t.double().reshape(-1, t.shape[-1]) for t in (dy, x, h, gate_up))
    m = x2.shape[0]
    a, b = pre.split(f, -1)
    dh, dh_off = dy @ wd.double(), (d + 8) * STEP * (dy.abs() @ wd.double().abs())
    value, s = unit(a, kind), slope(a, kind)
    dpre = torch.cat((dh * b * s, dh * value), -1)
    # s + a s (1 - s) t' adds up terms of at most 1 + |a| t' in magnitude, which may cancel
    grade = (1 + a.abs() * (1 if kind == "silu" else 1.6 * (1 + 0.14 * a * a))) * (kind != "relu") + (kind == "relu")
    off = half(dtype) * dpre.abs() + tiny(dtype) + torch.cat((dh_off * b.abs() * s.abs() + fast * dh.abs() * b.abs() * grade, dh_off * value.abs() + fast * dh.abs() * value.abs()), -1)
    w2 = wgu.double()
    want = dpre @ w2
    within(dx.reshape(want.shape), want, half(dtype) * want.abs() + off @ w2.abs() + (2 * f + 8) * STEP * ((dpre.abs() + off) @ w2.abs()) + tiny(dtype), "d_x")
    want = dpre.t() @ x2
    within(dwgu, want, half(dtype) * want.abs() + off.t() @ x2.abs() + (m + 8) * STEP * ((dpre.abs() + off).t() @ x2.abs()) + tiny(dtype), "d_w_gate_up")
    want = dy.t() @ h2
    within(dwd, want, half(dtype) * want.abs() + (m + 8) * STEP * (dy.abs().t() @ h2.abs()) + tiny(dtype), "d_w_down")


SHAPES = [
    # tokens, width, hidden
    (1, 64, 64), (1, 1024, 512), (2, 136, 264), (4, 1024, 1000), (7, 512, 128), (8, 96, 2048), (9, 256, 192), (16, 328, 520), (17, 128, 128),
    (32, 512, 256), (33, 256, 200), (100, 64, 72), (128, 256, 256), (129, 520, 136), (255, 128, 1032), (257, 264, 384), (300, 72, 128), (512, 256, 640),
    (700, 8, 8), (1000, 320, 1160), (1500, 840, 2056), (1921, 1000, 1504), (8300, 40, 8), (5, 2400, 64), (12, 2400, 72), (20, 2400, 64), (24, 512, 264), (64, 40, 6200), (40, 24, 16400), (3, 64, 4200), (30, 8, 5000), (5, 15, 9), (40, 33, 70), (130, 100, 61),
]  # fmt: skip


@pytest.mark.parametrize("kind", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_backward(cuda, shape, dtype, kind):
    m, d, f = shape
    x, wgu, wd, dy = operands(cuda, m, d, f, dtype, seed=m + d)
    y, gate_up, h = gated_mlp_forward(x, wgu, wd, activation=kind)
    assert y.shape == (m, d) and gate_up.shape == (m, 2 * f) and h.shape == (m, f) and y.dtype == gate_up.dtype == h.dtype == dtype
    check_forward(x, wgu, wd, kind, y, gate_up, h)
    grads = gated_mlp_backward(dy, x, wgu, wd, gate_up, h, activation=kind)
    device_status()
    check_backward(dy, x, wgu, wd, gate_up, h, kind, *grads)


@pytest.mark.parametrize("m", [1, 8, 24, 200, 1000])
def test_without_what_the_backward_pass_needs(cuda, m):
    x, wgu, wd, _ = operands(cuda, m, 256, 392, torch.bfloat16)
    kept = gated_mlp_forward(x, wgu, wd)
    y, gate_up, h = gated_mlp_forward(x, wgu, wd, save=False)
    assert gate_up is None and torch.equal(y, kept[0]) and torch.equal(h, kept[2])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(3, 64, 96), (300, 136, 264), (41, 30, 17)])
def test_residual(cuda, shape, dtype):
    m, d, f = shape
    x, wgu, wd, r = operands(cuda, m, d, f, dtype)
    y, gate_up, h = gated_mlp_forward(x, wgu, wd, residual=r)
    check_forward(x, wgu, wd, "silu", y, gate_up, h, residual=r)


@pytest.mark.parametrize("m", [5, 300])
def test_batches_views_and_transposed_weights(cuda, m):
    """Leading dimensions, rows wider than their matrix, weights that lie the other way round, operands that begin off a 16-byte line."""
    d, f, dtype = 128, 192, torch.bfloat16
    x, wgu, wd, dy = operands(cuda, 2 * m, d, f, dtype)
    x3 = torch.cat((x, x), 1)[:, :d].view(2, m, d)
    dy3 = torch.cat((dy, dy), 1)[:, d:].view(2, m, d)

    def off_line(t):
        room = torch.empty(t.numel() + 1, dtype=t.dtype, device=cuda)
        room[1:] = t.reshape(-1)
        return room[1:].view(t.shape)

    for a, b, c, e in ((x3, wgu, wd, dy3), (x3, wgu.t().contiguous().t(), wd.t().contiguous().t(), dy3), (off_line(x3), off_line(wgu), off_line(wd), off_line(dy3))):
        y, gate_up, h = gated_mlp_forward(a, b, c)
        assert y.shape == (2, m, d) and gate_up.shape == (2, m, 2 * f) and h.shape == (2, m, f)
        check_forward(a, b, c, "silu", y, gate_up, h)
        grads = gated_mlp_backward(e, a, b, c, gate_up, h)
        assert grads[0].shape == (2, m, d) and grads[1].shape == wgu.shape and grads[2].shape == wd.shape
        check_backward(e, a, b, c, gate_up, h, "silu", *grads)
    device_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("m", [3, 300])
def test_activations_far_out(cuda, m, kind, dtype):
    """Gates of up to +-1000, where exponentials over- and underflow: values and slopes are their limits, and nothing is NaN."""
    d = f = 64
    x = torch.zeros(m, d, device=cuda)
    x[:, 0] = torch.linspace(-1000.0, 1000.0, m, device=cuda)
    x[:, 1] = 1.0
    wgu = torch.zeros(2 * f, d, device=cuda)
    wgu[:f, 0] = torch.linspace(0.0, 1.0, f, device=cuda)
    wgu[f:, 1] = 1.0
    wd = torch.eye(f, device=cuda)
    x, wgu, wd, dy = (t.to(dtype) for t in (x, wgu, wd, torch.ones(m, d, device=cuda)))
    y, gate_up, h = gated_mlp_forward(x, wgu, wd, activation=kind)
    check_forward(x, wgu, wd, kind, y, gate_up, h)
    grads = gated_mlp_backward(dy, x, wgu, wd, gate_up, h, activation=kind)
    assert all(bool(g.isfinite().all()) for g in grads)
    check_backward(dy, x, wgu, wd, gate_up, h, kind, *grads)


@pytest.mark.parametrize("m", [4, 300])
def test_nan_stays_in_its_row(cuda, m):
    x, wgu, wd, _ = operands(cuda, m, 128, 256, torch.bfloat16)
    want = gated_mlp_forward(x, wgu, wd)
    x = x.clone()
    x[1, 3] = float("nan")
    for got, was in zip(gated_mlp_forward(x, wgu, wd), want):
        assert bool(got[1].isnan().all())
        keep = torch.arange(m, device=cuda) != 1
        assert torch.equal(got[keep], was[keep])


def test_parameters_and_results_of_autograd(cuda):
    """Weights as torch's parameters: results are plain tensors, and the weights stay what they were."""
    x, wgu, wd, dy = operands(cuda, 40, 64, 96, torch.bfloat16)
    want = gated_mlp_forward(x, wgu, wd)
    grads = gated_mlp_backward(dy, x, wgu, wd, want[1], want[2])
    p, q = torch.nn.Parameter(wgu), torch.nn.Parameter(wd)
    got = gated_mlp_forward(torch.nn.Parameter(x), p, q)
    again = gated_mlp_backward(dy, x, p, q, got[1], got[2])
    for a, b in zip((*got, *again), (*want, *grads)):
        assert torch.equal(a, b) and not a.requires_grad and type(a) is torch.Tensor


def test_no_tokens(cuda):
    x, wgu, wd, dy = operands(cuda, 0, 64, 72, torch.bfloat16)
    y, gate_up, h = gated_mlp_forward(x, wgu, wd)
    assert y.shape == (0, 64) and gate_up.shape == (0, 144) and h.shape == (0, 72)
    dx, dwgu, dwd = gated_mlp_backward(dy, x, wgu, wd, gate_up, h)
    device_status()
    assert dx.shape == (0, 64) and bool((dwgu == 0).all()) and bool((dwd == 0).all())  # empty sums


@pytest.mark.parametrize("kind", ["silu", "gelu", "relu"])
def test_gradients_against_differences(cuda, kind):
    m, d, f = 6, 24, 40
    x, wgu, wd, dy = operands(cuda, m, d, f, torch.float32)
    _, gate_up, h = gated_mlp_forward(x, wgu, wd, activation=kind)
    grads = gated_mlp_backward(dy, x, wgu, wd, gate_up, h, activation=kind)
    g = torch.Generator(device=cuda).manual_seed(1)

    def loss(at):
        pre = at[0] @ at[1].t()
        return ((unit(pre[:, :f], kind) * pre[:, f:]) @ at[2].t() * dy.double()).sum()

    at = [t.double() for t in (x, wgu, wd)]
    for _ in range(3):
        along = [torch.randn(t.shape, generator=g, device=cuda).double() for t in at]
        step = 1e-6
        up, down = (loss([t + e * v for t, v in zip(at, along)]) for e in (step, -step))
        parts = torch.cat([(p.double() * v).flatten() for p, v in zip(grads, along)])
        # three float32 sums of at most 80 products in a row, each off by 2^-23 a step of magnitudes at most 8 times the value; differences: step^2 and 1e-16 / step
        assert abs((up - down) / (2 * step) - parts.sum()) <= (3 * 88 * 8 * STEP + 1e-7) * parts.abs().sum()


@pytest.mark.parametrize("m", [4, 40, 700])
def test_repeats_streams_and_graphs(cuda, m):
    """The same bits on another stream, queued behind calls on other inputs, and from graphs that are replayed on two streams at once."""
    sets = [operands(cuda, m, 256, 520, torch.bfloat16, seed=k) for k in range(2)]

    def call(s, **more):
        y, gate_up, h = gated_mlp_forward(*s[:3], **more)
        return (y, gate_up, h, *gated_mlp_backward(s[3], *s[:3], gate_up, h, **more))

    want = []
    for s in sets:
        want.append(call(s))
        torch.cuda.synchronize()
    queued = [call(sets[k % 2]) for k in range(6)]
    torch.cuda.synchronize()
    for k, out in enumerate(queued):
        assert all(torch.equal(a, b) for a, b in zip(out, want[k % 2]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = call(sets[0], stream=side.cuda_stream)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graphs, outs = [], []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(s))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for out, w in zip(outs, want) for a, b in zip(out, w))
    device_status()


@pytest.mark.parametrize("shape", [(2600, 840, 2056), (1500, 840, 2056), (1777, 1096, 1288)])
def test_products_of_one_launch_are_those_of_several(cuda, shape):
    """The backward's last products, whether they share a launch or not, give the bits of lb_gemm's with K whole."""
    m, d, f = shape
    x, wgu, wd, dy = operands(cuda, m, d, f, torch.bfloat16)
    _, gate_up, h = gated_mlp_forward(x, wgu, wd)
    dx, dwgu, dwd = gated_mlp_backward(dy, x, wgu, wd, gate_up, h)
    assert torch.equal(dwd, gemm(dy.t(), h, torch.empty_like(wd), kernel="tcgen05"))
    check_backward(dy, x, wgu, wd, gate_up, h, "silu", dx, dwgu, dwd)


def test_on_the_packages_own_tensors(cuda):
    x, wgu, wd, dy = operands(cuda, 40, 48, 64, torch.float32)
    _, gate_up, h = want = gated_mlp_forward(x, wgu, wd)
    want = (*want, *gated_mlp_backward(dy, x, wgu, wd, gate_up, h))
    region = D.Region(32 << 20)
    own = []
    for t in (x, wgu, wd, dy):
        own.append(region.empty(tuple(t.shape), "float32"))
        own[-1].copy_from_host(t.cpu().numpy())
    y, gate_up, h = gated_mlp_forward(*own[:3], stream=0)
    got = (y, gate_up, h, *gated_mlp_backward(own[3], *own[:3], gate_up, h, stream=0))
    D.synchronize()
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a.numpy(), b.cpu().numpy())
