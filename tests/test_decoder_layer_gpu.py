"""A decoder layer's training step from the package's kernels alone - packed projection, norms and rotation of queries and keys, attention, projection,
gated block, each one's backward pass, clipping of all gradients - against the same layer differentiated in 64 bits; eager, and replayed from a
captured graph while eager graphs of the same leaves live."""

import math

import pytest
import torch

from lumen_b200.runtime import attention_backward, attention_forward, clip_grad_norm, device_status, gated_mlp_backward, gated_mlp_forward, gemm, qk_norm_rope, qk_norm_rope_backward

pytestmark = pytest.mark.gpu

EPS = 1e-6


def layer(cuda, b, s, n, nk, h, f, dtype, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    d = n * h

    def normal(*shape, scale):
        return (torch.randn(shape, generator=g, device=cuda) * scale).to(dtype)

    p = {"wqkv": normal((n + 2 * nk) * h, d, scale=d**-0.5), "wq": 1 + normal(h, scale=0.2), "wk": 1 + normal(h, scale=0.2), "wo": normal(d, d, scale=d**-0.5),
         "wgu": normal(2 * f, d, scale=d**-0.5), "wd": normal(d, f, scale=f**-0.5)}  # fmt: skip
    angle = torch.arange(s + 5, device=cuda, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(h // 2, device=cuda, dtype=torch.float64) / (h // 2))
    return p, normal(b, s, d, scale=1.0), normal(b, s, d, scale=0.3), angle.cos().float(), angle.sin().float(), torch.arange(s, device=cuda) + 5


def step(p, x, dy, cos, sin, positions, n, nk, h, max_norm):
    b, s, d = x.shape
    rows = x.reshape(b * s, d)

    def product(a, w, **more):
        return gemm(a, w, torch.empty(a.shape[0], w.shape[1], dtype=a.dtype, device=a.device), **more)

    qkv = product(rows, p["wqkv"].t()).view(b, s, n + 2 * nk, h)
    q, k, v = qkv.split((n, nk, nk), 2)
    at = {"positions": positions, "q_weight": p["wq"], "k_weight": p["wk"], "eps": EPS}
    qr, kr = qk_norm_rope(q, k, cos, sin, **at)
    o, lse = attention_forward(qr, kr, v, causal=True)
    u = product(o.view(b * s, d), p["wo"].t()) + rows
    y, gate_up, hidden = gated_mlp_forward(u, p["wgu"], p["wd"])
    y = y + u
    # backward
    dy2 = dy.reshape(b * s, d)
    du, dwgu, dwd = gated_mlp_backward(dy2, u, p["wgu"], p["wd"], gate_up, hidden)
    du = du + dy2
    do = product(du, p["wo"])
    dwo = product(du.t(), o.view(b * s, d))
    dqr, dkr, dv = attention_backward(qr, kr, v, o, do.view(b, s, n, h), lse, causal=True)
    d_qkv = torch.empty_like(qkv)
    dq, dk, dwq, dwk = qk_norm_rope_backward(dqr, dkr, q, k, cos, sin, out=(d_qkv[:, :, :n], d_qkv[:, :, n : n + nk]), **at)
    d_qkv[:, :, n + nk :] = dv
    d_qkv = d_qkv.view(b * s, -1)
    dx = product(d_qkv, p["wqkv"]) + du
    dwqkv = product(d_qkv.t(), rows)
    grads = {"wqkv": dwqkv, "wq": dwq, "wk": dwk, "wo": dwo, "wgu": dwgu, "wd": dwd}
    norm = clip_grad_norm(list(grads.values()), max_norm)
    return y.view(b, s, d), dx.view(b, s, d), norm, grads


def reference(p, x, dy, cos, sin, positions, n, nk, h):
    p = {k: v.double().requires_grad_() for k, v in p.items()}
    x = x.double().requires_grad_()
    b, s, d = x.shape
    q, k, v = (x @ p["wqkv"].t()).view(b, s, n + 2 * nk, h).split((n, nk, nk), 2)
    c, sn = cos.double()[positions][:, None], sin.double()[positions][:, None]

    def turned(t, w):
        z = t / (t.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w
        a, e = z.chunk(2, -1)
        return torch.cat((a * c - e * sn, e * c + a * sn), -1)

    q, k = turned(q, p["wq"]), turned(k, p["wk"])
    k, v = (t.repeat_interleave(n // nk, 2) for t in (k, v))
    scores = torch.einsum("bqnh,bknh->bnqk", q, k) / math.sqrt(h)
    scores = scores.masked_fill(torch.ones(s, s, device=x.device, dtype=torch.bool).triu(1), float("-inf"))
    o = torch.einsum("bnqk,bknh->bqnh", scores.softmax(-1), v).reshape(b, s, d)
    u = o @ p["wo"].t() + x
    gate, up = (u @ p["wgu"].t()).chunk(2, -1)
    y = (torch.nn.functional.silu(gate) * up) @ p["wd"].t() + u
    grads = torch.autograd.grad((y * dy.double()).sum(), (x, *p.values()))
    return y.detach(), grads[0], dict(zip(p, grads[1:]))


def far(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("shape, dtype", [((2, 130, 4, 2, 64, 520), torch.bfloat16), ((1, 257, 2, 1, 128, 328), torch.bfloat16), ((2, 33, 3, 1, 32, 72), torch.float32)])
def test_a_layers_training_step(cuda, shape, dtype):
    b, s, n, nk, h, f = shape
    p, x, dy, cos, sin, positions = layer(cuda, *shape, dtype)
    y_want, dx_want, want = reference(p, x, dy, cos, sin, positions, n, nk, h)
    total = math.sqrt(sum(float(t.square().sum()) for t in want.values()))
    y, dx, norm, grads = step(p, x, dy, cos, sin, positions, n, nk, h, 0.25 * total)
    device_status()
    # about twenty roundings lie between inputs and the last gradients, each at most half a step of its value; the layer passes on at most four times a
    # relative error (softmax, norm). In float32, sums of up to a few hundred products take a rounding's place.
    allowed = 20 * 4 * torch.finfo(dtype).eps / 2 * (1 if dtype == torch.bfloat16 else 64) / (2 if dtype == torch.bfloat16 else 1)
    assert far(y, y_want) < allowed and far(dx, dx_want) < allowed
    assert abs(float(norm) - total) < allowed * total
    for name, t in want.items():
        assert far(grads[name], t * 0.25) < 2 * allowed, name


def test_a_captured_step_beside_eager_ones(cuda):
    shape = (1, 130, 4, 2, 64, 264)
    b, s, n, nk, h, f = shape
    p, x, dy, cos, sin, positions = layer(cuda, *shape, torch.bfloat16)
    p = {k: v.requires_grad_() for k, v in p.items()}
    alive = sum((v.float() ** 2).sum() for v in p.values())  # an eager graph of the same leaves
    with torch.no_grad():
        want = step(p, x, dy, cos, sin, positions, n, nk, h, 1.0)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(p, x, dy, cos, sin, positions, n, nk, h, 1.0)
        for _ in range(3):
            graph.replay()
        again = step(p, x, dy, cos, sin, positions, n, nk, h, 1.0)
    alive.backward()
    torch.cuda.synchronize()
    for out in (got, again):
        assert all(torch.equal(a, b) for a, b in zip(out[:3], want[:3])) and all(torch.equal(out[3][k], want[3][k]) for k in want[3])
    assert all(torch.equal(v.grad, (2 * v.detach().float()).to(v.dtype)) for v in p.values())
