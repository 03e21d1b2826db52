"""Norms of queries and keys with the position rotation against the formula in 64 bits: head dims, pairings, partial rotations, types, strides and
alignments of either path, positions beyond the tables, and the gradients against differences."""

import numpy as np
import pytest
import torch

from lumen_b200 import device as D
from lumen_b200.runtime import device_status, qk_norm_rope, qk_norm_rope_backward

pytestmark = pytest.mark.gpu

EPS = 1e-6
# a float32 operation is off by 2^-24; a row's statistics take at most H / 8 + 8 of them in a chain, what follows fewer than 16
STEPS32 = 64 * 2.0**-24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tables(positions, pairs, device, seed=0):
    rate = 10000.0 ** (-torch.arange(pairs, device=device, dtype=torch.float64) / pairs)
    angle = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * rate
    return angle.cos().float(), angle.sin().float()


def halves(x, pairs, interleaved):
    r = x[..., : 2 * pairs]
    ends = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :pairs], r[..., pairs:])
    return (*ends, x[..., 2 * pairs :])


def joined(a, b, rest, interleaved):
    return torch.cat(((torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)), rest), -1)


def forward64(x, w, cos, sin, rows, interleaved):
    x = x.double()
    z = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
    z = z if w is None else z * w.double()
    a, b, rest = halves(z, cos.shape[1], interleaved)
    c, s = cos.double()[rows].unsqueeze(-2), sin.double()[rows].unsqueeze(-2)
    size = joined(a.abs() * c.abs() + b.abs() * s.abs(), b.abs() * c.abs() + a.abs() * s.abs(), rest.abs(), interleaved)
    return joined(a * c - b * s, b * c + a * s, rest, interleaved), size


def backward64(dy, x, w, cos, sin, rows, interleaved):
    """The gradients and, for each, the sum of the magnitudes that it is a sum of."""
    dy, x = dy.double(), x.double()
    r = 1.0 / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
    unit = x * r
    a, b, rest = halves(dy, cos.shape[1], interleaved)
    c, s = cos.double()[rows].unsqueeze(-2), sin.double()[rows].unsqueeze(-2)
    dz = joined(a * c + b * s, b * c - a * s, rest, interleaved)
    size = joined(a.abs() * c.abs() + b.abs() * s.abs(), b.abs() * c.abs() + a.abs() * s.abs(), rest.abs(), interleaved)
    ww = torch.ones_like(x[0, 0, 0]) if w is None else w.double()
    u, u_size = dz * ww, size * ww.abs()
    dx = r * (u - unit * (u * unit).mean(-1, keepdim=True))
    dx_size = r * (u_size + unit.abs() * (u_size * unit.abs()).mean(-1, keepdim=True))
    return (dx, dx_size), ((dz * unit).sum((0, 1, 2)), (size * unit.abs()).sum((0, 1, 2)))


def close(got, want, size, chain=1.0):
    """One rounding to the result's type (subnormal float16: a step of 2^-24), and float32's of what the value is a sum of."""
    tol = half_step(got.dtype) * want.abs() * (1 + 2.0**-8) + chain * STEPS32 * size + (2.0**-25 if got.dtype == torch.float16 else 0.0)
    off = (got.double() - want).abs() - tol
    assert bool((off <= 0).all()), f"off by up to {off.max().item():.3g} more than {tol.max().item():.3g}"


def case(device, b, s, n, nk, h, dtype, seed=0, packed=True, pad=0):
    g = torch.Generator(device=device).manual_seed(seed)
    if packed:
        both = (torch.randn(b, s, n + 2 * nk, h + pad, generator=g, device=device) * 1.5).to(dtype)
        q, k = both[:, :, :n, :h], both[:, :, n : n + nk, :h]
    else:
        q, k = ((torch.randn(b, s, m, h, generator=g, device=device) * 1.5).to(dtype) for m in (n, nk))
    dq, dk = (torch.randn(b, s, m, h, generator=g, device=device).to(dtype) for m in (n, nk))
    return q, k, dq, dk, g


CASES = [
    # b, s, n, nk, h, pairs, interleaved
    (2, 5, 4, 2, 64, 32, False),
    (1, 1, 1, 1, 128, 64, False),
    (3, 33, 7, 1, 128, 64, True),
    (2, 17, 5, 5, 80, 16, False),
    (2, 17, 5, 5, 80, 40, True),
    (1, 131, 3, 2, 256, 64, False),
    (4, 9, 2, 1, 96, 48, False),
    (2, 7, 3, 3, 16, 8, True),
    (2, 7, 3, 2, 48, 8, False),
    (2, 11, 3, 2, 31, 15, False),  # odd: by the element
    (2, 11, 3, 2, 6, 1, True),
    (1, 3, 2, 1, 2, 1, False),
    (1, 3, 2, 1, 33, 1, False),
    (2, 13, 17, 3, 72, 36, False),
    (1, 700, 12, 4, 64, 32, False),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", CASES)
def test_forward_and_backward(cuda, shape, dtype):
    b, s, n, nk, h, pairs, interleaved = shape
    q, k, dq, dk, g = case(cuda, b, s, n, nk, h, dtype)
    cos, sin = tables(4 * s + 3, pairs, cuda)
    rows = torch.randint(0, 4 * s + 3, (b, s), generator=g, device=cuda)
    wq = (1 + 0.3 * torch.randn(h, generator=g, device=cuda)).to(dtype)
    wk = 1 + 0.3 * torch.randn(h, generator=g, device=cuda)  # float32, whatever the rows' type
    out = qk_norm_rope(q, k, cos, sin, positions=rows, q_weight=wq, k_weight=wk, interleaved=interleaved)
    got = qk_norm_rope_backward(dq, dk, q, k, cos, sin, positions=rows, q_weight=wq, k_weight=wk, interleaved=interleaved)
    device_status()
    for x, w, dy, y, dx, dw in ((q, wq, dq, out[0], got[0], got[2]), (k, wk, dk, out[1], got[1], got[3])):
        assert y.dtype == dx.dtype == dtype and dw.dtype == w.dtype and y.shape == dx.shape == x.shape
        close(y, *forward64(x, w, cos, sin, rows, interleaved))
        (want_dx, dx_size), (want_dw, dw_size) = backward64(dy, x, w, cos, sin, rows, interleaved)
        close(dx, want_dx, dx_size)
        close(dw, want_dw, dw_size, chain=4.0)  # at most 256 sums in a chain at these sizes


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_strides_and_alignments(cuda, dtype, pad):
    """Rows whose starts are 16-byte aligned, and rows whose are not; results into views, transposed operands, reversed tables."""
    b, s, n, nk, h = 2, 19, 4, 2, 64
    q, k, dq, dk, g = case(cuda, b, s, n, nk, h, dtype, seed=pad, pad=pad)
    wide = torch.cat(tables(64, h // 2, cuda), 1)  # both tables beside one another
    cos, sin = wide[:, : h // 2], wide[:, h // 2 :]
    rows = torch.arange(s, device=cuda) + 3
    room = torch.full((b, n + nk, s, h + pad), 7.0, dtype=dtype, device=cuda)
    out = room[:, :n, :, :h].transpose(1, 2), room[:, n:, :, :h].transpose(1, 2)  # heads outermost
    got = qk_norm_rope(q, k, cos, sin, positions=rows.int(), out=out)
    assert got[0] is out[0] and got[1] is out[1]
    both = rows.expand(b, s)
    close(out[0], *forward64(q, None, cos, sin, both, False))
    close(out[1], *forward64(k, None, cos, sin, both, False))
    assert bool((room[..., h:] == 7.0).all())  # behind the rows: as it was
    back = qk_norm_rope_backward(*(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (dq, dk)), q, k, cos, sin, positions=both)
    assert back[2] is None and back[3] is None
    close(back[0], *backward64(dq, q, None, cos, sin, both, False)[0])
    close(back[1], *backward64(dk, k, None, cos, sin, both, False)[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("h", [64, 31])
def test_results_in_the_operands_place(cuda, dtype, h):
    q, k, dq, dk, g = case(cuda, 2, 37, 6, 3, h, dtype)
    cos, sin = tables(37, h // 2, cuda)
    w = (1 + 0.1 * torch.randn(h, generator=g, device=cuda)).to(dtype)
    want = qk_norm_rope(q, k, cos, sin, q_weight=w, k_weight=w)
    want_back = qk_norm_rope_backward(dq, dk, q, k, cos, sin, q_weight=w, k_weight=w)
    back = qk_norm_rope_backward(dq, dk, q, k, cos, sin, q_weight=w, k_weight=w, out=(dq, dk))
    assert all(torch.equal(a, b) for a, b in zip(back, want_back)) and back[0] is dq
    got = qk_norm_rope(q, k, cos, sin, q_weight=w, k_weight=w, out=(q, k))
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[0] is q


@pytest.mark.parametrize("h", [64, 31])
def test_positions_are_clamped_into_the_tables(cuda, h):
    q, k, *_ = case(cuda, 1, 6, 2, 2, h, torch.float32)
    cos, sin = tables(10, h // 2, cuda)
    far = torch.tensor([-(2**40), -1, 0, 9, 10, 2**40], device=cuda)
    near = torch.tensor([0, 0, 0, 9, 9, 9], device=cuda)
    assert all(torch.equal(a, b) for a, b in zip(qk_norm_rope(q, k, cos, sin, positions=far), qk_norm_rope(q, k, cos, sin, positions=near)))
    none = qk_norm_rope(q, k, cos, sin)
    counted = qk_norm_rope(q, k, cos, sin, positions=torch.arange(6, device=cuda, dtype=torch.int32))
    assert all(torch.equal(a, b) for a, b in zip(none, counted))


@pytest.mark.parametrize("h", [64, 31])
def test_values_at_the_edges(cuda, h):
    """Zero rows give zeros (and gradients of 1 / sqrt(eps)); rows of float32's large and small values; a NaN or an infinity stays in its row."""
    x = torch.zeros(1, 6, 1, h, device=cuda)
    x[0, 1], x[0, 2] = 1e18, 1e-18
    x[0, 3, 0, 5], x[0, 4, 0, 5] = float("nan"), float("inf")
    x[0, 5] = 1.0
    cos, sin = tables(6, h // 2, cuda)
    q, _ = qk_norm_rope(x, x, cos, sin)
    d, *_ = qk_norm_rope_backward(torch.ones_like(x), torch.ones_like(x), x, x, cos, sin)
    fine = [0, 1, 2, 5]
    rows = torch.arange(6, device=cuda)[None]
    close(q[:, fine], *forward64(x[:, fine], None, cos, sin, rows[:, fine], False))
    (dx, size), _ = backward64(torch.ones_like(x), x, None, cos, sin, rows, False)
    close(d[:, fine], dx[:, fine], size[:, fine])
    assert bool(q[0, 3].isnan().all()) and bool(q[0, 4].isnan().any()) and bool(d[0, 3].isnan().all())


@pytest.mark.parametrize("shape", [(0, 4, 2, 1, 64), (2, 0, 2, 1, 64), (2, 4, 0, 0, 64), (1, 2, 3, 0, 64), (0, 4, 2, 1, 31)])
def test_nothing_to_do(cuda, shape):
    b, s, n, nk, h = shape
    q, k, dq, dk, _ = case(cuda, b, s, n, nk, h, torch.bfloat16, packed=False)
    cos, sin = tables(8, h // 2, cuda)
    w = torch.ones(h, dtype=torch.bfloat16, device=cuda)
    out = qk_norm_rope(q, k, cos, sin, q_weight=w, k_weight=w)
    assert out[0].shape == q.shape and out[1].shape == k.shape
    *_, dwq, dwk = qk_norm_rope_backward(dq, dk, q, k, cos, sin, q_weight=w, k_weight=w)
    device_status()
    assert bool((dwk == 0).all()) and (q.numel() > 0 or bool((dwq == 0).all()))  # an empty sum


@pytest.mark.parametrize("s", [3, 3001])
@pytest.mark.parametrize("h", [64, 72, 31])
def test_no_eps(cuda, h, s):
    """eps = 0, heads that no group divides: what has no row adds nothing to the weights' gradients."""
    q, k, dq, dk, g = case(cuda, 1, s, 9, 3, h, torch.float32)
    cos, sin = tables(s, h // 2 // 4 * 4, cuda)
    w = 1 + 0.3 * torch.randn(h, generator=g, device=cuda)
    zero = qk_norm_rope_backward(dq, dk, q, k, cos, sin, q_weight=w, k_weight=w, eps=0.0)
    some = qk_norm_rope_backward(dq, dk, q, k, cos, sin, q_weight=w, k_weight=w, eps=1e-30)  # float32 sees no difference
    assert all(torch.equal(a, b) and bool(a.isfinite().all()) for a, b in zip(zero, some))


@pytest.mark.parametrize("h, interleaved", [(64, False), (80, True), (31, False)])
def test_gradients_against_differences(cuda, h, interleaved):
    q, k, dq, dk, g = case(cuda, 2, 3, 2, 1, h, torch.float32)
    pairs = h // 2
    cos, sin = tables(16, pairs, cuda)
    rows = torch.randint(0, 16, (2, 3), generator=g, device=cuda)
    w = 1 + 0.3 * torch.randn(h, generator=g, device=cuda)
    got = qk_norm_rope_backward(dq, dk, q, k, cos, sin, positions=rows, q_weight=w, k_weight=w, interleaved=interleaved)
    for x, dy, dx, dw in ((q, dq, got[0], got[2]), (k, dk, got[1], got[3])):
        for _ in range(3):
            vx, vw = torch.randn(x.shape, generator=g, device=cuda).double(), torch.randn(h, generator=g, device=cuda).double()
            step = 1e-5
            up, down = ((forward64(x.double() + e * vx, w.double() + e * vw, cos, sin, rows, interleaved)[0] * dy.double()).sum() for e in (step, -step))
            parts = torch.cat(((dx.double() * vx).flatten(), dw.double() * vw))
            # float32 gradients: 64 roundings of each part's magnitude, at most twice its own where rows cancel; differences: step^2 and 1e-16 / step
            assert abs((up - down) / (2 * step) - parts.sum()) <= 4 * STEPS32 * parts.abs().sum() * 8 + 1e-7 * parts.abs().sum()


@pytest.mark.parametrize("n, nk, h, pairs, interleaved, dtype", [(16, 4, 64, 32, False, torch.bfloat16), (7, 5, 128, 64, False, torch.float16), (15, 1, 80, 16, True, torch.float32),
                                                                 (13, 3, 256, 128, False, torch.bfloat16), (9, 3, 31, 15, False, torch.bfloat16)])  # fmt: skip
def test_many_rows_repeat_bit_for_bit_and_agree_with_few(cuda, n, nk, h, pairs, interleaved, dtype):
    """More rows than the grid has threads, numbers of heads that nothing divides: weights' gradients add up in a fixed order, and a row alone
    is what it is among others, to a rounding."""
    q, k, dq, dk, g = case(cuda, 3, 2501, n, nk, h, dtype)
    cos, sin = tables(2501, pairs, cuda)
    w = (1 + 0.3 * torch.randn(h, generator=g, device=cuda)).to(dtype)
    first = qk_norm_rope_backward(dq, dk, q, k, cos, sin, q_weight=w, k_weight=w, interleaved=interleaved)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, qk_norm_rope_backward(dq, dk, q, k, cos, sin, q_weight=w, k_weight=w, interleaved=interleaved)))
    rows = torch.arange(2501, device=cuda).expand(3, 2501)
    for x, dy, dx, dw in ((q, dq, first[0], first[2]), (k, dk, first[1], first[3])):
        (want_dx, dx_size), (want_dw, dw_size) = backward64(dy, x, w, cos, sin, rows, interleaved)
        close(dx, want_dx, dx_size)
        close(dw, want_dw, dw_size, chain=4.0)
    whole = qk_norm_rope(q, k, cos, sin, q_weight=w, k_weight=w, interleaved=interleaved)
    for at in (0, 1, 1250, 2500):
        one = qk_norm_rope(q[1:2, at : at + 1], k[1:2, at : at + 1], cos, sin, positions=torch.tensor([at], device=cuda), q_weight=w, k_weight=w, interleaved=interleaved)
        for a, b, x in ((one[0][0, 0], whole[0][1, at], q[1, at]), (one[1][0, 0], whole[1][1, at], k[1, at])):  # another kernel adds a row up in another order
            want, size = forward64(x, w, cos, sin, torch.tensor(at, device=cuda), interleaved)
            close(a, want, size)
            close(b, want, size)


def test_streams_graphs_and_overlapping_calls(cuda):
    """Another stream than the current one, and two graphs of the backward pass replayed on two streams at once: each call has its own workspace."""
    sets = []
    for seed in range(2):
        q, k, dq, dk, g = case(cuda, 2, 333, 8, 2, 64, torch.bfloat16, seed=seed)
        w = (1 + 0.3 * torch.randn(64, generator=g, device=cuda)).to(torch.bfloat16)
        sets.append((dq, dk, q, k, w))
    cos, sin = tables(333, 32, cuda)

    def call(s, **more):
        return qk_norm_rope_backward(*s[:4], cos, sin, q_weight=s[4], k_weight=s[4], **more)

    want = [call(s) for s in sets]
    torch.cuda.synchronize()
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


def test_on_the_packages_own_tensors(cuda):
    """The same bits from tensors of the package's own memory."""
    q, k, dq, dk, g = case(cuda, 1, 9, 4, 2, 64, torch.float32, packed=False)
    cos, sin = tables(9, 32, cuda)
    w = 1 + 0.3 * torch.randn(64, generator=g, device=cuda)
    want = (*qk_norm_rope(q, k, cos, sin, q_weight=w, k_weight=w), *qk_norm_rope_backward(dq, dk, q, k, cos, sin, q_weight=w, k_weight=w))
    region = D.Region(32 << 20)

    def own(t):
        x = region.empty(tuple(t.shape), "float32")
        x.copy_from_host(t.cpu().numpy())
        return x

    q, k, dq, dk, cos, sin, w = (own(t) for t in (q, k, dq, dk, cos, sin, w))
    got = (*qk_norm_rope(q, k, cos, sin, q_weight=w, k_weight=w, stream=0), *qk_norm_rope_backward(dq, dk, q, k, cos, sin, q_weight=w, k_weight=w, stream=0))
    D.synchronize()
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a.numpy(), b.cpu().numpy())
