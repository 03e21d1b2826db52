"""Softmax cross entropy of a projection to a vocabulary and its backward pass against the formula in 64 bits: one token to many, vocabularies around
the spans and in several pieces, every type and reduction, rows that do not count and what may stand in them, layouts, and the gradients against differences."""

import numpy as np
import pytest
import torch

from lumen_b200 import device as D
from lumen_b200.runtime import device_status, linear_cross_entropy, linear_cross_entropy_backward

pytestmark = pytest.mark.gpu

# A float32 sum of K products drops at most 2^-23 of the running sum's magnitude a step.
STEP = 2.0**-23
IGNORED = -100


def half(dtype):
    return torch.finfo(dtype).eps / 2 * (1 + 2.0**-8)


def within(got, want, tol, what):
    off = (got.double() - want).abs() - tol
    assert bool((off <= 0).all()), f"{what}: off by up to {off.max().item():.3g} more than allowed"


def operands(cuda, t, d, v, dtype, ignored=0.0, seed=0, scale=1.5):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = torch.randn((t, d), generator=g, device=cuda).to(dtype)
    w = (torch.randn((v, d), generator=g, device=cuda) * scale * d**-0.5).to(dtype)
    targets = torch.randint(0, v, (t,), generator=g, device=cuda)
    targets[torch.rand(t, generator=g, device=cuda) < ignored] = IGNORED
    return x, w, targets


def logits_of(x, w):
    """The logits in 64 bits, how far float32 sums may be off, and the largest of each row."""
    x, w = x.double(), w.double()
    return x @ w.t(), (x.shape[1] + 8) * STEP * (x.abs() @ w.abs().t())


def check_forward(x, w, targets, reduction, loss, lse, ignored=IGNORED):
    z, off = logits_of(x, w)
    v = w.shape[0]
    want = torch.logsumexp(z, -1)
    # exponentials within 2^-21 (argument's rounding apart), each of up to V / 128 + 64 sums of a row in a chain rounded; largest logit and logarithm rounded
    tol = off.amax(-1) + (v / 128 + 64) * 2.0**-21 + 2.0**-21 * (want.abs() + z.abs().amax(-1))
    within(lse, want, tol, "lse")
    counts = targets != ignored
    at = targets.clamp(0, v - 1)[:, None]
    losses = torch.where(counts, want - z.gather(-1, at)[:, 0], 0.0)
    tol = torch.where(counts, tol + off.gather(-1, at)[:, 0] + 2.0**-23 * (want.abs() + losses.abs()), 0.0)
    if reduction == "none":
        return within(loss, losses, tol, "loss")
    n = max(1, int(counts.sum())) if reduction == "mean" else 1
    within(loss, losses.sum() / n, tol.sum() / n + 2.0**-23 * losses.sum().abs() / n, "loss")


def check_backward(x, w, targets, lse, reduction, d_loss, d_x, d_w, ignored=IGNORED, rounding=None):
    dtype, v = x.dtype, w.shape[0]
    counts = targets != ignored
    x = torch.where(counts[:, None], x, 0.0)
    z, off = logits_of(x, w)
    g = counts.double() * (1.0 if d_loss is None else d_loss.double())
    if reduction == "mean":
        g = g / max(1, int(counts.sum()))
    p = torch.exp(z - lse.double()[:, None])
    hit = torch.nn.functional.one_hot(targets.clamp(0, v - 1), v)
    dz = torch.where(counts[:, None], (p - hit) * g[:, None], 0.0)
    # p by its argument's error (that of the logit, of the products with log2 e) and the exponential's, g by its quotient's, dz by its rounding;
    # float16's dz is scaled so that the largest |g| is 2^12 or more, and is rounded to multiples of 2^-24 or finer
    dz_off = p * (off + 2.0**-20 + 2.0**-22 * (z.abs() + lse.double().abs()[:, None])) * g.abs()[:, None] + dz.abs() * (2.0**-21 + (rounding if rounding is not None else half(dtype) if dtype != torch.float32 else 0))
    dz_off = torch.where(counts[:, None], dz_off + (2.0**-37 * g.abs().max() if dtype == torch.float16 else 1e-37), 0.0)
    tiny = 2.0**-25 if dtype == torch.float16 else 1e-37

    def sums(a, a_off, b, n, got, what):
        want, b = a @ b, b.abs()
        within(got, want, half(dtype) * want.abs() + a_off @ b + (n + 8) * STEP * ((a.abs() + a_off) @ b) * (1 + half(dtype)) + tiny, what)

    sums(dz, dz_off * (1 + half(dtype)), w.double(), v, d_x, "d_x")
    sums(dz.t(), dz_off.t() * (1 + half(dtype)), x.double(), x.shape[0], d_w, "d_weight")


SHAPES = [
    # tokens, width, classes
    (1, 64, 256), (1, 1024, 5000), (2, 8, 1), (2, 16, 2), (3, 40, 7), (4, 256, 30011), (7, 136, 129), (8, 512, 4096), (9, 64, 1000), (16, 328, 2048), (17, 72, 5003),
    (31, 104, 127), (32, 512, 513), (33, 64, 128), (61, 1024, 4099), (100, 264, 255), (127, 40, 257), (128, 128, 256), (129, 256, 1031), (200, 8, 12000),
    (256, 128, 256), (257, 520, 385), (300, 1120, 3001), (511, 72, 129), (700, 8, 8), (1000, 320, 1160), (1531, 96, 700), (2600, 64, 520), (5000, 16, 40),
    (20000, 8, 9), (5, 15, 9), (40, 33, 70), (130, 100, 61), (600, 24, 1), (65, 4096, 300), (1400, 520, 4001), (2600, 840, 3001), (3000, 264, 10000), (300, 101, 2003),
]  # fmt: skip


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_backward(cuda, shape, dtype):
    t, d, v = shape
    x, w, targets = operands(cuda, t, d, v, dtype, ignored=0.2 * (t % 2), seed=t + d)
    g = torch.Generator(device=cuda).manual_seed(3)
    for reduction in ("none", "sum", "mean"):
        loss, lse = linear_cross_entropy(x, w, targets, reduction=reduction)
        assert loss.shape == (targets.shape if reduction == "none" else ()) and lse.shape == targets.shape and loss.dtype == lse.dtype == torch.float32
        check_forward(x, w, targets, reduction, loss, lse)
        d_loss = torch.randn(t, generator=g, device=cuda) if reduction == "none" else torch.full((), 0.75, device=cuda) if reduction == "sum" else None
        d_x, d_w = linear_cross_entropy_backward(d_loss, x, w, targets, lse, reduction=reduction)
        assert d_x.shape == x.shape and d_w.shape == w.shape and d_x.dtype == d_w.dtype == dtype
        check_backward(x, w, targets, lse, reduction, d_loss, d_x, d_w)
    device_status()


@pytest.mark.parametrize("dtype, shape", [(torch.bfloat16, (600, 16, 230001)), (torch.float16, (610, 16, 230001)), (torch.float32, (600, 16, 120001)), (torch.bfloat16, (600, 15, 120001)), (torch.float32, (60, 8, 1200001)), (torch.float32, (16, 8, 4300001)),
                                          (torch.bfloat16, (8192, 1024, 20001)), (torch.float16, (8200, 1000, 20001))])  # fmt: skip
def test_a_vocabulary_in_several_pieces(cuda, dtype, shape):
    x, w, targets = operands(cuda, *shape, dtype, ignored=0.1)
    targets[0], targets[1] = shape[2] - 1, 0
    loss, lse = linear_cross_entropy(x, w, targets)
    check_forward(x, w, targets, "mean", loss, lse)
    check_backward(x, w, targets, lse, "mean", None, *linear_cross_entropy_backward(None, x, w, targets, lse))
    device_status()


@pytest.mark.parametrize("t", [3, 40])
def test_offsets_past_32_bits(cuda, t):
    """Weights and their gradient of more than 2^31 elements."""
    d, v = 16384, 140001
    x, w, targets = operands(cuda, t, d, v, torch.bfloat16)
    targets[0], targets[1], targets[2] = v - 1, v - 5, IGNORED
    loss, lse = linear_cross_entropy(x, w, targets, reduction="none")
    z, off = (torch.cat(parts, 1) for parts in zip(*(logits_of(x, some) for some in w.split(8192))))
    want = torch.logsumexp(z, -1)
    within(lse, want, off.amax(-1) + (v / 128 + 64) * 2.0**-21 + 2.0**-21 * (want.abs() + z.abs().amax(-1)), "lse")
    assert float(loss[2]) == 0 and abs(float(loss[0]) - float(want[0] - z[0, v - 1])) < 1e-3
    d_x, d_w = linear_cross_entropy_backward(None, x, w, targets, lse, reduction="none")
    last = slice(v - 300, v)
    counts = (targets != IGNORED)[:, None]
    dz = (torch.exp(z - lse.double()[:, None]) - torch.nn.functional.one_hot(targets.clamp(min=0), v)) * counts
    for rows in (last, slice(0, 300)):  # a gradient's every term is a rounded dz times an element
        part = dz[:, rows].t()
        within(d_w[rows], part @ x.double(), 2 * half(torch.bfloat16) * (part.abs() @ x.double().abs()) + 1e-6, "d_weight")
    want = sum(dz[:, k : k + 8192] @ w[k : k + 8192].double() for k in range(0, v, 8192))
    size = sum(dz[:, k : k + 8192].abs() @ w[k : k + 8192].double().abs() for k in range(0, v, 8192))
    within(d_x, want, 2 * half(torch.bfloat16) * size, "d_x")


@pytest.mark.parametrize("dtype, shape", [(torch.bfloat16, (300001, 8, 16385)), (torch.float32, (70001, 8, 300)), (torch.float16, (66001, 7, 40))])
def test_rows_in_several_rounds(cuda, dtype, shape):
    x, w, targets = operands(cuda, *shape, dtype, ignored=0.1)
    mean, lse = linear_cross_entropy(x, w, targets)
    losses, again = linear_cross_entropy(x, w, targets, reduction="none")
    assert torch.equal(lse, again)
    some = torch.cat((torch.arange(0, shape[0], shape[0] // 999, device=cuda), torch.arange(shape[0] - 300, shape[0], device=cuda)))
    check_forward(x[some], w, targets[some], "none", losses[some], lse[some])
    counts = int((targets != IGNORED).sum())
    total = float(losses.double().sum())
    assert abs(float(mean) - total / counts) <= 2.0**-23 * abs(total) / counts
    device_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t", [4, 6, 25, 300])
def test_what_stands_in_rows_that_do_not_count(cuda, t, dtype):
    x, w, targets = operands(cuda, t, 72, 500, dtype, ignored=0.4)
    targets[:3] = IGNORED
    targets[3] = 7
    want = [linear_cross_entropy(x, w, targets, reduction=r) for r in ("none", "mean")]
    grads = linear_cross_entropy_backward(None, x, w, targets, want[1][1])
    y = x.clone()
    y[0], y[1], y[2, 5] = float("nan"), float("inf"), float("-inf")
    for k, r in enumerate(("none", "mean")):
        loss, lse = linear_cross_entropy(y, w, targets, reduction=r)
        assert torch.equal(loss, want[k][0]) and torch.equal(lse[3:], want[k][1][3:])
    got = linear_cross_entropy_backward(None, y, w, targets, lse)
    assert torch.equal(got[0], grads[0]) and torch.equal(got[1], grads[1]) and not got[0][targets == IGNORED].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("t", [1, 40, 300])
def test_no_row_counts(cuda, t, dtype):
    x, w, targets = operands(cuda, t, 64, 300, dtype)
    targets[:] = IGNORED
    for reduction in ("none", "sum", "mean"):
        loss, lse = linear_cross_entropy(x, w, targets, reduction=reduction)
        assert not loss.any() and bool(torch.isfinite(lse).all())
        d_x, d_w = linear_cross_entropy_backward(None, x, w, targets, lse, reduction=reduction)
        assert not d_x.any() and not d_w.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_rows(cuda, dtype):
    x, w, targets = operands(cuda, 0, 64, 300, dtype)
    loss, lse = linear_cross_entropy(x, w, targets)
    assert float(loss) == 0 and lse.shape == (0,)
    d_x, d_w = linear_cross_entropy_backward(None, x, w, targets, lse)
    assert d_x.shape == (0, 64) and d_w.shape == w.shape and not d_w.any()
    assert linear_cross_entropy(x, w, targets, reduction="none")[0].shape == (0,)


@pytest.mark.parametrize("t", [5, 200])
def test_classes_outside_the_vocabulary_and_what_is_ignored(cuda, t):
    x, w, targets = operands(cuda, t, 64, 300, torch.bfloat16)
    targets[0], targets[1], targets[2] = -5, 300, 2**40 + 3
    clamped = targets.clamp(0, 299)
    for ignored in (-100, 17, int(clamped[3])):
        a, b = (linear_cross_entropy(x, w, ids, reduction="none", ignore_index=ignored) for ids in (targets, clamped))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        check_forward(x, w, clamped, "none", *a, ignored=ignored)
        a, b = (linear_cross_entropy_backward(None, x, w, ids, a[1], reduction="none", ignore_index=ignored) for ids in (targets, clamped))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    narrow = clamped.int()
    assert torch.equal(linear_cross_entropy(x, w, narrow)[0], linear_cross_entropy(x, w, clamped)[0])
    # what is ignored is told before anything is clamped
    assert float(linear_cross_entropy(x, w, targets, reduction="none", ignore_index=300)[0][1]) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t", [4, 6, 14, 30, 260])
def test_layouts(cuda, t, dtype):
    x, w, targets = operands(cuda, t, 64, 300, dtype, ignored=0.2)
    want_loss, want_lse = linear_cross_entropy(x, w, targets, reduction="none")
    g = torch.rand(t, device=cuda)
    want = linear_cross_entropy_backward(g, x, w, targets, want_lse, reduction="none")

    def near(a, b):  # another layout may take another kernel: both within half a step and the sums' roundings of the same values
        assert float((a.double() - b.double()).norm()) <= 4 * half(dtype if a.dtype == dtype else torch.float32) * (1 if dtype != torch.float32 else 64) * float(b.double().norm()) + 1e-4 * (a.dtype != dtype)

    wide = torch.randn(t, 100, device=cuda).to(dtype)
    wide[:, 20:84] = x
    every = [(wide[:, 20:84], w), (wide[:, 20:84].clone().t().contiguous().t(), w), (x, w.t().contiguous().t()), (x.view(2, t // 2, 64), w)]
    spread = torch.zeros(t, 3, dtype=torch.int64, device=cuda)
    spread[:, 1] = targets
    lse3 = torch.zeros(t, 2, device=cuda)
    lse3[:, 0] = want_lse
    for x2, w2 in every:
        lead = x2.shape[:-1]
        ids = spread[:, 1] if x2.dim() == 2 else targets.view(lead)
        loss, lse = linear_cross_entropy(x2, w2, ids, reduction="none")
        assert loss.shape == lse.shape == lead
        near(loss.reshape(-1), want_loss), near(lse.reshape(-1), want_lse)
        d_x, d_w = linear_cross_entropy_backward(g.view(lead), x2, w2, ids, lse3[:, 0] if x2.dim() == 2 else want_lse.view(lead), reduction="none")
        assert d_x.shape == x2.shape
        near(d_x.reshape(t, 64), want[0]), near(d_w, want[1])
    # one gradient for all rows, as a broadcast view
    one = torch.full((1,), 0.5, device=cuda)
    a = linear_cross_entropy_backward(one.expand(t), x, w, targets, want_lse, reduction="none")
    b = linear_cross_entropy_backward(torch.full((t,), 0.5, device=cuda), x, w, targets, want_lse, reduction="none")
    c = linear_cross_entropy_backward(one.view(()), x, w, targets, want_lse, reduction="sum")
    assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(a, b, c))
    # a single row
    loss, lse = linear_cross_entropy(x[3], w, targets[3], reduction="none")
    assert loss.shape == lse.shape == ()
    near(lse, want_lse[3])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("t", [3, 12, 30, 150])
def test_logits_of_any_size(cuda, t, dtype):
    x, w, targets = operands(cuda, t, 64, 400, dtype, scale=600.0)  # up to some thousands: exponentials of them are infinite
    loss, lse = linear_cross_entropy(x, w, targets, reduction="none")
    check_forward(x, w, targets, "none", loss, lse)
    check_backward(x, w, targets, lse, "none", None, *linear_cross_entropy_backward(None, x, w, targets, lse, reduction="none"))
    x[1, 0] = float("nan")  # stays in its row
    loss, lse = linear_cross_entropy(x, w, targets, reduction="none")
    bad = torch.isnan(lse)
    assert bad[1] and int(bad.sum()) == 1 and int(torch.isnan(loss).sum()) == 1
    w[5] = float("-inf")
    x[:] = 1.0
    loss, lse = linear_cross_entropy(x, w, torch.zeros_like(targets), reduction="none")
    assert bool(torch.isfinite(lse).all()) and bool(torch.isfinite(loss).all())


@pytest.mark.parametrize("scale", [2.0**-12, 1.0, 2.0**14])
def test_small_and_large_gradients_in_float16(cuda, scale):
    """What reaches the products keeps float16's precision whatever the loss is scaled by."""
    x, w, targets = operands(cuda, 400, 64, 300, torch.float16, ignored=0.2)
    _, lse = linear_cross_entropy(x, w, targets)
    d_loss = torch.full((), scale, device=cuda)
    check_backward(x, w, targets, lse, "mean", d_loss, *linear_cross_entropy_backward(d_loss, x, w, targets, lse))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(65, 64, 1031), (200, 64, 1031), (100, 15, 1031), (1100, 128, 2000), (2000, 1024, 4000)], ids=lambda s: "x".join(map(str, s)))
def test_one_gradient_of_all_rows_is_not_rounded(cuda, shape, dtype):
    """A gradient in the middle of two values of the type: dz is (p - [class]) times it, and only the first is rounded: by half a step of values
    below one where the class is the row's, by half a step of any value elsewhere."""
    t, d, v = shape
    x, w, targets = operands(cuda, t, d, v, dtype, seed=5, scale=0.1)
    targets.copy_(torch.randperm(v, device=cuda)[:t])
    _, lse = linear_cross_entropy(x, w, targets, reduction="sum")
    d_loss = torch.full((), 1.0 + torch.finfo(dtype).eps / 2, device=cuda)
    d_x, d_w = linear_cross_entropy_backward(d_loss, x, w, targets, lse, reduction="sum")
    rounding = torch.full((t, v), half(dtype), device=cuda, dtype=torch.float64)
    rounding[torch.arange(t, device=cuda), targets] = half(dtype) / 2 * (1 + 2.0**-8)  # of a value above 1 - 2^-8
    check_backward(x, w, targets, lse, "sum", d_loss, d_x, d_w, rounding=rounding)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 64, 300), (2, 8, 1), (14, 328, 5003), (33, 15, 130), (40, 33, 70), (64, 1024, 4096), (60, 16, 2300001)], ids=lambda s: "x".join(map(str, s)))
def test_few_rows_gradients_are_rounded_once(cuda, shape, dtype):
    """dz in two parts: half a step of half a step is left."""
    t, d, v = shape
    x, w, targets = operands(cuda, t, d, v, dtype, ignored=0.2 * (t % 2 and t > 1), seed=t)
    g = torch.Generator(device=cuda).manual_seed(3)
    for reduction in ("none", "mean"):
        _, lse = linear_cross_entropy(x, w, targets, reduction=reduction)
        d_loss = torch.randn(t, generator=g, device=cuda) if reduction == "none" else None
        d_x, d_w = linear_cross_entropy_backward(d_loss, x, w, targets, lse, reduction=reduction)
        check_backward(x, w, targets, lse, reduction, d_loss, d_x, d_w, rounding=half(dtype) ** 2)
    device_status()


@pytest.mark.parametrize("t", [5, 70, 300])
def test_gradients_against_differences(cuda, t):
    x, w, targets = operands(cuda, t, 48, 200, torch.float32, ignored=0.2)
    loss, lse = linear_cross_entropy(x, w, targets)
    d_x, d_w = linear_cross_entropy_backward(None, x, w, targets, lse)
    g = torch.Generator(device=cuda).manual_seed(1)
    for which, grad in ((0, d_x), (1, d_w)):
        along = torch.randn(grad.shape, generator=g, device=cuda)
        along /= along.norm()
        step = 2.0**-4
        at = [x, w]
        values = []
        for sign in (1, -1):
            moved = list(at)
            moved[which] = at[which] + sign * step * along
            values.append(linear_cross_entropy(moved[0], moved[1], targets, reduction="none")[0].double())
        n = int((targets != IGNORED).sum())
        slope = float((values[0] - values[1]).sum()) / (2 * step) / n
        # a central difference is off by step^2 / 6 times the third derivative along the unit vector: (|x| or |w| times a row's part of it)^3, at most 8^3 / n here over
        # the rows; each loss by 2^-19 / step
        size = 8.0**3 * step**2 / 6 + 2.0**-19 / step
        assert abs(slope - float((grad.double() * along.double()).sum())) <= size * n**-0.5


@pytest.mark.parametrize("shape", [(4, 256, 3000), (200, 256, 3000), (300, 72, 500)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_repeats_replays_and_streams(cuda, shape, dtype):
    x, w, targets = operands(cuda, *shape, dtype, ignored=0.1)

    def both():
        loss, lse = linear_cross_entropy(x, w, targets)
        return loss, lse, *linear_cross_entropy_backward(loss, x, w, targets, lse)

    want = both()
    graphs, got = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            got.append(both())
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        there = [both() for _ in range(3)]
    here = [both() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(2):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for out in (*got, *there, *here):
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    given = torch.cuda.Stream()
    given.wait_stream(torch.cuda.current_stream())
    loss, lse = linear_cross_entropy(x, w, targets, stream=given.cuda_stream)
    grads = linear_cross_entropy_backward(loss, x, w, targets, lse, stream=given.cuda_stream)
    given.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((loss, lse, *grads), want))


def test_on_the_packages_own_tensors(cuda):
    x, w, targets = operands(cuda, 40, 64, 300, torch.float32)
    loss, lse = linear_cross_entropy(x, w, targets)
    want = loss, lse, *linear_cross_entropy_backward(None, x, w, targets, lse)
    region = D.Region(32 << 20)
    own = []
    for t, dtype in ((x, "float32"), (w, "float32"), (targets, "int64")):
        own.append(region.empty(tuple(t.shape), dtype))
        own[-1].copy_from_host(t.cpu().numpy())
    loss, lse = linear_cross_entropy(*own, stream=0)
    got = loss, lse, *linear_cross_entropy_backward(None, *own, lse, stream=0)
    D.synchronize()
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a.numpy(), b.cpu().numpy())
