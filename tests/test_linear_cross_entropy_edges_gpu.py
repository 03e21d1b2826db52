"""Softmax cross entropy of a projection where its ways through the kernels end: pieces of the vocabulary with a single class or too few for a shared launch, infinities, NaN and the
largest values in what counts, logits far from zero, widths whose gradient no tile stores."""

import pytest
import torch

from lumen_b200.runtime import device_status, linear_cross_entropy, linear_cross_entropy_backward
from tests.test_linear_cross_entropy_gpu import IGNORED, check_backward, check_forward, half, operands, within

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


def defined(x, w, targets):
    """Losses, log-sum-exp and the gradients of the losses' sum by the definition in 64 bits, whatever x and w hold."""
    x, w = x.double(), w.double()
    z = x @ w.t()
    counts, at = targets != IGNORED, targets.clamp(min=0)[:, None]
    lse = torch.logsumexp(z, -1)
    loss = torch.where(counts, lse - z.gather(-1, at)[:, 0], 0.0)
    p = torch.exp(z - lse[:, None]) - torch.nn.functional.one_hot(at[:, 0], w.shape[0])
    dz = torch.where(counts[:, None], p, 0.0)
    return loss, lse, dz @ w, dz.t() @ torch.where(counts[:, None], x, 0.0)


def check_infinities(got, want, what):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN"
    assert torch.equal(got == float("inf"), want == float("inf")) and torch.equal(got == float("-inf"), want == float("-inf")), f"{what}: infinities"


def check_finite(got, want, what):
    """Where an infinity meets the zeros that a float32 value's or a gradient's smaller parts are, it is NaN."""
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), what


# every way: a token on the CUDA cores and on the tensor cores, a few, with and without vectors, some, tiles of one CTA and of two, logits in memory
INFINITE = [(1, 600, 500), (2, 600, 500), (3, 72, 500), (6, 72, 500), (6, 73, 500), (14, 72, 500), (25, 72, 500), (25, 73, 500), (40, 72, 500), (60, 72, 9001), (300, 72, 500), (300, 73, 500),
            (300, 200, 1003), (2000, 72, 1003)]  # fmt: skip


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", INFINITE, ids=lambda s: "x".join(map(str, s)))
def test_infinities_and_nan_in_rows_that_count(cuda, shape, dtype):
    """What is not finite stays so, and in its own row: losses and log-sum-exp as defined, other rows bit for bit, gradients not finite where the definition's are not."""
    x, w, targets = operands(cuda, *shape, dtype, seed=7)
    clean = linear_cross_entropy(x, w, targets, reduction="none")
    for bad in ((float("inf"),), (float("-inf"),), (float("nan"),), (float("inf"), float("inf")), (float("inf"), float("-inf"))):
        y = x.clone()
        y[0, 3 : 3 + len(bad)] = torch.tensor(bad, device=cuda, dtype=dtype)
        loss, lse = linear_cross_entropy(y, w, targets, reduction="none")
        want = defined(y, w, targets)
        check_infinities(loss, want[0], "loss"), check_infinities(lse, want[1], "lse")
        assert not bool(torch.isfinite(lse[0])) and torch.equal(loss[1:], clean[0][1:]) and torch.equal(lse[1:], clean[1][1:])
        assert not bool(torch.isfinite(linear_cross_entropy(y, w, targets)[0]))
        d_x, d_w = linear_cross_entropy_backward(None, y, w, targets, lse, reduction="none")
        check_finite(d_x, want[2], "d_x"), check_finite(d_w, want[3], "d_weight")
    device_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", INFINITE, ids=lambda s: "x".join(map(str, s)))
def test_infinities_in_the_weights(cuda, shape, dtype):
    """A class that is minus infinity takes no part, and costs infinitely much where it is the target; one that is infinity takes all."""
    x, w, targets = operands(cuda, *shape, dtype, seed=8)
    x = x.abs() + 0.125
    targets[targets == 5] = 6
    w[5] = float("-inf")
    loss, lse = linear_cross_entropy(x, w, targets, reduction="none")
    check_forward(x, torch.cat((w[:5], w[6:])), torch.where(targets > 5, targets - 1, targets), "none", loss, lse)
    for change in (("target", 5, None), ("infinity", 7, float("inf")), ("nan", 9, float("nan"))):
        ids, v = targets.clone(), w.clone()
        if change[0] == "target":
            ids[0] = change[1]
        else:
            v[change[1]] = change[2]
        loss, lse = linear_cross_entropy(x, v, ids, reduction="none")
        want = defined(x, v, ids)
        check_infinities(loss, want[0], "loss"), check_infinities(lse, want[1], "lse")
        d_x, d_w = linear_cross_entropy_backward(None, x, v, ids, lse, reduction="none")
        check_finite(d_x, want[2], "d_x"), check_finite(d_w, want[3], "d_weight")
    device_status()


@pytest.mark.parametrize("shape", INFINITE, ids=lambda s: "x".join(map(str, s)))
def test_the_largest_values(cuda, shape):
    """float32 values between bfloat16's largest and float32's."""
    x, w, targets = operands(cuda, *shape, torch.float32, seed=9)
    x[0, 3], x[-1, 4] = 3.402e38, -3.4e38
    w[:, 3:5] *= 2.0**-20
    loss, lse = linear_cross_entropy(x, w, targets, reduction="none")
    check_forward(x, w, targets, "none", loss, lse)
    w[3, 2], w[4, 2] = 3.4e38, -3.4e38  # logits of both signs that are as large
    x[:, 2] *= 2.0**-20
    loss, lse = linear_cross_entropy(x, w, targets, reduction="none")
    check_forward(x, w, targets, "none", loss, lse)


@pytest.mark.parametrize("shape", INFINITE, ids=lambda s: "x".join(map(str, s)))
def test_gradients_by_the_largest_values(cuda, shape):
    """Logits without them: a float32 logit of 1e32 is 1e25 apart from the next, and its exponential nothing."""
    x, w, targets = operands(cuda, *shape, torch.float32, seed=10)
    x[0, 3], x[-1, 4] = 3.402e38, -3.4e38
    w[:, 3:5] = 0.0
    loss, lse = linear_cross_entropy(x, w, targets, reduction="none")
    check_forward(x, w, targets, "none", loss, lse)
    check_backward(x, w, targets, lse, "none", None, *linear_cross_entropy_backward(None, x, w, targets, lse, reduction="none"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", INFINITE, ids=lambda s: "x".join(map(str, s)))
def test_logits_far_from_zero(cuda, shape, dtype):
    """Multiples of 2^20 and more, all exact: the largest logit is the log-sum-exp, a row's probability is its largest logit's, and every result is a sum of a few exact values."""
    t, d, v = shape
    g = torch.Generator(device=cuda).manual_seed(11)
    x = (torch.randint(-8, 9, (t, d), generator=g, device=cuda) * 2.0**8).to(dtype)
    w = (torch.randint(-8, 9, (v, d), generator=g, device=cuda) * 2.0 ** (12 if dtype == torch.float16 else 30)).to(dtype)
    targets = torch.randint(0, v, (t,), generator=g, device=cuda)
    z = x.double() @ w.double().t()
    top = z.amax(-1)
    loss, lse = linear_cross_entropy(x, w, targets, reduction="none")
    assert torch.equal(lse.double(), top) and torch.equal(loss.double(), top - z.gather(-1, targets[:, None])[:, 0])
    dz = (z == top[:, None]).double() - torch.nn.functional.one_hot(targets, v)
    d_x, d_w = linear_cross_entropy_backward(None, x, w, targets, lse, reduction="none")
    assert torch.equal(d_x, (dz @ w.double()).to(dtype)) and torch.equal(d_w, (dz.t() @ x.double()).to(dtype))
    device_status()


@pytest.mark.parametrize("shape", [(22199, 17072, 5915), (31585, 12424, 4715)])
def test_a_last_piece_whose_units_the_table_does_not_hold(cuda, shape):
    """Both products of a whole piece share a launch; of a few classes behind it, whose shares are less even, they have one each."""
    t, d, v = shape
    x, w, targets = operands(cuda, t, d, v, torch.bfloat16, ignored=0.1)
    targets[0], targets[1] = v - 1, v - 2
    _, lse = linear_cross_entropy(x, w, targets, reduction="none")
    d_x, d_w = linear_cross_entropy_backward(None, x, w, targets, lse, reduction="none")
    counts = (targets != IGNORED)[:, None]
    for rows in (slice(0, 150), slice(t - 150, t)):  # a gradient's every term is a rounded dz times an element
        dz = (torch.exp(x[rows].double() @ w.double().t() - lse[rows].double()[:, None]) - torch.nn.functional.one_hot(targets[rows].clamp(min=0), v)) * counts[rows]
        within(d_x[rows], dz @ w.double(), 2 * half(torch.bfloat16) * (dz.abs() @ w.double().abs()) + 1e-6, "d_x")
    for classes in (slice(0, 100), slice(v - 100, v)):
        ids = torch.arange(v, device=cuda)[classes]
        dz = (torch.exp(x.double() @ w[classes].double().t() - lse.double()[:, None]) - (targets[:, None] == ids).double()) * counts
        within(d_w[classes], dz.t() @ x.double(), 2 * half(torch.bfloat16) * (dz.t().abs() @ x.double().abs()) + 1e-6, "d_weight")
    device_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(4, 516, 140001), (5, 516, 140001), (61, 514, 140001), (100, 516, 140001), (300, 524, 270001)], ids=lambda s: "x".join(map(str, s)))
def test_a_gradient_that_no_tiles_store_in_several_pieces(cuda, shape, dtype):
    x, w, targets = operands(cuda, *shape, dtype, ignored=0.2 * (shape[0] % 2))
    targets[0], targets[1] = shape[2] - 1, 0
    loss, lse = linear_cross_entropy(x, w, targets)
    check_forward(x, w, targets, "mean", loss, lse)
    check_backward(x, w, targets, lse, "mean", None, *linear_cross_entropy_backward(None, x, w, targets, lse))
    device_status()
