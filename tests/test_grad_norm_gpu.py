"""The global gradient norm and clipping by it against sums in 64 bits: types and layouts in any mix, sizes around a vector and a chunk, more tensors
than a launch takes, values at the ends of float32, in place and not."""

import math

import numpy as np
import pytest
import torch

from lumen_b200 import device as D
from lumen_b200.runtime import clip_grad_norm, device_status, grad_norm

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float32, torch.float16]


def norm64(tensors):
    return math.sqrt(sum(float(t.double().square().sum()) for t in tensors))


def check_norm(got, want):
    """Groups of eight squares in float32 (9 roundings of 2^-24, halved by the root), sums in 64 bits, one rounding to float32."""
    assert got.dtype == torch.float32 and got.shape == ()
    assert abs(float(got) - want) <= 6 * 2.0**-24 * want, (float(got), want)


def check_scaled(got, x, factor):
    """One rounding of the factor and one of the product in float32, one to the tensor's type (or half a step of its subnormals)."""
    want = x.double() * factor
    tiny = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134, torch.float32: 2.0**-150}[x.dtype]
    tol = (torch.finfo(x.dtype).eps / 2 * (1 + 2.0**-8) + 8 * 2.0**-24) * want.abs() + tiny
    assert bool(((got.double() - want).abs() <= tol).all())


def tensors(cuda, sizes, seed=0, dtypes=TYPES, scale=1.0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return [(torch.randn(n, generator=g, device=cuda) * scale).to(dtypes[k % len(dtypes)]) for k, n in enumerate(sizes)]


def factor_of(total, most):
    return min(1.0, most / (total + 1e-6))


SIZES = [
    [1], [7], [8], [0], [0, 5, 0], [3, 4, 5, 15, 16, 17, 31],
    [4095, 4096, 4097, 8191, 8192, 8193], [100001, 1, 65536, 333],
    [3000001], list(range(0, 300)), [2] * 241, [1000] * 480 + [0, 1],
]  # fmt: skip


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("dtypes", [TYPES, TYPES[:1], TYPES[1:2]], ids=["mixed", "bf16", "f32"])
def test_norm_and_clipping(cuda, sizes, dtypes):
    xs = tensors(cuda, sizes, dtypes=dtypes)
    total = norm64(xs)
    check_norm(grad_norm(xs), total)
    for share in (0.3, 2.0):
        most = share * total
        outs = [torch.full_like(x, 7.0) for x in xs]
        check_norm(clip_grad_norm(xs, most, out=outs), total)
        for x, out in zip(xs, outs):
            check_scaled(out, x, factor_of(total, most))
            if share > 1:
                assert torch.equal(x, out)
        place = [x.clone() for x in xs]
        check_norm(clip_grad_norm(place, most), total)
        assert all(torch.equal(a, b) for a, b in zip(place, outs))
    device_status()


def test_layouts_and_alignments(cuda):
    """Transposed and permuted dense tensors, views that begin anywhere, operand and result aligned differently; what lies around a view stays."""
    base = tensors(cuda, [5000, 5000, 5000], seed=1)
    xs = []
    for x in base:
        xs += [x[1 : 1 + 63].view(9, 7).t(), x[100 : 100 + 120].view(4, 5, 6).permute(2, 0, 1), x[303:1304], x[1400:1400]]
    total = norm64(xs)
    check_norm(grad_norm(xs), total)
    rooms = [torch.full((5000,), 7.0, dtype=x.dtype, device=cuda) for x in base]
    outs = []
    for r in rooms:
        outs += [r[2 : 2 + 63].view(9, 7).t(), r[100 : 100 + 120].view(4, 5, 6).permute(2, 0, 1), r[310:1311], r[1400:1400]]
    clip_grad_norm(xs, 0.5 * total, out=outs)
    for x, out in zip(xs, outs):
        check_scaled(out, x, factor_of(total, 0.5 * total))
    for r in rooms:
        assert bool((r[:2] == 7).all() and (r[65:100] == 7).all() and (r[220:310] == 7).all() and (r[1311:] == 7).all())
    before = [x.clone() for x in base]
    clip_grad_norm(xs, 0.5 * total)
    for a, b in zip(base, before):
        assert torch.equal(a[:1], b[:1]) and torch.equal(a[64:100], b[64:100]) and torch.equal(a[220:303], b[220:303]) and torch.equal(a[1304:], b[1304:])
    for x, out in zip(xs, outs):
        assert torch.equal(x, out)


@pytest.mark.parametrize("value", [3e38, 1e25, 1e-25, 1e-38, 1e-42])
def test_values_whose_squares_leave_float32(cuda, value):
    xs = [torch.full((1000,), value, device=cuda), torch.tensor([value], device=cuda)]
    if value < 1e30:
        xs.append(torch.full((33,), value, device=cuda).to(torch.bfloat16))
    total = norm64(xs)
    if total < 3.4e38:
        got = float(grad_norm(xs))
        assert abs(got - total) <= 6 * 2.0**-24 * total + 2.0**-149
    else:
        assert math.isinf(float(grad_norm(xs)))
    outs = [torch.empty_like(x) for x in xs]
    clip_grad_norm(xs, 1.0, out=outs)
    for x, out in zip(xs, outs):
        check_scaled(out, x, factor_of(total, 1.0))


def test_infinite_and_nan_norms(cuda):
    for bad in (float("inf"), float("nan")):
        xs = tensors(cuda, [100, 200], seed=3)
        xs[1][7] = bad
        norm = grad_norm(xs)
        assert math.isinf(float(norm)) if math.isinf(bad) else math.isnan(float(norm))
        clip_grad_norm(xs, 1.0)
        if math.isinf(bad):
            assert bool((xs[0] == 0).all()) and bool(xs[1][7].isnan()) and int(xs[1].isnan().sum()) == 1
        else:
            assert bool(xs[0].isnan().all()) and bool(xs[1].isnan().all())


def test_bounds_of_zero_and_a_zero_norm(cuda):
    xs = tensors(cuda, [50, 60])
    clip_grad_norm(xs, 0.0)
    assert all(bool((x == 0).all()) for x in xs)
    assert float(clip_grad_norm(xs, 1.0)) == 0.0 and all(bool((x == 0).all()) for x in xs)


def test_no_tensors(cuda):
    assert float(grad_norm([], like=torch.empty(0, device=cuda))) == 0.0
    assert float(clip_grad_norm([], 1.0, like=torch.empty(0, device=cuda))) == 0.0
    with pytest.raises(ValueError, match="like"):
        grad_norm([])


def test_a_tensor_given_twice(cuda):
    x = tensors(cuda, [1000])[0]
    check_norm(grad_norm([x, x]), math.sqrt(2.0) * norm64([x]))
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm([x, x], 1.0)
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm([x, x[10:20]], 1.0)
    outs = [torch.empty_like(x), torch.empty_like(x)]
    clip_grad_norm([x, x], 1.0, out=outs)
    assert torch.equal(*outs)
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm([x[:500], x[500:]], 1.0, out=[x[500:], outs[0][:500]])


def test_repeats_bit_for_bit_on_any_stream_and_in_graphs(cuda):
    sets = [tensors(cuda, [300000, 17, 4096, 70001], seed=k) for k in range(2)]
    outs = [[torch.empty_like(x) for x in xs] for xs in sets]

    def call(k, **more):
        return clip_grad_norm(sets[k], 3.0, out=outs[k], **more)

    want = [(call(k).clone(), [o.clone() for o in outs[k]]) for k in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    norm = call(0, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(norm, want[0][0])
    graphs, norms = [], []
    for k in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norms.append(call(k))
        graphs.append(graph)
    for out in outs:
        for o in out:
            o.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for k in range(2):
        assert torch.equal(norms[k], want[k][0]) and all(torch.equal(a, b) for a, b in zip(outs[k], want[k][1]))


def test_a_tensor_on_another_gpu_is_refused(cuda):
    """A stand-in that says it lives on GPU 1 while GPU 0 is current: nothing is launched."""

    class Elsewhere:
        shape, dtype, is_cuda = (4,), "float32", True
        get_device = staticmethod(lambda: 1)
        data_ptr = staticmethod(lambda: 1 << 20)
        stride = staticmethod(lambda: (1,))

    x = torch.ones(4, device=cuda)
    for call in (lambda: clip_grad_norm([x, Elsewhere()], 1.0), lambda: clip_grad_norm([x], 1.0, out=[Elsewhere()]), lambda: grad_norm([x, Elsewhere()])):
        with pytest.raises(ValueError, match="a tensor is on GPU 1, the current one is GPU 0"):
            call()
    assert torch.equal(x, torch.ones_like(x))


def test_from_several_threads(cuda):
    """Two threads, each on a stream of its own, clip their own tensors at once."""
    import threading

    sets = [tensors(cuda, [70001, 333, 4096], seed=k) for k in range(2)]
    want = [float(grad_norm(xs)) for xs in sets]
    torch.cuda.synchronize()
    got = [None, None]

    def work(k):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got[k] = [float(clip_grad_norm(sets[k], 1e9)) for _ in range(50)]

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(set(g) == {w} for g, w in zip(got, want))


def test_on_the_packages_own_tensors(cuda):
    xs = tensors(cuda, [1000, 33], dtypes=[torch.float32])
    region = D.Region(32 << 20)
    own = []
    for x in xs:
        own.append(region.empty(tuple(x.shape), "float32"))
        own[-1].copy_from_host(x.cpu().numpy())
    want = clip_grad_norm(xs, 2.0)
    got = clip_grad_norm(own, 2.0, stream=0)
    D.synchronize()
    assert got.item() == float(want)
    for a, b in zip(own, xs):
        np.testing.assert_array_equal(a.numpy(), b.cpu().numpy())
