"""The AdamW step over lists of tensors against the formula in 64 bits, its moments bit for bit against the same products and sums in float32: every
type of weights, gradients and moments, sizes around blocks and chunks, memory that vectors do not fit, clipping, scalars on the device, and what
stands in tensors that hold no numbers."""

import math

import numpy as np
import pytest
import torch

from lumen_b200 import device as D
from lumen_b200.runtime import adamw_state, adamw_step, clip_grad_norm, device_status, grad_norm

pytestmark = pytest.mark.gpu

BETAS, EPS = (0.9, 0.999), 1e-8


def half(dtype):
    return torch.finfo(dtype).eps / 2 * (1 + 2.0**-8)


def e4m3(codes):
    return codes.view(torch.float8_e4m3fn).float()


def blocks(x):
    """`x` flat, in rows of 256 with zeros behind its end."""
    x = x.reshape(-1)
    return torch.cat((x, x.new_zeros(-x.numel() % 256))).view(-1, 256)


def held(x, lowest):
    """Codes and scales of float32 `x` as the operator's description says, in float32, each operation rounded."""
    rows = blocks(x)
    most = rows.abs().amax(-1, keepdim=True)
    top = torch.full_like(most, 448.0)
    q = rows * torch.where(most < 2.0**-100, torch.zeros_like(most), torch.div(top, most))
    q = q.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float()
    if lowest:
        q = torch.where((q == 0) & (rows > 0), 2.0**-9, q)
    scale = torch.where(most < 2.0**-100, torch.zeros_like(most), torch.div(most, top))
    return q.to(torch.float8_e4m3fn).view(torch.uint8).view(-1)[: x.numel()], scale.view(-1)


def rounds_to(codes, scale, x, off, lowest, what):
    """Whether codes and scales hold `x` (64 bits, known up to `off`): the scale is the block's largest value over 448, with three roundings, and each code the
    nearest e4m3 value to x / scale, up to what x is off by and as many roundings."""
    rows, off = blocks(x), blocks(off)
    most = rows.abs().amax(-1)
    assert bool(((scale.double() - most / 448).abs() <= off.amax(-1) / 448 + 2.0**-21 * most / 448 + 1e-30).all()), f"{what}: scales"
    unit = scale.double()[:, None].clamp(min=1e-300)
    q, want = e4m3(blocks(codes)).double(), rows / unit
    _, exponent = torch.frexp(want)
    half_step = torch.exp2((exponent - 5).clamp(min=-10).double())  # what lies between two powers of two is a sixteenth of the lower one from its neighbours' middle
    near = (q - want).abs() <= half_step + off / unit + 2.0**-20 * want.abs()
    if lowest:
        near |= (q == 2.0**-9) & (want < 2.0**-9) & (rows > 0)
        assert bool((q > 0)[rows > 1e-18].all()), f"{what}: something became zero"
    near |= (scale == 0)[:, None] & (q == 0)
    assert bool(near.view(-1)[: x.numel()].all()) and not bool(q.view(-1)[x.numel() :].any()), f"{what}: codes"


def values(codes, scale):
    return (e4m3(blocks(codes)) * scale[:, None]).view(-1)[: codes.numel()]


class Model:
    """A list of tensors with their moments, and copies of all of it from before a step."""

    def __init__(self, cuda, sizes, dtypes, bits=32, grads=None, masters=False, seed=0, begun=True, offset=0):
        g = torch.Generator(device=cuda).manual_seed(seed)

        def normal(n, scale=1.0):
            return torch.randn(n + offset, generator=g, device=cuda)[offset:] * scale

        def moved(x, dtype):  # memory `offset` elements off an aligned place
            out = torch.empty(x.numel() + offset, dtype=dtype, device=cuda)[offset:]
            return out.copy_(x)

        self.bits = bits
        self.params, self.grads, self.m, self.v, self.masters = [], [], [], [], [] if masters else None
        self.ms, self.vs = ([], []) if bits == 8 else (None, None)
        for k, n in enumerate(sizes):
            dtype = dtypes[k % len(dtypes)]
            rms = 10.0 ** float(-1 - k % 4) * torch.exp(normal(n))
            w = normal(n, 0.05)
            self.params.append(moved(w, dtype))
            self.grads.append(moved(rms * normal(n), grads or dtype))
            if masters:
                self.masters.append(moved(w, torch.float32) if dtype != torch.float32 else None)
            m, v = (0.3 * rms * normal(n), rms.square() * torch.rand(n, generator=g, device=cuda)) if begun else (torch.zeros(n, device=cuda), torch.zeros(n, device=cuda))
            if bits == 8:
                for x, codes, scales, lowest in ((m, self.m, self.ms, False), (torch.sqrt(v), self.v, self.vs, True)):
                    c, s = held(x, lowest)
                    codes.append(moved(c, torch.uint8)), scales.append(s)
            else:
                self.m.append(moved(m, torch.float32)), self.v.append(moved(v, torch.float32))
        self.before = [[None if t is None else t.clone() for t in ts] if ts is not None else None for ts in (self.params, self.grads, self.m, self.v, self.ms, self.vs, self.masters)]

    def step(self, step, **more):
        adamw_step(self.params, self.grads, self.m, self.v, step, betas=BETAS, eps=EPS, exp_avg_scale=self.ms, exp_avg_sq_scale=self.vs, masters=self.masters, **more)

    def everything(self):
        return [t for ts in (self.params, self.grads, self.m, self.v, self.ms or [], self.vs or [], self.masters or []) for t in ts if t is not None]

    def check(self, step, lr=1e-3, weight_decay=1e-2, factor=None):
        b1, b2 = BETAS
        params, grads, ms, vs, mss, vss, masters = self.before
        for k, p in enumerate(params):
            assert torch.equal(self.grads[k], grads[k])
            g = grads[k].float()
            if factor is not None:
                g = g * factor
            m, v = (values(ms[k], mss[k]), values(vs[k], vss[k]).square()) if self.bits == 8 else (ms[k], vs[k])
            m32, v32 = m * b1 + g * (1 - b1), v * b2 + g * g * (1 - b2)
            for got, scale, want, lowest in ((self.m[k], self.ms and self.ms[k], m32, False), (self.v[k], self.vs and self.vs[k], v32, True)):
                if self.bits == 32:
                    assert torch.equal(got, want), f"tensor {k}: a moment"
                    continue
                # roots and products of a few roundings each, 2^-21 of what is added up
                size = (m.double() * b1).abs() + (g.double() * (1 - b1)).abs()
                exact = torch.sqrt(v.double() * b2 + g.double() ** 2 * (1 - b2)) if lowest else m.double() * b1 + g.double() * (1 - b1)
                rounds_to(got, scale, exact, 2.0**-21 * (exact if lowest else size), lowest, f"tensor {k}")
            m64, v64 = m.double() * b1 + g.double() * (1 - b1), v.double() * b2 + g.double() ** 2 * (1 - b2)
            c1, c2 = 1 / (1 - b1**step), 1 / (1 - b2**step)
            start = masters[k] if masters and masters[k] is not None else p
            den = torch.sqrt(v64 * c2) + EPS
            up = lr * m64 * c1 / den
            want = start.double() * (1 - lr * weight_decay) - up
            # two products and a sum round m and v (betas in float32 too), the root and the quotient a few times more
            tol = 2.0**-20 * up.abs() + lr * c1 * 2.0**-21 * (m.double().abs() * b1 + g.double().abs() * (1 - b1)) / den + 2.0**-22 * (want.abs() + start.double().abs())
            if masters and masters[k] is not None:
                assert bool(((self.masters[k].double() - want).abs() <= tol).all())
                assert torch.equal(self.params[k], self.masters[k].to(p.dtype))
            else:
                tiny = 2.0**-25 if p.dtype == torch.float16 else 0.0
                assert bool(((self.params[k].double() - want).abs() <= tol + half(p.dtype) * (want.abs() + tol) * (p.dtype != torch.float32) + tiny).all()), f"tensor {k}: weights"


SIZES = [1, 7, 255, 256, 257, 4095, 4096, 4097, 8192, 8200, 70001, 300000]
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grads", [None, torch.float32], ids=["alike", "float32"])
@pytest.mark.parametrize("masters", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_a_step(cuda, dtype, masters, grads, bits):
    model = Model(cuda, SIZES, [dtype], bits, grads, masters)
    model.step(3)
    device_status()
    model.check(3)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [1, 2, 4, 8])
def test_memory_off_the_vectors(cuda, offset, bits):
    model = Model(cuda, [5, 300, 5000, 20001], TYPES, bits, offset=offset)
    model.step(11, lr=0.01, weight_decay=0.1)
    model.check(11, 0.01, 0.1)


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_of_a_model_at_odd_places_of_one_arena(cuda, bits):
    """Views one behind the other: what lies around each stays as it is."""
    sizes = [3, 1000, 257, 0, 8191, 12]
    model = Model(cuda, sizes, [torch.bfloat16], bits)
    arenas = {}
    for name, ts in (("params", model.params), ("grads", model.grads), ("m", model.m), ("v", model.v)):
        arena = torch.full((sum(sizes) + 2 * len(sizes) + 1,), 7, dtype=ts[0].dtype, device=cuda)
        at = 1
        for k, n in enumerate(sizes):
            ts[k] = arena[at : at + n].copy_(ts[k])
            at += n + 2
        arenas[name] = arena
    model.step(5)
    model.check(5)
    for arena in arenas.values():
        at = 1
        for n in sizes:
            assert bool((arena[at - 1] == 7).all()) and bool((arena[at + n] == 7).all())
            at += n + 2


@pytest.mark.parametrize("bits", [32, 8])
def test_the_first_step_and_the_ones_behind_it(cuda, bits):
    model = Model(cuda, [70000, 33, 1 << 20], TYPES, bits, begun=False)
    model.m, model.v, model.ms, model.vs = adamw_state(model.params, bits)
    assert [t.dtype for t in model.m] == [torch.uint8 if bits == 8 else torch.float32] * 3 and (model.ms is None) == (bits == 32)
    for step in (1, 2, 3):
        model.before = [[t.clone() for t in ts] if ts is not None else None for ts in (model.params, model.grads, model.m, model.v, model.ms, model.vs, model.masters)]
        model.step(step)
        model.check(step)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("share", [0.25, 3.0])
def test_clipping_on_the_way(cuda, share, bits):
    model = Model(cuda, [70000, 33, 4096, 9000], TYPES, bits, grads=torch.float32)
    norm = grad_norm(model.grads)
    most = share * float(norm)
    model.step(7, norm=norm, max_norm=most)
    factor = min(1.0, most / (float(norm) + 1e-6))
    model.check(7, factor=float(np.float32(factor)))
    if bits == 8:
        return
    other = Model(cuda, [70000, 33, 4096, 9000], TYPES, bits, grads=torch.float32)
    clip_grad_norm(other.grads, most)
    other.step(7)
    # the norm that clips in memory has 64 bits, the one that is handed on 24: factors differ by 2^-24 of them for that and 2^-24 for their own roundings, gradients
    # by two roundings more, and the products and the sum of a moment are rounded in both
    for k, (a, b) in enumerate(zip(model.m, other.m)):
        size = 0.9 * model.before[2][k].abs() + 0.1 * other.grads[k].abs()
        assert bool(((a.double() - b.double()).abs() <= 2.0**-21 * size.double()).all())


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
def test_scalars_on_the_device(cuda, kind):
    a, b = (Model(cuda, [5000, 300], TYPES) for _ in range(2))
    a.step(12, lr=0.02)
    b.step(torch.full((), 12, dtype=kind, device=cuda), lr=torch.full((1,), 0.02, device=cuda))
    assert all(torch.equal(x, y) for x, y in zip(a.m + a.v, b.m + b.v))
    # 0.02 is a float32 on the device, a float64 on the host
    assert all(float((x.double() - y.double()).abs().max()) <= 2.0**-7 * float(x.double().abs().max()) * half(x.dtype) * 256 for x, y in zip(a.params, b.params))
    b.check(12, lr=float(np.float32(0.02)))


@pytest.mark.parametrize("bits", [32, 8])
def test_replays_of_a_captured_step(cuda, bits):
    sizes = [70000, 33, 4096]
    eager, graphed = (Model(cuda, sizes, TYPES, bits) for _ in range(2))
    step, lr = torch.ones((), dtype=torch.int64, device=cuda), torch.full((), 1e-3, device=cuda)
    norm = torch.ones((), device=cuda)
    alive = graphed.params[0].clone().requires_grad_()
    kept = (alive * alive).sum()  # an eager graph beside the captured one
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        graphed.step(step, lr=lr, norm=norm, max_norm=0.5)
    assert all(torch.equal(a, b) for a, b in zip(graphed.everything(), eager.everything()))  # capturing runs nothing
    for k in range(1, 4):
        step.fill_(k), lr.fill_(1e-3 / k), norm.fill_(0.3 * k)
        graph.replay()
        eager.step(k, lr=float(np.float32(1e-3 / k)), norm=norm, max_norm=0.5)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(graphed.everything(), eager.everything()))
    kept.backward()


def test_two_streams_and_two_calls_at_once(cuda):
    models = [Model(cuda, [300000, 33, 4096], TYPES, bits, seed=3) for bits in (32, 8, 32, 8)]
    for m in models[:2]:
        m.step(2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    models[2].step(2, stream=side.cuda_stream)
    models[3].step(2)
    torch.cuda.synchronize()
    for a, b in zip(models[:2], models[2:]):
        assert all(torch.equal(x, y) for x, y in zip(a.everything(), b.everything()))


def test_more_tensors_than_a_launch_takes(cuda):
    for bits in (32, 8):
        model = Model(cuda, [1 + 37 * (k % 50) for k in range(700)], TYPES, bits)
        model.step(4)
        model.check(4)


@pytest.mark.parametrize("bits", [32, 8])
def test_offsets_past_32_bits(cuda, bits):
    """A parameter of more than 2^31 elements moves as its end does by itself."""
    n, end = (1 << 31) + 1000, 1000 + 256 * 40
    p, g = torch.zeros(n, dtype=torch.bfloat16, device=cuda), torch.zeros(n, dtype=torch.bfloat16, device=cuda)
    p[-end:] = torch.randn(end, device=cuda).to(torch.bfloat16)
    g[-end:] = torch.randn(end, device=cuda).to(torch.bfloat16)
    small, grad = p[-end:].clone(), g[-end:].clone()
    for params, grads in (([p], [g]), ([small], [grad])):
        m, v, ms, vs = adamw_state(params, bits)
        adamw_step(params, grads, m, v, 1, exp_avg_scale=ms, exp_avg_sq_scale=vs)
        if params[0] is p:
            kept = m[0][-end:].clone(), v[0][-end:].clone()
            assert not p[: 1 << 20].any()
            del m, v, ms, vs
    assert torch.equal(p[-end:], small) and torch.equal(kept[0], m[0]) and torch.equal(kept[1], v[0])


def test_shapes_strides_and_what_autograd_knows(cuda):
    p = torch.randn(40, 24, device=cuda).to(torch.bfloat16).t().requires_grad_()
    g = torch.randn_like(p.detach())
    m, v, _, _ = adamw_state([p])
    assert m[0].stride() == p.stride() and g.stride() == p.stride() and not m[0].requires_grad
    flat = [p.detach().t().clone().reshape(-1), g.t().reshape(-1)]
    fm, fv, _, _ = adamw_state(flat[:1])
    (p * p).sum().backward()
    kept = (p * p).sum()
    before = p._version
    adamw_step([p], [g], m, v, 1)
    adamw_step(flat[:1], flat[1:], fm, fv, 1)
    assert p._version > before and torch.equal(p.detach().t().reshape(-1), flat[0]) and torch.equal(m[0].t().reshape(-1), fm[0])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()
    # the same gradient for two parameters
    a, b = torch.ones(300, device=cuda), torch.ones(300, device=cuda)
    m, v, _, _ = adamw_state([a, b])
    adamw_step([a, b], [g.reshape(-1)[:300].float()] * 2, m, v, 1)
    assert torch.equal(a, b) and not torch.equal(a, torch.ones_like(a))
    adamw_step([], [], [], [], 1)


@pytest.mark.parametrize("bits", [32, 8])
def test_zeros_infinities_and_nan(cuda, bits):
    n = 1024
    p, g = torch.ones(n, device=cuda), torch.zeros(n, device=cuda)
    state = adamw_state([p], bits)

    def step(k):
        adamw_step([p], [g], state[0], state[1], k, weight_decay=0.0, exp_avg_scale=state[2], exp_avg_sq_scale=state[3])

    step(1)
    assert bool((p == 1).all()) and not any(t.any() for ts in state if ts for t in ts)  # zeros stay zeros
    g[300], g[600], g[601] = 1.0, 1e-15, 1e10
    step(2)
    assert float(p[300]) < 1 and bool((p[:256] == 1).all()) and bool(torch.isfinite(p).all())
    if bits == 8:
        # what is not zero keeps a denominator that is not zero
        assert state[1][0][300] == 0x7E and state[1][0][600] == 1 and state[1][0][602] == 0
    g[:] = 0.5
    g[10], g[900] = float("nan"), float("inf")
    step(3)
    assert bool(torch.isnan(p[10])) and bool(torch.isfinite(p[256:768]).all())
    if bits == 8:  # a block's scale is its largest value's
        assert bool(torch.isnan(state[2][0][0])) and bool(torch.isfinite(state[2][0][1:3]).all()) and not bool(torch.isfinite(state[2][0][3]))


def test_on_the_packages_own_tensors(cuda):
    for bits in (32, 8):
        model = Model(cuda, [5000], [torch.float32], bits, begun=False)
        region = D.Region(32 << 20)
        own = []
        for t in (model.params[0], model.grads[0]):
            own.append(region.empty(tuple(t.shape), "float32"))
            own[-1].copy_from_host(t.cpu().numpy())
        state = adamw_state(own[:1], bits)
        D.synchronize()
        for k in (1, 2):
            model.step(k)
            adamw_step(own[:1], own[1:], state[0], state[1], k, betas=BETAS, eps=EPS, exp_avg_scale=state[2], exp_avg_sq_scale=state[3], stream=0)
        D.synchronize()
        np.testing.assert_array_equal(own[0].numpy(), model.params[0].cpu().numpy())
        np.testing.assert_array_equal(state[1][0].numpy(), model.v[0].cpu().numpy())


def test_moments_in_8_bits_follow_those_in_32(cuda):
    """Over many steps of normal gradients the update in 8 bits stays near the one in 32: the mean of the denominators' ratio is within a tenth of one, and
    its spread within a third, as the kernel's description of its roundings says."""
    n = 1 << 16
    g = torch.Generator(device=cuda).manual_seed(0)
    rms = 1e-3 * torch.exp(torch.randn(n, generator=g, device=cuda))
    wide, narrow = torch.zeros(n, device=cuda), torch.zeros(n, device=cuda)
    a, b = adamw_state([wide], 32), adamw_state([narrow], 8)
    for k in range(1, 601):
        grad = [rms * torch.randn(n, generator=g, device=cuda)]
        adamw_step([wide], grad, a[0], a[1], k, betas=(0.9, 0.99))
        adamw_step([narrow], grad, b[0], b[1], k, betas=(0.9, 0.99), exp_avg_scale=b[2], exp_avg_sq_scale=b[3])
    ratio = values(b[1][0], b[3][0]) / torch.sqrt(a[1][0])
    assert abs(float(ratio.mean()) - 1) < 0.1 and float(ratio.std()) < 1 / 3 and math.isfinite(float(narrow.sum()))
