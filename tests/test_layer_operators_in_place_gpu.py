"""Results that a caller's tensors take: autograd knows that they have changed."""

import pytest
import torch

from lumen_b200.runtime import clip_grad_norm, grad_norm, qk_norm_rope, qk_norm_rope_backward

pytestmark = pytest.mark.gpu


def kept(x):
    """A tensor and a value whose backward pass reads it."""
    y = x * 1.0
    return y, (y * y).sum()


def test_a_backward_pass_that_kept_a_changed_tensor_says_so(cuda):
    g = torch.Generator(device=cuda).manual_seed(0)
    x = torch.randn(2, 5, 3, 64, generator=g, device=cuda).requires_grad_()
    cos, sin = torch.ones(5, 32, device=cuda), torch.zeros(5, 32, device=cuda)

    def changed(call):
        q, a = kept(x)
        k, b = kept(x)
        call(q, k)
        for value in (a, b):
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                value.backward()

    changed(lambda q, k: qk_norm_rope(q, k, cos, sin, out=(q, k)))
    changed(lambda q, k: qk_norm_rope(x.detach(), x.detach(), cos, sin, out=(q, k)))
    changed(lambda q, k: qk_norm_rope_backward(q, k, x.detach(), x.detach(), cos, sin, out=(q, k)))
    changed(lambda q, k: clip_grad_norm([q, k], 0.1))
    changed(lambda q, k: clip_grad_norm([x.detach(), x.detach()], 0.1, out=[q, k]))


def test_tensors_that_are_only_read_stay_as_they_are(cuda):
    x = torch.ones(2, 5, 3, 64, device=cuda).requires_grad_()
    cos, sin = torch.ones(5, 32, device=cuda), torch.zeros(5, 32, device=cuda)
    q, value = kept(x)
    qk_norm_rope(q, q, cos, sin)
    qk_norm_rope_backward(q, q, q, q, cos, sin)
    grad_norm([q])
    clip_grad_norm([q], 0.1, out=[torch.empty_like(q)])
    value.backward()
    assert torch.equal(x.grad, 2 * x.detach())


def test_in_inference_mode(cuda):
    """Its tensors keep no count of changes."""
    with torch.inference_mode():
        x = torch.ones(2, 5, 3, 64, device=cuda)
        y = x.clone()
        cos, sin = torch.ones(5, 32, device=cuda), torch.zeros(5, 32, device=cuda)
        want = qk_norm_rope(x, x, cos, sin)
        got = qk_norm_rope(x, y, cos, sin, out=(x, y))
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[0] is x
        clip_grad_norm([x, y], 0.5)
        assert abs(float(grad_norm([x, y])) - 0.5) < 1e-4


def test_any_collection_of_tensors(cuda):
    """A dictionary's values, a generator, the rows of a matrix: as a list of them."""
    g = torch.Generator(device=cuda).manual_seed(1)
    x = [torch.randn(n, generator=g, device=cuda) for n in (5, 300, 7)]
    want = [t.clone() for t in x]
    norm = clip_grad_norm(want, 1.0)
    for wrap in (lambda ts: dict(enumerate(ts)).values(), lambda ts: (t for t in ts), tuple):
        got, out = [t.clone() for t in x], [torch.empty_like(t) for t in x]
        assert torch.equal(grad_norm(wrap(got)), norm)
        assert torch.equal(clip_grad_norm(wrap(got), 1.0, out=wrap(out)), norm) and all(torch.equal(a, b) for a, b in zip(out, want))
        assert torch.equal(clip_grad_norm(wrap(got), 1.0, like=x[0]), norm) and all(torch.equal(a, b) for a, b in zip(got, want))
    rows = torch.randn(4, 6, generator=g, device=cuda)
    flat = rows.clone()
    clip_grad_norm([flat], 0.5)
    clip_grad_norm(rows, 0.5)
    assert torch.allclose(rows, flat, rtol=1e-6, atol=0.0)  # sums of other groups
    q = torch.randn(1, 3, 2, 64, generator=g, device=cuda)
    cos, sin = torch.ones(3, 32, device=cuda), torch.zeros(3, 32, device=cuda)
    want = qk_norm_rope(q, q, cos, sin)
    got = qk_norm_rope(q, q, cos, sin, out=(torch.empty_like(q) for _ in range(2)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
