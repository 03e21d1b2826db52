"""Calls of a decoder layer's operators whose results lie in memory that the call also reads, or writes a second time, on stand-ins for tensors. No GPU: a call
that is in order gets as far as the library's error that there is none."""

import pytest
import torch

from lumen_b200 import _lib
from tests.test_host_path import Array

if torch.cuda.is_available():  # the calls that are in order would run, on stand-ins' memory
    pytest.skip("refusals are tested where nothing can run", allow_module_level=True)

ROOM = 1 << 24  # bytes between tensors that are apart


class At(Array):
    """A stand-in at byte `at`."""

    def __init__(self, at, shape, strides=None, dtype="bfloat16"):
        if strides is None:
            strides = [1] * len(shape)
            for d in range(len(shape) - 2, -1, -1):
                strides[d] = strides[d + 1] * max(shape[d + 1], 1)  # as torch counts them where there are no elements
        super().__init__(shape, dtype, strides)
        self.at = at

    def data_ptr(self):
        return (1 << 30) + self.at


def take(nbytes):
    return At(60 * ROOM, (nbytes,), dtype="uint8")


def refused(match):
    return pytest.raises(_lib.LumenError, match=match)


def in_order():
    return pytest.raises(_lib.LumenError, match="no usable CUDA device")


B, S, N, NK, H = 2, 5, 4, 2, 64
Q, K = (B, S, N, H), (B, S, NK, H)


def rope(**change):
    a = {"eps": 1e-6, "interleaved": False, "q": At(0, Q), "k": At(ROOM, K), "cos": At(2 * ROOM, (16, 32), dtype="float32"), "sin": At(3 * ROOM, (16, 32), dtype="float32"),
         "positions": At(4 * ROOM, (B, S), dtype="int64"), "wq": At(5 * ROOM, (H,)), "wk": At(6 * ROOM, (H,)), "q_out": At(7 * ROOM, Q), "k_out": At(8 * ROOM, K)}  # fmt: skip
    assert not change.keys() - a.keys()
    a.update(change)
    _lib.host().qk_norm_rope(*a.values(), 0)


def back(**change):
    a = {"eps": 1e-6, "interleaved": False, "dq_out": At(0, Q), "dk_out": At(ROOM, K), "q": At(2 * ROOM, Q), "k": At(3 * ROOM, K),
         "cos": At(4 * ROOM, (16, 32), dtype="float32"), "sin": At(5 * ROOM, (16, 32), dtype="float32"), "positions": None, "wq": At(6 * ROOM, (H,)),
         "wk": At(7 * ROOM, (H,)), "dq": At(8 * ROOM, Q), "dk": At(9 * ROOM, K), "dwq": At(10 * ROOM, (H,)), "dwk": At(11 * ROOM, (H,)), "take": take}  # fmt: skip
    assert not change.keys() - a.keys()
    a.update(change)
    _lib.host().qk_norm_rope_bwd(*a.values(), 0)


PACKED = [S * (N + 2 * NK) * H, (N + 2 * NK) * H, H, 1]
OUTER = [(N + NK) * S * H, H, S * H, 1]  # heads outermost
WIDE = [S * N * 2 * H, N * 2 * H, 2 * H, 1]  # rows of two heads


@pytest.mark.parametrize("change", [
    {},
    {"q_out": At(0, Q)},
    {"q_out": At(0, Q), "k_out": At(ROOM, K)},
    {"q": At(0, Q, PACKED), "k": At(2 * N * H, K, PACKED), "q_out": At(0, Q, PACKED), "k_out": At(2 * N * H, K, PACKED)},
    {"q_out": At(0, Q, OUTER), "k_out": At(2 * N * S * H, K, OUTER), "q": At(7 * ROOM, Q)},
    {"q": At(0, Q, WIDE), "q_out": At(2 * H, Q, WIDE)},  # the rows' other halves
    {"k": At(0, Q), "k_out": At(ROOM, Q), "q_out": At(8 * ROOM, Q)},  # keys that are the queries
    {"q_out": At(2 * B * S * N * H, Q)},  # right behind
    {"q": At(0, (0, S, N, H)), "k": At(0, (0, S, NK, H)), "q_out": At(0, (0, S, N, H)), "k_out": At(0, (0, S, NK, H)), "positions": None},
])  # fmt: skip
def test_rotation_in_order(change):
    if 0 in change.get("q", At(0, Q)).shape:
        rope(**change)  # nothing to do
        return
    with in_order():
        rope(**change)


@pytest.mark.parametrize("change, match", [
    ({"q_out": At(7 * ROOM, Q), "k_out": At(7 * ROOM, K)}, "keys' result shares GPU memory with the queries' result"),
    ({"k": At(ROOM, Q), "q_out": At(ROOM, Q), "k_out": At(0, Q)}, "queries' result shares GPU memory with the keys"),  # swapped
    ({"q_out": At(0, Q), "k": At(0, Q), "k_out": At(8 * ROOM, Q)}, "queries' result shares GPU memory with the keys"),  # in place, of keys that are the queries
    ({"q_out": At(16, Q)}, "queries' result shares GPU memory with the queries"),  # part of a row further
    ({"q_out": At(2 * H, Q)}, "queries' result shares GPU memory with the queries"),  # a head further
    ({"q_out": At(0, Q, [S * N * H, H, S * H, 1])}, "queries' result shares GPU memory with the queries"),  # other rows' places
    ({"q_out": At(2 * B * S * N * H - 2, Q)}, "queries' result shares GPU memory with the queries"),  # its last element
    ({"k_out": At(2 * H, K, PACKED), "q": At(0, Q, PACKED)}, "keys' result shares GPU memory with the queries"),
    ({"q_out": At(7 * ROOM, Q, [S * N * H, N * H, 16, 1])}, "elements of the queries' result share GPU memory"),
    ({"q_out": At(2 * ROOM + 64, Q)}, "shares GPU memory with cos"),
    ({"k_out": At(3 * ROOM - 2, K)}, "shares GPU memory with sin"),
    ({"k_out": At(4 * ROOM + 8, K)}, "shares GPU memory with positions"),
    ({"q_out": At(5 * ROOM, Q)}, "shares GPU memory with the queries' weight"),
    ({"q_out": At(6 * ROOM, Q)}, "shares GPU memory with the keys' weight"),
])  # fmt: skip
def test_rotation_refusals(change, match):
    with refused(match):
        rope(**change)


@pytest.mark.parametrize("change", [
    {},
    {"dq": At(0, Q), "dk": At(ROOM, K)},  # in the gradients' place
    {"dq": At(2 * ROOM, Q), "dk": At(3 * ROOM, K)},  # in the rows' place
    {"dq": At(8 * ROOM, Q, PACKED), "dk": At(8 * ROOM + 2 * N * H, K, PACKED)},
    {"dwq": At(6 * ROOM, (H,))},  # written behind the last row
    {"wq": None, "dwq": None},
])  # fmt: skip
def test_rotation_backward_in_order(change):
    with in_order():
        back(**change)


@pytest.mark.parametrize("change, match", [
    ({"dq": At(0, Q), "dk": At(2 * H, K)}, "keys' gradient shares GPU memory with"),
    ({"dk_out": At(ROOM, Q), "k": At(3 * ROOM, Q), "dq": At(ROOM, Q), "dk": At(0, Q)}, "queries' gradient shares GPU memory with the gradient of the keys' result"),
    ({"k": At(3 * ROOM, Q), "dk_out": At(ROOM, Q), "dq": At(3 * ROOM, Q), "dk": At(9 * ROOM, Q)}, "queries' gradient shares GPU memory with the keys"),
    ({"dq": At(32, Q)}, "queries' gradient shares GPU memory with the gradient of the queries' result"),
    ({"dq": At(9 * ROOM, Q)}, "keys' gradient shares GPU memory with the queries' gradient"),
    ({"dwk": At(10 * ROOM, (H,))}, "keys' weight's gradient shares GPU memory with the queries' weight's gradient"),
    ({"dwq": At(10 * ROOM + 64, (H,)), "dwk": At(10 * ROOM + 128, (H,))}, "keys' weight's gradient shares GPU memory"),
    ({"dwq": At(2 * ROOM + 512, (H,))}, "queries' weight's gradient shares GPU memory with the queries"),
    ({"dwq": At(8 * ROOM + 512, (H,))}, "queries' weight's gradient shares GPU memory with the queries' gradient"),
    ({"dwk": At(6 * ROOM, (H,))}, "keys' weight's gradient shares GPU memory with the queries' weight"),
    ({"dq": At(8 * ROOM, Q, [S * N * H, N * H, H - 1, 1])}, "elements of the queries' gradient share GPU memory"),
])  # fmt: skip
def test_rotation_backward_refusals(change, match):
    with refused(match):
        back(**change)


def test_one_description_for_both_sides():
    """The C entry given one tensor as queries and keys: the place of one is not the other's own."""
    import ctypes

    lib = _lib.lib()
    lib.lb_qk_norm_rope.restype = ctypes.c_int
    desc = (ctypes.c_float * 2)(1e-6, 0.0)

    def view(at, shape, dtype=10):
        t = _lib.LbTensor()
        t.ptr, t.dtype, t.rank, step = (1 << 30) + at, dtype, len(shape), 1
        for d in range(len(shape) - 1, -1, -1):
            t.shape[d], t.stride[d], step = shape[d], step, step * shape[d]
        return ctypes.byref(t)

    q, table, other = view(0, Q), view(ROOM, (16, 32), 11), view(2 * ROOM, Q)
    with refused("queries' result shares GPU memory with the keys"):
        _lib.check(lib.lb_qk_norm_rope(desc, q, q, table, table, None, None, None, q, other, None))
    with in_order():
        _lib.check(lib.lb_qk_norm_rope(desc, q, q, table, table, None, None, None, other, view(3 * ROOM, Q), None))


@pytest.mark.parametrize("rank", [-5, 0, 2, 9, 1 << 24])
def test_weights_of_any_rank(rank):
    """A description of more dimensions than there are places for is not read beyond them."""
    import ctypes

    def view(*shape, dtype=10, rank=None):
        t, step = _lib.LbTensor(), 1
        t.ptr, t.dtype, t.rank = 4096, dtype, len(shape) if rank is None else rank
        for d in range(len(shape) - 1, -1, -1):
            t.shape[d], t.stride[d], step = shape[d], step, step * shape[d]
        return ctypes.byref(t)

    lib, desc = _lib.lib(), (ctypes.c_float * 2)(1e-6, 0.0)
    with refused("queries' weight must be \\[64\\]"):
        _lib.check(lib.lb_qk_norm_rope(desc, view(*Q), view(*K), view(16, 32, dtype=11), view(16, 32, dtype=11), None, view(H, rank=rank), None, view(*Q), view(*K), None))


# ---- gated block ----------------------------------------------------------------------------------------------------

D, F = 64, 96


def gated(lead=(10,), **change):
    a = {"act": 0, "x": At(0, (*lead, D)), "wgu": At(ROOM, (2 * F, D)), "wd": At(2 * ROOM, (D, F)), "residual": None, "y": At(3 * ROOM, (*lead, D)),
         "gate_up": At(4 * ROOM, (*lead, 2 * F)), "h": At(5 * ROOM, (*lead, F)), "take": take}  # fmt: skip
    assert not change.keys() - a.keys()
    a.update(change)
    _lib.host().gated_mlp_fwd(*a.values(), 0)


def gated_back(lead=(10,), **change):
    a = {"act": 0, "dy": At(0, (*lead, D)), "x": At(ROOM, (*lead, D)), "wgu": At(2 * ROOM, (2 * F, D)), "wd": At(3 * ROOM, (D, F)), "gate_up": At(4 * ROOM, (*lead, 2 * F)),
         "h": At(5 * ROOM, (*lead, F)), "dx": At(6 * ROOM, (*lead, D)), "dwgu": At(7 * ROOM, (2 * F, D)), "dwd": At(8 * ROOM, (D, F)), "take": take}  # fmt: skip
    assert not change.keys() - a.keys()
    a.update(change)
    _lib.host().gated_mlp_bwd(*a.values(), 0)


@pytest.mark.parametrize("lead", [(0,), (3, 0), (0, 3), (5, 0, 2), (2, 5, 0), (0, 0), (1, 0, 7)])
def test_batches_without_tokens(lead):
    gated(lead)  # nothing to do
    gated(lead, residual=At(6 * ROOM, (*lead, D)), gate_up=None)
    with in_order():  # the weights' gradients are empty sums
        gated_back(lead)


def test_operands_in_any_direction():
    """Rows that go backwards through memory: what they cover lies in front of their first one."""
    up, down = At(3 * ROOM, (10, D)), At(3 * ROOM + 2 * 9 * D, (10, D), [-D, 1])
    with refused("shares memory with an operand"):
        gated(x=down, y=up)
    with in_order():
        gated(x=At(3 * ROOM, (10, D), [-D, 1]), y=At(3 * ROOM + 2 * D, (10, D)))
    with refused("shares memory with an operand"):
        gated_back(h=At(6 * ROOM + 2 * 9 * F, (10, F), [-F, 1]), dx=At(6 * ROOM, (10, D)))
    with in_order():  # every other row, and the rows between them
        gated(x=At(0, (10, D), [2 * D, 1]), y=At(2 * D, (10, D), [2 * D, 1]))


def test_sizes_of_scratch_do_not_ask_where_memory_is():
    import ctypes

    def view(*shape):
        t = _lib.LbTensor()
        t.ptr, t.dtype, t.rank = 4096, 10, 2
        t.shape[0], t.shape[1], t.stride[0], t.stride[1] = *shape, shape[1], 1
        return ctypes.byref(t)

    lib, got = _lib.lib(), ctypes.c_size_t()
    x, wgu, wd, gate_up, h = view(200, D), view(2 * F, D), view(D, F), view(200, 2 * F), view(200, F)
    _lib.check(lib.lb_gated_mlp_fwd_scratch_bytes(0, x, wgu, wd, x, gate_up, h, ctypes.byref(got)))
    _lib.check(lib.lb_gated_mlp_bwd_scratch_bytes(0, x, x, wgu, wd, gate_up, h, x, wgu, wd, ctypes.byref(got)))
    assert got.value >= 200 * 2 * F * 2  # both projections' gradients


# ---- clipping -------------------------------------------------------------------------------------------------------


def clip(tensors, out, norm, most=1.0):
    _lib.host().clip_grad_norm(tensors, out, most, norm, take, 0)


def test_the_norms_place():
    x, y, empty = At(0, (10,), dtype="float32"), At(ROOM, (9,)), At(64, (0, 3))
    for at in (-4, 40, ROOM - 4, ROOM + 20, 64):
        with in_order():
            clip([x, y, empty], None, At(at, (), dtype="float32"))
    with in_order():
        clip([x], [At(2 * ROOM, (10,), dtype="float32")], At(40, (1,), dtype="float32"))
    for at in (0, 36, ROOM, ROOM + 16):
        with refused("the norm and tensor [01] share memory"):
            clip([x, y], None, At(at, (), dtype="float32"))
    for at in (4, 2 * ROOM + 36):
        with refused("the norm and (tensor|result) 0 share memory"):
            clip([x], [At(2 * ROOM, (10,), dtype="float32")], At(at, (), dtype="float32"))
    with in_order():  # the norm alone is written behind the last read
        clip([x], None, At(0, (), dtype="float32"), None)
