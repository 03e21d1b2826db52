"""What the operators of a decoder layer's step refuse, on stand-ins for tensors: wrong shapes, dtypes, layouts and workspaces are errors before anything
is launched. No GPU: a call that is in order gets as far as the library's error that there is none."""

import pytest
import torch

from lumen_b200 import _lib
from tests.test_host_path import Array

if torch.cuda.is_available():  # the calls that are in order would run, on stand-ins' memory
    pytest.skip("refusals are tested where nothing can run", allow_module_level=True)


def take(nbytes):
    return Array((nbytes,), "uint8")


def refused(match):
    return pytest.raises(_lib.LumenError, match=match)


def reaches_the_gpu():
    return pytest.raises(_lib.LumenError, match="CUDA|driver|device|GPU")


class At(Array):
    """A stand-in somewhere else in memory."""

    def __init__(self, shape, dtype="float32", at=0, **more):
        super().__init__(shape, dtype, **more)
        self.at = at

    def data_ptr(self):
        return (1 << 30) + self.at


class Torch(At):
    def __init__(self, shape, dtype="float32", at=0, device=0, contiguous=True):
        super().__init__(shape, dtype, at)
        self.device_index, self.contiguous = device, contiguous

    def get_device(self):
        return self.device_index

    def is_contiguous(self):
        return self.contiguous

    def numel(self):
        n = 1
        for d in self.shape:
            n *= d
        return n


# ---- rotation -------------------------------------------------------------------------------------------------------


def rope(**change):
    a = {"eps": 1e-6, "interleaved": False, "q": Array((2, 5, 4, 64)), "k": Array((2, 5, 2, 64)), "cos": Array((16, 32)), "sin": Array((16, 32)), "positions": None,
         "wq": None, "wk": None, "q_out": Array((2, 5, 4, 64)), "k_out": Array((2, 5, 2, 64))}  # fmt: skip
    a.update(change)
    _lib.host().qk_norm_rope(*a.values(), 0)


def rope_back(**change):
    a = {"eps": 1e-6, "interleaved": False, "dq_out": Array((2, 5, 4, 64)), "dk_out": Array((2, 5, 2, 64)), "q": Array((2, 5, 4, 64)), "k": Array((2, 5, 2, 64)),
         "cos": Array((16, 32)), "sin": Array((16, 32)), "positions": None, "wq": Array((64,)), "wk": Array((64,)), "dq": Array((2, 5, 4, 64)),
         "dk": Array((2, 5, 2, 64)), "dwq": Array((64,)), "dwk": Array((64,)), "take": take}  # fmt: skip
    a.update(change)
    _lib.host().qk_norm_rope_bwd(*a.values(), 0)


def test_rotation_in_order():
    with reaches_the_gpu():
        rope()
    with reaches_the_gpu():
        rope(positions=Array((2, 5), "int64"), wq=Array((64,)), wk=Array((64,)))
    with reaches_the_gpu():
        rope_back()


@pytest.mark.parametrize("change, match", [
    ({"q": Array((5, 4, 64))}, "must be \\[batch, sequence, heads, head dim\\]"),
    ({"q": Array((2, 5, 4, 64), "float64"), "k": Array((2, 5, 2, 64), "float64")}, "must share a dtype"),
    ({"k": Array((2, 5, 2, 64), "bfloat16")}, "must share a dtype"),
    ({"k": Array((2, 4, 2, 64))}, "must share batch, sequence and head dim"),
    ({"q": Array((2, 5, 4, 257)), "k": Array((2, 5, 2, 257))}, "head dims of 1 to 256"),
    ({"q": Array((2, 5, 4, 0)), "k": Array((2, 5, 2, 0))}, "head dims of 1 to 256"),
    ({"cos": Array((16, 33)), "sin": Array((16, 33))}, "33 pairs must be 1 to 32"),
    ({"cos": Array((16, 0)), "sin": Array((16, 0))}, "0 pairs must be 1 to 32"),
    ({"cos": Array((16, 32), "bfloat16")}, "float32 tables of one shape"),
    ({"sin": Array((15, 32))}, "float32 tables of one shape"),
    ({"cos": Array((4, 32)), "sin": Array((4, 32))}, "hold 4 positions, the sequence has 5"),
    ({"cos": Array((0, 32)), "sin": Array((0, 32)), "positions": Array((5,), "int32")}, "no position"),
    ({"positions": Array((5,), "float32")}, "int32 or int64"),
    ({"positions": Array((4,), "int32")}, "\\[sequence\\] or \\[batch, sequence\\]"),
    ({"positions": Array((1, 5), "int32")}, "\\[sequence\\] or \\[batch, sequence\\]"),
    ({"wq": Array((32,))}, "queries' weight must be \\[64\\]"),
    ({"wk": Array((64,), "float16")}, "keys' weight must be \\[64\\]"),
    ({"wk": Array((64,), strides=[2])}, "dense"),
    ({"q_out": Array((2, 5, 2, 64))}, "a result must have"),
    ({"q_out": Array((2, 5, 4, 64), strides=[1280, 256, 0, 1])}, "broadcast view"),
    ({"eps": -1.0}, "eps"),
    ({"eps": float("nan")}, "eps"),
    ({"q": Array((1 << 20, 1 << 12, 1, 64), strides=[0, 0, 0, 1]), "k": Array((1 << 20, 1 << 12, 1, 64), strides=[0, 0, 0, 1])}, "rows in one call"),
])  # fmt: skip
def test_rotation_refusals(change, match):
    with refused(match):
        rope(**change)


@pytest.mark.parametrize("change, match", [
    ({"dq_out": Array((2, 5, 2, 64))}, "a gradient must have"),
    ({"dk": Array((2, 5, 2, 64), "bfloat16")}, "a gradient must have"),
    ({"dwq": None}, "a weight has a gradient"),
    ({"wk": None}, "a weight has a gradient"),
    ({"dwk": Array((64,), "bfloat16")}, "a weight's gradient must have"),
])  # fmt: skip
def test_rotation_backward_refusals(change, match):
    with refused(match):
        rope_back(**change)


def test_rotation_scratch():
    import ctypes

    lib = _lib.lib()
    lib.lb_qk_norm_rope_bwd_scratch_bytes.restype = ctypes.c_size_t
    assert lib.lb_qk_norm_rope_bwd_scratch_bytes(0) == 0 and lib.lb_qk_norm_rope_bwd_scratch_bytes(-3) == 0
    assert 0 < lib.lb_qk_norm_rope_bwd_scratch_bytes(64) < lib.lb_qk_norm_rope_bwd_scratch_bytes(256) < 1 << 24
    with pytest.raises(RuntimeError, match="memory"):  # what the allocator says reaches the caller

        def none(nbytes):
            raise RuntimeError("out of memory")

        rope_back(take=none)


# ---- gated block ----------------------------------------------------------------------------------------------------


def apart(a, change):
    """The call's arguments with `change`, each stand-in in memory of its own unless it says where it is."""
    a.update(change)
    for k, t in enumerate(a.values()):
        if type(t) is Array:
            t.data_ptr = lambda at=(k + 1) << 24: at
    return a.values()


def gated(**change):
    t = "bfloat16"
    a = {"act": 0, "x": Array((10, 64), t), "wgu": Array((192, 64), t), "wd": Array((64, 96), t), "residual": None, "y": Array((10, 64), t),
         "gate_up": Array((10, 192), t), "h": Array((10, 96), t), "take": take}  # fmt: skip
    _lib.host().gated_mlp_fwd(*apart(a, change), 0)


def gated_back(**change):
    t = "bfloat16"
    a = {"act": 0, "dy": Array((10, 64), t), "x": Array((10, 64), t), "wgu": Array((192, 64), t), "wd": Array((64, 96), t), "gate_up": Array((10, 192), t),
         "h": Array((10, 96), t), "dx": Array((10, 64), t), "dwgu": Array((192, 64), t), "dwd": Array((64, 96), t), "take": take}  # fmt: skip
    _lib.host().gated_mlp_bwd(*apart(a, change), 0)


def test_gated_block_in_order():
    t = "bfloat16"
    with reaches_the_gpu():
        gated()
    with reaches_the_gpu():
        gated(gate_up=None, residual=Array((10, 64), t))
    with reaches_the_gpu():
        gated(x=Array((2, 5, 64), t), y=Array((2, 5, 64), t))
    with reaches_the_gpu():
        gated_back()


@pytest.mark.parametrize("change, match", [
    ({"act": 3}, "unknown activation"),
    ({"act": -1}, "unknown activation"),
    ({"x": Array((64,), "bfloat16")}, "rank 2 or more"),
    ({"x": Array((10, 64), "float64")}, "float16, bfloat16 or float32"),
    ({"x": Array((10, 64), "float16")}, "w_gate_up must be \\[192, 64\\]"),
    ({"x": Array((10, 0), "bfloat16")}, "width or hidden size of zero"),
    ({"wgu": Array((0, 64), "bfloat16")}, "width or hidden size of zero"),
    ({"wgu": Array((193, 64), "bfloat16")}, "even number of rows"),
    ({"wgu": Array((1, 192, 64), "bfloat16")}, "must have rank 2"),
    ({"wd": Array((96, 64), "bfloat16")}, "w_down must be \\[64, 96\\]"),
    ({"y": Array((10, 96), "bfloat16")}, "y must be \\[10, 64\\]"),
    ({"y": Array((10, 64), "float32")}, "y must be \\[10, 64\\]"),
    ({"y": Array((10, 64), "bfloat16", strides=[1, 10])}, "y must be row-major"),
    ({"y": Array((10, 64), "bfloat16", strides=[0, 1])}, "rows of y overlap"),
    ({"gate_up": Array((10, 96), "bfloat16")}, "gate_up must be \\[10, 192\\]"),
    ({"h": Array((9, 96), "bfloat16")}, "h must be \\[10, 96\\]"),
    ({"h": None}, "h is missing"),
    ({"residual": Array((10, 96), "bfloat16")}, "residual must be"),
    ({"residual": Array((10, 64), "bfloat16", strides=[1, 10])}, "residual must be row-major"),
    ({"x": Array((3, 4, 64), "bfloat16", strides=[1000, 64, 1])}, "not evenly spaced"),
])  # fmt: skip
def test_gated_block_refusals(change, match):
    with refused(match):
        gated(**change)


def test_gated_block_scratch():
    """Float32 operands without what is kept: the projections need a place."""
    t = "float32"
    place = {"x": Array((10, 64), t), "wgu": Array((192, 64), t), "wd": Array((64, 96), t), "y": Array((10, 64), t), "gate_up": None, "h": Array((10, 96), t)}
    with refused("bytes of scratch are needed, 16-byte aligned"):
        gated(**place, take=lambda nbytes: At((nbytes,), "uint8", 8))
    with refused("bytes of scratch are needed, 16-byte aligned"):
        gated_back(take=lambda nbytes: At((nbytes,), "uint8", 8))
    with reaches_the_gpu():
        gated(**place)


def test_gated_block_results_in_operands_memory():
    t = "bfloat16"
    here = {"x": At((10, 64), t), "y": At((10, 64), t, 2 * 10 * 64)}
    with reaches_the_gpu():  # one behind the other
        gated(**here)
    with reaches_the_gpu():  # columns of one matrix
        gated(x=At((10, 64), t, strides=[128, 1]), y=At((10, 64), t, 128, strides=[128, 1]))
    for change in ({"x": At((10, 64), t), "y": At((10, 64), t)}, {"x": At((10, 64), t), "y": At((10, 64), t, 2 * 10 * 64 - 16)},
                   {"x": At((10, 64), t, strides=[128, 1]), "y": At((10, 64), t, 112, strides=[128, 1])}, {"wgu": At((192, 64), t), "h": At((10, 96), t, 4096)},
                   {"residual": At((10, 64), t), "y": At((10, 64), t)}):  # fmt: skip
        with refused("shares memory with an operand"):
            gated(**change)
    with refused("two results share memory"):
        gated(h=At((10, 96), t), gate_up=At((10, 192), t, 1024))
    with refused("shares memory with an operand"):
        gated_back(x=At((10, 64), t), dx=At((10, 64), t))
    with refused("two results share memory"):
        gated_back(dwd=At((64, 96), t), dwgu=At((192, 64), t))


def test_tensors_without_memory():
    none, t = At((10, 64), "bfloat16", -(1 << 30)), "bfloat16"
    with refused("x has no memory"):
        gated(x=none)
    with refused("queries has no memory"):
        rope(q=At((2, 5, 4, 64), at=-(1 << 30)))
    with refused("positions has no memory or is not aligned"):
        rope(positions=At((5,), "int64", 4))
    with refused("a result has no memory or is not aligned"):
        rope(q_out=At((2, 5, 4, 64), at=2))
    with refused("tensor 0 has no memory"):
        clip([At((5,), at=-(1 << 30))])
    with refused("one float32 value"):
        clip([At((5,))], norm=At((), at=2))


def test_a_residual_of_float32_is_refused():
    t = "float32"
    with refused("16-bit results"):
        gated(x=Array((10, 64), t), wgu=Array((192, 64), t), wd=Array((64, 96), t), residual=Array((10, 64), t), y=Array((10, 64), t), gate_up=None, h=Array((10, 96), t))


@pytest.mark.parametrize("change, match", [
    ({"dy": Array((10, 96), "bfloat16")}, "d_y must be"),
    ({"gate_up": Array((10, 192), "bfloat16", strides=[1, 10])}, "gate_up must be row-major"),
    ({"h": Array((10, 95), "bfloat16")}, "h must be"),
    ({"dx": Array((10, 64), "float32")}, "d_x must be"),
    ({"dwgu": Array((64, 192), "bfloat16")}, "d_w_gate_up must be"),
    ({"dwd": Array((64, 96), "bfloat16", strides=[0, 1])}, "rows of d_w_down overlap"),
])  # fmt: skip
def test_gated_block_backward_refusals(change, match):
    with refused(match):
        gated_back(**change)


# ---- clipping -------------------------------------------------------------------------------------------------------


def clip(tensors, out=None, most=1.0, norm=None, take=take):
    _lib.host().clip_grad_norm(tensors, out, most, norm or At((), "float32", 1 << 28), take, 0)


def test_clipping_in_order():
    for out in (None, [At((5, 3), at=4096), At((8,), "bfloat16", 8192)]):
        with reaches_the_gpu():
            clip([At((5, 3)), At((8,), "bfloat16", 1024)], out)
    with reaches_the_gpu():
        clip([At((5, 3)), At((5, 3))], None, None)  # the norm alone counts a tensor as often as it is there
    with reaches_the_gpu():
        clip([At((4, 6), strides=[1, 4]), At((0, 4), at=4)], None)
    with reaches_the_gpu():
        clip([], None)


@pytest.mark.parametrize("tensors, out, match", [
    ([At((5,), "int32")], None, "is int32"),
    ([At((5, 4), strides=[5, 1])], None, "not dense"),
    ([At((5, 4), strides=[0, 1])], None, "not dense"),
    ([At((5,), strides=[2])], None, "not dense"),
    ([At((2, 2), strides=[1, 1])], None, "not dense"),
    ([At((5,), at=2)], None, "not aligned"),
    ([At((5,))], [At((5,), at=4097)], "not aligned"),
    ([At((5,))], [At((4,), at=4096)], "shape, strides and dtype"),
    ([At((5,))], [At((5,), "bfloat16", at=4096)], "shape, strides and dtype"),
    ([At((2, 3))], [At((2, 3), at=4096, strides=[1, 2])], "shape, strides and dtype"),
    ([At((8,)), At((8,))], None, "share memory"),
    ([At((8,)), At((8,), at=28)], None, "share memory"),
    ([At((8,)), At((8,), at=64)], [At((8,), at=4096), At((8,), at=4112)], "share memory"),
    ([At((8,)), At((8,), at=64)], [At((8,), at=4096), At((8,), at=16)], "share memory"),
    ([At((8,))], [At((8,), at=4)], "share memory"),
])  # fmt: skip
def test_clipping_refusals(tensors, out, match):
    with refused(match):
        clip(tensors, out)


def test_more_clipping_refusals():
    for most in (-1.0, float("nan"), float("inf")):
        with refused("max_norm"):
            clip([At((5,))], None, most)
    with pytest.raises(ValueError, match="2 tensors and 1 results"):
        clip([At((5,)), At((5,), at=64)], [At((5,), at=4096)])
    with pytest.raises(TypeError, match="sequence"):
        clip(3)
    with refused("one float32 value"):
        clip([At((5,))], norm=At((2,), at=1 << 20))
    with refused("one float32 value"):
        clip([At((5,))], norm=At((), "bfloat16", 1 << 20))
    with refused("16-byte aligned"):
        clip([At((5,))], take=lambda nbytes: At((nbytes,), "uint8", 8))


@pytest.mark.parametrize("tensor", [torch.zeros(5), torch.zeros(4, 6).t(), torch.nn.Parameter(torch.zeros(3)), torch.zeros(0, 3, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.complex64)])
def test_torch_tensors_on_the_host(tensor):
    """What torch's exchange table tells is refused like what its methods tell."""
    with pytest.raises((ValueError, TypeError), match="expected a CUDA tensor|no lumen dtype"):
        clip([tensor])


def test_tensors_on_the_host():
    with pytest.raises(ValueError, match="expected a CUDA tensor"):
        clip([Torch((5,), device=-1)])
    with pytest.raises(ValueError, match="expected a CUDA tensor"):
        rope(q=Torch((2, 5, 4, 64), device=-1))
    with pytest.raises(ValueError, match="expected a CUDA tensor"):
        gated(x=Torch((10, 64), "bfloat16", device=-1))
    with pytest.raises(ValueError, match="expected a CUDA tensor"):
        clip([Array((5,), cuda=False)])


def test_without_a_gpu_the_entries_say_so():
    from lumen_b200 import runtime

    x = torch.zeros(2, 3, 4, 64)
    table = torch.zeros(8, 32)
    for call in (lambda: runtime.qk_norm_rope(x, x, table, table), lambda: runtime.gated_mlp_forward(x, x, x), lambda: runtime.grad_norm([x]),
                 lambda: runtime.clip_grad_norm([x], 1.0)):  # fmt: skip
        with pytest.raises(RuntimeError, match="no CUDA device"):
            call()
