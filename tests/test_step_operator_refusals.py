"""What the linear cross entropy and the AdamW step refuse, on stand-ins for tensors: wrong shapes, dtypes, layouts, shared memory and workspaces are
errors before anything is launched. No GPU: a call that is in order gets as far as the library's error that there is none."""

import pytest
import torch

from lumen_b200 import _lib, runtime
from tests.test_host_path import Array

if torch.cuda.is_available():  # the calls that are in order would run, on stand-ins' memory
    pytest.skip("refusals are tested where nothing can run", allow_module_level=True)


class At(Array):
    """A stand-in somewhere in memory."""

    def __init__(self, shape, dtype="float32", at=0, **more):
        super().__init__(shape, dtype, **more)
        self.at = at << 24

    def data_ptr(self):
        return (1 << 30) + self.at


class Nowhere(Array):
    def data_ptr(self):
        return 0


def take(nbytes):
    return At((nbytes,), "uint8", 63)


def refused(match):
    return pytest.raises(_lib.LumenError, match=match)


def reaches_the_gpu():
    return pytest.raises(_lib.LumenError, match="CUDA|driver|device|GPU")


# ---- cross entropy --------------------------------------------------------------------------------------------------


def loss(**change):
    a = {"reduction": 2, "ignored": -100, "x": At((2, 5, 64), "bfloat16", 0), "weight": At((300, 64), "bfloat16", 1), "targets": At((2, 5), "int64", 2), "loss": At((), at=3),
         "lse": At((2, 5), at=4), "take": take}  # fmt: skip
    a.update(change)
    _lib.host().linear_cross_entropy(*a.values(), 0)


def loss_back(**change):
    a = {"reduction": 2, "ignored": -100, "d_loss": At((), at=8), "x": At((2, 5, 64), "bfloat16", 0), "weight": At((300, 64), "bfloat16", 1),
         "targets": At((2, 5), "int64", 2), "lse": At((2, 5), at=4), "d_x": At((2, 5, 64), "bfloat16", 5), "d_weight": At((300, 64), "bfloat16", 6), "take": take}  # fmt: skip
    a.update(change)
    _lib.host().linear_cross_entropy_bwd(*a.values(), 0)


def test_cross_entropy_in_order():
    for change in ({}, {"reduction": 0, "loss": At((2, 5), at=3)}, {"reduction": 1}, {"targets": At((2, 5), "int32", 2)}, {"targets": At((2, 5), "int64", 2, strides=[15, 3])},
                   {"weight": At((300, 64), "bfloat16", 1, strides=[1, 300])}, {"loss": At((1,), at=3)}):  # fmt: skip
        with reaches_the_gpu():
            loss(**change)
    for change in ({}, {"d_loss": None}, {"reduction": 0, "d_loss": At((2, 5), at=8, strides=[0, 0])}, {"lse": At((2, 5), at=4, strides=[10, 2])}):
        with reaches_the_gpu():
            loss_back(**change)


@pytest.mark.parametrize("change, match", [
    ({"reduction": 3}, "unknown reduction"),
    ({"x": At((2, 5, 64), "float64")}, "float16, bfloat16 or float32"),
    ({"x": At((2, 5, 64), "float16")}, "of x's dtype"),
    ({"weight": At((300, 63), "bfloat16", 1)}, "weight must be \\[classes, 64\\]"),
    ({"weight": At((3, 100, 64), "bfloat16", 1)}, "weights must be \\[classes, width\\]"),
    ({"weight": At((0, 64), "bfloat16", 1)}, "vocabulary of zero"),
    ({"targets": At((10,), "int64", 2)}, "targets must have the shape"),
    ({"targets": At((5, 2), "int64", 2)}, "targets must have the shape"),
    ({"targets": At((2, 5), "float32", 2)}, "int32 or int64"),
    ({"targets": Nowhere((2, 5), "int64")}, "no memory"),
    ({"x": At((2, 5, 64), "bfloat16", strides=[1000, 64, 1])}, "not evenly spaced"),
    ({"loss": At((2, 5), at=3)}, "one float32 value"),
    ({"loss": At((), "bfloat16", at=3)}, "one float32 value"),
    ({"reduction": 0}, "loss must be float32 of the targets' shape"),
    ({"lse": At((2, 4), at=4)}, "lse must be float32"),
    ({"lse": At((2, 5), "float64", at=4)}, "lse must be float32"),
    ({"lse": At((2, 5), at=4, strides=[0, 0])}, "dense"),
    ({"lse": At((2, 5), at=0)}, "shares memory with an operand"),
    ({"loss": At((), at=4)}, "two results share memory"),
    ({"take": lambda nbytes: Nowhere((nbytes,), "uint8")}, "bytes of scratch are needed"),
])  # fmt: skip
def test_cross_entropy_refusals(change, match):
    with refused(match):
        loss(**change)


@pytest.mark.parametrize("change, match", [
    ({"d_loss": At((2, 5), at=8)}, "one float32 value"),
    ({"d_loss": At((), "float64", at=8)}, "one float32 value"),
    ({"reduction": 0}, "d_loss must be float32 of the targets' shape"),
    ({"d_x": At((2, 5, 64), "float32", 5)}, "shape and dtype of x"),
    ({"d_x": At((2, 4, 64), "bfloat16", 5)}, "shape and dtype of x"),
    ({"d_x": At((2, 5, 64), "bfloat16", 5, strides=[5, 1, 10])}, "row-major"),
    ({"d_x": At((2, 5, 64), "bfloat16", 5, strides=[0, 0, 1])}, "overlap"),
    ({"d_weight": At((64, 300), "bfloat16", 6)}, "shape and dtype of the weights"),
    ({"d_weight": At((300, 64), "bfloat16", 1)}, "shares memory with an operand"),
    ({"d_x": At((2, 5, 64), "bfloat16", 6)}, "two results share memory"),
    ({"lse": At((10,), at=4)}, "lse must be float32"),
    ({"take": lambda nbytes: Nowhere((nbytes,), "uint8")}, "bytes of scratch are needed"),
])  # fmt: skip
def test_cross_entropy_backward_refusals(change, match):
    with refused(match):
        loss_back(**change)


def test_reductions_by_name():
    with pytest.raises(ValueError, match="reduction must be one of"):
        runtime._reduction("average")


# ---- AdamW ----------------------------------------------------------------------------------------------------------


def step(**change):
    a = {"params": [At((1000,), "bfloat16", 0), At((20, 30), "float32", 1)], "grads": [At((1000,), "bfloat16", 2), At((20, 30), "float32", 3)],
         "m": [At((1000,), at=4), At((20, 30), at=5)], "v": [At((1000,), at=6), At((20, 30), at=7)], "ms": None, "vs": None, "masters": None, "step": 1, "lr": 1e-3, "b1": 0.9,
         "b2": 0.999, "eps": 1e-8, "decay": 0.01, "norm": None, "max_norm": 0.0}  # fmt: skip
    a.update(change)
    _lib.host().adamw_step(*a.values(), 0)


EIGHT = {"m": [At((1000,), "uint8", 4), At((20, 30), "uint8", 5)], "v": [At((1000,), "uint8", 6), At((20, 30), "uint8", 7)], "ms": [At((4,), at=8), At((3,), at=9)],
         "vs": [At((4,), at=10), At((3,), at=11)]}  # fmt: skip


def test_a_step_in_order():
    for change in ({}, EIGHT, {"grads": [At((1000,), "float32", 2), At((20, 30), "float32", 3)]}, {"masters": [At((1000,), at=12), None]}, {"lr": 1}, {"lr": At((), at=12)},
                   {"step": At((1,), "int32", 12)}, {"norm": At((), at=12), "max_norm": 1.0}, {"grads": [At((1000,), "float32", 2), At((20, 30), "float32", 2)]}):  # fmt: skip
        with reaches_the_gpu():
            step(**change)


@pytest.mark.parametrize("change, match", [
    ({"params": [At((1000,), "float64", 0), At((20, 30), "float32", 1)]}, "parameter 0 is float64"),
    ({"params": [At((1000,), "bfloat16", 0, strides=[2]), At((20, 30), "float32", 1)]}, "parameter 0 is not dense"),
    ({"grads": [At((1000,), "float16", 2), At((20, 30), "float32", 3)]}, "gradient 0 is float16, not bfloat16"),
    ({"grads": [At((1000,), "bfloat16", 2), At((30, 20), "float32", 3)]}, "gradient 1 must have its parameter's shape"),
    ({"grads": [At((1000,), "bfloat16", 2), At((20, 30), "float32", 3, strides=[1, 20])]}, "gradient 1 must have its parameter's shape and strides"),
    ({"m": [At((1000,), "bfloat16", 4), At((20, 30), at=5)]}, "first moment 0 is bfloat16, not float32"),
    ({"v": [At((1000,), at=6), At((600,), at=7)]}, "second moment 1 must have"),
    ({"m": [At((1000,), at=4), At((20, 30), at=4)]}, "share memory"),
    ({"m": [At((1000,), at=2), At((20, 30), at=5)]}, "share memory"),
    ({"params": [At((1000,), "bfloat16", 0), At((20, 30), "float32", 0)]}, "share memory"),
    ({"norm": At((), at=6), "max_norm": 1.0}, "share memory"),
    ({"ms": EIGHT["ms"]}, "both moments have scales"),
    ({**EIGHT, "ms": [At((3,), at=8), At((3,), at=9)]}, "scales of parameter 0 must be dense float32 \\[4\\]"),
    ({**EIGHT, "vs": [At((4,), "bfloat16", at=10), At((3,), at=11)]}, "scales of parameter 0"),
    ({**EIGHT, "v": [At((1000,), at=6), At((20, 30), "uint8", 7)]}, "second moment 0 is float32, not uint8"),
    ({**EIGHT, "vs": [At((4,), at=8), At((3,), at=11)]}, "share memory"),
    ({"masters": [None, At((20, 30), at=12)]}, "parameter 1 is float32 itself"),
    ({"masters": [At((1000,), "bfloat16", at=12), None]}, "float32 copy 0 is bfloat16"),
    ({"masters": [At((999,), at=12), None]}, "float32 copy 0 must have"),
    ({"masters": [At((1000,), at=6), None]}, "share memory"),
    ({"step": 0}, "counted from 1"),
    ({"step": At((2,), "int32", 12)}, "the step count"),
    ({"step": At((), "float64", 12)}, "the step count"),
    ({"lr": At((), "bfloat16", 12)}, "the learning rate"),
    ({"lr": float("nan")}, "lr must be finite"),
    ({"eps": -1e-8}, "eps must not be negative"),
    ({"b1": 1.0}, "betas"),
    ({"b2": -0.1}, "betas"),
    ({"decay": float("inf")}, "weight_decay must be finite"),
    ({"norm": At((), at=12), "max_norm": -1.0}, "max_norm"),
    ({"norm": At((2,), at=12), "max_norm": 1.0}, "the norm"),
    ({"m": [Nowhere((1000,)), At((20, 30), at=5)]}, "first moment 0 has no memory"),
])  # fmt: skip
def test_step_refusals(change, match):
    with refused(match):
        step(**change)


@pytest.mark.parametrize("change, match", [
    ({"grads": [At((1000,), "bfloat16", 2)]}, "2 parameters and 1 gradients"),
    ({"masters": [None]}, "2 parameters and 1 float32 copies"),
])  # fmt: skip
def test_lists_of_other_lengths(change, match):
    with pytest.raises(ValueError, match=match):
        step(**change)


def test_what_the_wrapper_refuses(monkeypatch):
    monkeypatch.setattr(runtime, "require_cuda", lambda: None)
    p = [At((10,))]
    with pytest.raises(ValueError, match="both the norm and max_norm"):
        runtime.adamw_step(p, p, p, p, 1, max_norm=1.0)
    with pytest.raises(ValueError, match="bits must be 8 or 32"):
        runtime.adamw_state(p, bits=16)
