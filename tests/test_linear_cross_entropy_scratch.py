"""How much scratch the linear cross entropy asks for: pieces of the vocabulary bound all that grows with it. No GPU: the sizes are arithmetic."""

import ctypes

import pytest

from lumen_b200 import _lib

MB = 1 << 20


class Desc(ctypes.Structure):
    _fields_ = [("reduction", ctypes.c_int32), ("reserved", ctypes.c_int32), ("ignore_index", ctypes.c_int64)]


def scratch(t, d, v, dtype, backward):
    x, w, targets = _lib.dense(1 << 40, dtype, (t, d)), _lib.dense(1 << 41, dtype, (v, d)), _lib.dense(1 << 42, "int64", (t,))
    desc, out = Desc(2, 0, -100), ctypes.c_size_t()
    if backward:
        rc = _lib.lib().lb_linear_cross_entropy_bwd_scratch_bytes(*map(ctypes.byref, (desc, x, w, targets, x, w, out)))
    else:
        rc = _lib.lib().lb_linear_cross_entropy_scratch_bytes(*map(ctypes.byref, (desc, x, w, targets, out)))
    _lib.check(rc)
    return out.value


DTYPES = ["bfloat16", "float16", "float32"]


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_rows_need_nothing(dtype):
    for d, v in ((4096, 131072), (4100, 131072), (101, 3)):
        assert scratch(0, d, v, dtype, True) == 0 and scratch(0, d, v, dtype, False) < 4096


@pytest.mark.parametrize("dtype", DTYPES)
def test_few_rows_in_one_pass_keep_no_copy_of_the_gradient(dtype):
    item = 4 if dtype == "float32" else 2
    for d in (4096, 4100):  # 4100: rows of the gradient that no tile stores
        # logits in memory (of rows that TMA does not take), dz (two parts of 16 bits), x as often, and d_x's ranges: four blocks an SM, of 512 columns each
        assert scratch(4, d, 131072, dtype, True) <= 4 * (131072 + 64) * 4 + 2 * 4 * (131072 + 64 + d + 64) * item + 4 * 148 * 512 * 4 * 4 + 4 * d * 4 + 8192


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t", [5, 61, 100, 300, 4000])
@pytest.mark.parametrize("shape", [(4096, 131072), (4100, 131072), (101, 5000001), (16384, 200000), (520, 1000003)])
def test_pieces_bound_it(dtype, t, shape):
    """256 MB each of logits, dz and what the weights or their gradient need beside them, a dozen x, and eight bytes of each row's 128 logits in the forward pass."""
    d, v = shape
    assert scratch(t, d, v, dtype, True) <= 3 * 256 * MB + 64 * 65536 + 12 * t * (d + 64) * 4 + 40 * MB
    assert scratch(t, d, v, dtype, False) <= 3 * 256 * MB + 64 * 65536 + 3 * t * (d + 64) * 4 + 8 * t * (v // 128 + 2) + 8 * MB
