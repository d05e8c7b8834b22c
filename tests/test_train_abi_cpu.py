"""The C entry points of the AdamW step: the struct that hosts were built with
keeps its size, and the numbered form refuses what it cannot take."""
import ctypes

import pytest

from paraconv2d_b200 import _lib
from test_train_cpu import INVALID, ONE, WORKSPACE, _tensor

lib = _lib.cabi()


def test_tensors_lie_as_ever():
    assert ctypes.sizeof(_lib.AdamWTensor) == 96 and _lib.AdamWTensor.decay.offset == 88
    assert lib.pc2d_abi_version() == 1


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("number,bytes,code", [(-1, 64, INVALID), (2 ** 31, 64, INVALID), (2 ** 31 - 1, 8, WORKSPACE),
                                               (0, 8, WORKSPACE), (None, 8, WORKSPACE)])
def test_numbers(number, bytes, code, bits):
    tensors = (_lib.AdamWTensor * 2)(*(_tensor(scales=ONE) for _ in range(2)))
    numbers = None if number is None else (ctypes.c_int64 * 2)(5, number)
    st = lib.pc2d_adamw_step_numbered(bits, tensors, 2, numbers, ONE, None, 0.1, 0.9, 0.99, 1e-8, 0.1, None, 0, ONE, bytes,
                                      None)
    assert st == code
