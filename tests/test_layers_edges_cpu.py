"""Calls of the layers beside ParaConv2d that have to be refused before
anything is launched, or that a tracer makes: without a GPU."""
import pytest

from paraconv2d_b200 import _lib

lib = _lib.cabi()
INVALID = _lib.PC2D_ERR_INVALID_ARGUMENT
ONE = 256  # an aligned address: every call here ends before it is used


@pytest.mark.parametrize("dtype,size", [(0, 4), (2, 2), (3, 2)])
@pytest.mark.parametrize("which", ["B", "C"])
def test_scan_step_refuses_inputs_off_a_vector_boundary(dtype, size, which):
    """The step reads B and C by vectors."""
    at = dict(B=ONE, C=ONE)
    at[which] += size
    st = lib.pc2d_ssm_scan_step(dtype, ONE, ONE, ONE, ONE, at["B"], at["C"], None, None, None, None, 1, 2, 2, 4, 16, 1,
                                ONE, None)
    assert st == INVALID and b"aligned" in lib.pc2d_last_error()
