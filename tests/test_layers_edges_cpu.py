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


CONV_FORWARD = dict(input=ONE, weight=ONE, bias=ONE, init=ONE, lengths=ONE, out=ONE, final=ONE)
CONV_BACKWARD = dict(grad=ONE, gfinal=ONE, input=ONE, weight=ONE, bias=ONE, init=ONE, lengths=ONE, dx=ONE, dw=ONE,
                     db=ONE, dinit=ONE)
CONV_STEP = dict(input=ONE, state=ONE, weight=ONE, bias=ONE, slots=ONE, out=ONE)
SCAN_FORWARD = dict(u=ONE, delta=ONE, A=ONE, B=ONE, C=ONE, skip=ONE, z=ONE, bias=ONE, init=ONE, lengths=ONE, out=ONE,
                    final=ONE, ckpt=ONE)
SCAN_BACKWARD = dict(grad=ONE, gfinal=ONE, u=ONE, delta=ONE, A=ONE, B=ONE, C=ONE, skip=ONE, z=ONE, bias=ONE,
                     lengths=ONE, ckpt=ONE, du=ONE, dd=ONE, dA=ONE, dB=ONE, dC=ONE, dskip=ONE, dz=ONE, dbias=ONE,
                     dinit=ONE)
SCAN_STEP = dict(u=ONE, delta=ONE, state=ONE, A=ONE, B=ONE, C=ONE, skip=ONE, z=ONE, bias=ONE, slots=ONE, out=ONE)
WS = 1 << 40  # (a size; nothing is allocated)


def _refused(call, arrays, **off):
    assert call(*[v + off.get(k, 0) for k, v in arrays.items()]) == INVALID, off
    assert b"aligned" in lib.pc2d_last_error(), (off, lib.pc2d_last_error())


@pytest.mark.parametrize("call,arrays", [
    (lambda *p: lib.pc2d_causal_conv_forward(3, 3, *p[:5], 2, 3, 5, 4, 1, *p[5:], None), CONV_FORWARD),
    (lambda *p: lib.pc2d_causal_conv_backward(3, 3, *p[:7], 2, 3, 5, 4, 1, *p[7:], ONE, WS, None), CONV_BACKWARD),
    (lambda *p: lib.pc2d_causal_conv_step(3, 3, *p[:5], 2, 2, 3, 4, 1, p[5], None), CONV_STEP),
    (lambda *p: lib.pc2d_ssm_scan_forward(3, *p[:10], 1, 2, 4, 5, 16, 1, *p[10:], ONE, WS, None), SCAN_FORWARD),
    (lambda *p: lib.pc2d_ssm_scan_backward(3, *p[:12], 1, 2, 4, 5, 16, 1, *p[12:], ONE, WS, None), SCAN_BACKWARD),
    (lambda *p: lib.pc2d_ssm_scan_step(3, *p[:10], 1, 2, 2, 4, 16, 1, p[10], None), SCAN_STEP)],
    ids=["conv_forward", "conv_backward", "conv_step", "scan_forward", "scan_backward", "scan_step"])
def test_arrays_off_their_elements_boundary_are_refused(call, arrays):
    """An odd address, for each array of each call in turn."""
    for k in arrays:
        _refused(call, arrays, **{k: 1})


def test_wider_elements_off_their_boundary_are_refused():
    """float32 weights, and numbers of lengths and slots, two bytes off."""
    for k in ("weight", "bias", "lengths"):
        _refused(lambda *p: lib.pc2d_causal_conv_forward(3, 0, *p[:5], 2, 3, 5, 4, 1, *p[5:], None), CONV_FORWARD, **{k: 2})
    for k in ("skip", "bias", "lengths", "dA", "dskip", "dbias"):
        _refused(lambda *p: lib.pc2d_ssm_scan_backward(3, *p[:12], 1, 2, 4, 5, 16, 1, *p[12:], ONE, WS, None),
                 SCAN_BACKWARD, **{k: 2})
    for k in ("weight", "bias", "slots"):
        _refused(lambda *p: lib.pc2d_causal_conv_step(3, 0, *p[:5], 2, 2, 3, 4, 1, p[5], None), CONV_STEP, **{k: 2})
    for k in ("skip", "bias", "slots"):
        _refused(lambda *p: lib.pc2d_ssm_scan_step(3, *p[:10], 1, 2, 2, 4, 16, 1, p[10], None), SCAN_STEP, **{k: 2})
    for dtype, size in ((0, 4), (1, 8), (2, 2), (3, 2)):
        for k in range(3):
            at = [ONE + (size // 2 if i == k else 0) for i in range(3)]  # input, residual, output
            assert lib.pc2d_dropout(dtype, at[0], at[1], ONE, 0.5, 8, at[2], None) == INVALID
        assert lib.pc2d_dropout(dtype, ONE, None, ONE + 4, 0.5, 8, ONE, None) == INVALID
    assert lib.pc2d_dropout_next_key(ONE + 4, ONE, None) == INVALID
    assert lib.pc2d_dropout_next_key(ONE, ONE + 4, None) == INVALID
