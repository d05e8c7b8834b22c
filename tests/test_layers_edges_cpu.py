"""Calls of the layers beside ParaConv2d that have to be refused before
anything is launched, or that a tracer makes: without a GPU."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch._subclasses.fake_tensor import FakeTensorMode, UnsupportedOperatorException

import paraconv2d_b200 as pc
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


def _fw_calls():
    """Each entry point with each of its tensors that can carry a derivative."""
    r = lambda *s: torch.randn(*s)  # noqa: E731
    key = torch.tensor([1, 2])
    x, w, one = r(2, 6, 8), r(6, 4), r(2, 6)
    yield "dropout", lambda t: pc.dropout(t["x"], 0.5, key, residual=t["residual"]), dict(x=x, residual=r(2, 6, 8))
    yield "causal_conv", lambda t: pc.causal_conv(t["x"], t["w"], t["b"], None, t["init"]), dict(x=x, w=w, b=r(6), init=r(2, 6, 3))
    yield "causal_conv_step", lambda t: pc.causal_conv_step(t["x"], t["state"], t["w"], t["b"]), dict(
        x=one, state=r(2, 6, 3), w=w, b=r(6))
    scan = dict(u=x, delta=x, A=r(6, 4), B=r(2, 1, 4, 8), C=r(2, 1, 4, 8), D=r(6), z=x, bias=r(6), init=r(2, 6, 4))
    yield "ssm_scan", lambda t: pc.ssm_scan(t["u"], t["delta"], t["A"], t["B"], t["C"], t["D"], t["z"], t["bias"], True,
                                            t["init"]), scan
    step = dict(u=one, delta=one, state=r(2, 6, 4), A=r(6, 4), B=r(2, 1, 4), C=r(2, 1, 4), D=r(6), z=one, bias=r(6))
    yield "ssm_scan_step", lambda t: pc.ssm_scan_step(t["u"], t["delta"], t["state"], t["A"], t["B"], t["C"], t["D"],
                                                      t["z"], t["bias"]), step


FW = {name: (call, tensors) for name, call, tensors in _fw_calls()}


@pytest.mark.parametrize("name", list(FW))
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(name, grad):
    """With a tangent in any input: an error that says so, not an output
    without a derivative.  (Before the refusal of tensors on the CPU.)"""
    call, tensors = FW[name]
    for k, v in tensors.items():
        with fwd.dual_level():
            dual = fwd.make_dual(v.clone().requires_grad_() if grad and "step" not in name else v, torch.ones_like(v))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call({**tensors, k: dual})
        with pytest.raises(NotImplementedError, match="CUDA tensors only|CPU"):
            call(tensors)


@pytest.mark.parametrize("name", ["dropout", "causal_conv", "ssm_scan"])
def test_jvp_is_refused(name):
    call, tensors = FW[name]
    k = next(iter(tensors))
    with pytest.raises((NotImplementedError, RuntimeError), match="forward-mode|functorch"):
        torch.func.jvp(lambda v: call({**tensors, k: v}), (tensors[k],), (torch.ones_like(tensors[k]),))


@pytest.mark.parametrize("name", list(FW))
@pytest.mark.parametrize("grad", [False, True])
def test_fake_tensors_are_refused_as_a_tracer_expects(name, grad, recwarn):
    """Tensors without data (a tracer's) on a GPU that need not be there: no
    kernel's host code runs on them, and the error is the tracer's own."""
    call, tensors = FW[name]
    key = {"key": torch.zeros(2, dtype=torch.int64)}
    with FakeTensorMode():
        t = {k: torch.empty(v.shape, device="cuda", dtype=v.dtype) for k, v in {**tensors, **key}.items()}
        if grad and "step" not in name:
            t[next(iter(tensors))].requires_grad_()
        if name == "dropout":
            call = lambda t: pc.dropout(t["x"], 0.5, t["key"], residual=t["residual"])  # noqa: E731
        with pytest.raises(UnsupportedOperatorException):
            call(t)
    assert not [w for w in recwarn if "data pointer" in str(w.message)]
