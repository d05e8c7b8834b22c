"""The AdamW step on the GPU: small decays, infinite weights, and the optimizer's
counts and random numbers."""
import pytest
import torch

import paraconv2d_b200 as pc

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("masters", [False, True])
@pytest.mark.parametrize("lr,decay", [(1e-6, 1e-2), (1e-5, 1e-2), (1e-3, 0.1)])
def test_a_weight_is_rounded_once(lr, decay, masters, bits):
    """What a step takes of a weight, its decay included, is summed first and then subtracted: beside that rounding of the
    weight there are only those of the step (16 cover its root, quotient and factors) and of the decay."""
    n, g = 1 << 20, gen(1)
    w, grad = torch.randn(n, generator=g), torch.randn(n, generator=g)
    held = w.to(DEV)
    p = held.bfloat16() if masters else held
    m, v, s = (None if t is None else t.to(DEV) for t in pc.adamw_new_state(torch.empty(n), bits))
    pc.adamw_step([p], [grad.to(DEV).to(p.dtype)], [m], [v], torch.zeros(1, dtype=torch.int64, device=DEV), lr=lr,
                  weight_decay=decay, masters=[held] if masters else None, scales=None if s is None else [s])
    g32 = grad.to(p.dtype).double()
    step = lr * g32 / (g32.abs() + 1e-8)
    want = w.double() * (1 - lr * decay) - step
    tol = want.abs() * 2.0 ** -24 * (1 + 2.0 ** -20) + 16 * 2.0 ** -24 * (step.abs() + lr * decay * w.double().abs())
    error = (held.cpu().double() - want).abs()
    assert (error <= tol).all(), (int((error > tol).sum()), float((error / tol).max()))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("decay", [0.0, 0.1])
def test_infinite_weights_stay_infinite(decay, bits):
    p = torch.ones(300, device=DEV)
    p[3], p[270] = float("inf"), float("-inf")
    m, v, s = (None if t is None else t.to(DEV) for t in pc.adamw_new_state(torch.empty(300), bits))
    pc.adamw_step([p], [torch.ones_like(p)], [m], [v], torch.zeros(1, dtype=torch.int64, device=DEV), lr=0.1,
                  weight_decay=decay, scales=None if s is None else [s])
    assert p[3] == float("inf") and p[270] == -float("inf")
    p[3] = p[270] = 0.0
    assert p.isfinite().all()
