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


# ------------------------------------------------------------------ optimizer

def pair(bits, n=1000, **kw):
    """Two parameters of the same values, and the optimizer of them."""
    w = torch.randn(n, generator=gen(2))
    params = [torch.nn.Parameter(w.to(DEV)) for _ in range(2)]
    return params, pc.ParaboloidAdamW(params, lr=1e-2, state_bits=bits, seed=7, **kw)


def give(params, on, grad):
    for p, g in zip(params, on):
        p.grad = grad.clone() if g else None


@pytest.mark.parametrize("bits", [32, 8])
def test_a_count_is_not_split_in_a_capture(bits):
    """A parameter that lost its gradient since the first step would need a count of its own, which a graph would start
    from the same number at every replay: refused; after a step outside it can be captured."""
    (a, b), opt = pair(bits)
    grad = torch.randn(1000, generator=gen(3)).to(DEV)
    give((a, b), (1, 1), grad)
    opt.step()
    b.grad = None
    with pytest.raises(RuntimeError, match="captur"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    opt.step()
    assert opt.state[a]["step"].tolist() == [2] and opt.state[b]["step"].tolist() == [1]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        graph.replay()
    (c, d), eager = pair(bits)
    give((c, d), (1, 1), grad)
    eager.step()
    d.grad = None
    for _ in range(4):
        eager.step()
    assert opt.state[a]["step"].tolist() == eager.state[c]["step"].tolist() == [5]
    assert opt.state[b]["step"].tolist() == [1]
    assert torch.equal(a, c) and torch.equal(b, d)


@pytest.mark.parametrize("bits", [32, 8])
def test_no_state_is_made_in_a_capture(bits):
    """A graph would clear the moments at every replay."""
    (a, b), opt = pair(bits)
    grad = torch.ones(1000, device=DEV)
    give((a, b), (1, 1), grad)
    with pytest.raises(RuntimeError, match="captur"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    give((a, b), (1, 0), grad)
    opt.step()
    give((a, b), (1, 1), grad)
    with pytest.raises(RuntimeError, match="captur"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    opt.step()
    assert opt.state[a]["step"].tolist() == [2] and opt.state[b]["step"].tolist() == [1]
