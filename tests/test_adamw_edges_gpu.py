"""The AdamW step on the GPU: small decays, infinite weights, and the optimizer's
counts and random numbers."""
import copy

import pytest
import torch

import train_ref as ref
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


def codes_of(params, opt):
    return [[opt.state[p][k].cpu() for k in ("exp_avg", "exp_avg_sq", "scales")] for p in params]


@pytest.mark.parametrize("how", ["together", "one by one", "groups"])
def test_random_numbers_belong_to_the_parameter(how):
    """Each parameter's moments are rounded by the numbers of its place among all parameters, whichever others a step
    takes and whatever group it is in."""
    (a, b), opt = pair(8)
    if how == "groups":
        opt = pc.ParaboloidAdamW([{"params": [a]}, {"params": [b], "weight_decay": 0.0}], lr=1e-2, state_bits=8, seed=7)
    grad = torch.randn(1000, generator=gen(4))
    for on in ((1, 0), (0, 1)) if how == "one by one" else ((1, 1),):
        give((a, b), on, grad.to(DEV))
        opt.step()
    new = [pc.adamw_new_state(torch.empty(1000), 8) for _ in range(2)]
    c = dict(params=[a.detach().cpu()] * 2, grads=[grad] * 2, masters=None, m=[s[0] for s in new], v=[s[1] for s in new],
             scales=[s[2] for s in new])
    want = ref.adamw(c, 1, lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, seed=7)
    got = codes_of((a, b), opt)
    for (m, v, s), w in zip(got, want):
        assert torch.equal(m, w["m_code"]) and torch.equal(v, w["v_code"]) and torch.equal(s, w["scales"])
    assert not torch.equal(got[0][0], got[1][0]) and not torch.equal(got[0][1], got[1][1])


@pytest.mark.parametrize("bits", [32, 8])
def test_a_checkpoint_of_counts_that_met(bits):
    """Parameters that missed different steps and have equal counts go on alike, reloaded or not."""
    grads = torch.randn(8, 1000, generator=gen(5)).to(DEV)

    def run(params, opt, steps):
        for i, on in steps:
            give(params, on, grads[i])
            opt.step()

    params, opt = pair(bits)
    run(params, opt, [(0, (1, 0)), (1, (0, 1))])
    values, kept = [p.detach().clone() for p in params], copy.deepcopy(opt.state_dict())
    more = [(i, (1, 1)) for i in range(2, 6)]
    run(params, opt, more)
    others, opt2 = pair(bits)
    with torch.no_grad():
        for p, v in zip(others, values):
            p.copy_(v)
    opt2.load_state_dict(kept)
    run(others, opt2, more)
    for p, q in zip(params, others):
        assert torch.equal(p, q)
        for k in opt.state[p]:
            assert torch.equal(opt.state[p][k], opt2.state[q][k]), k


def test_numbers_of_the_function():
    """adamw_step's own numbers: the list's places unless given."""
    n = 600
    grad = torch.randn(n, generator=gen(6))

    def call(**kw):
        states = [[t.to(DEV) for t in pc.adamw_new_state(torch.empty(n), 8)] for _ in range(3)]
        pc.adamw_step([torch.zeros(n, device=DEV) for _ in range(3)], [grad.to(DEV)] * 3, [s[0] for s in states],
                      [s[1] for s in states], torch.zeros(1, dtype=torch.int64, device=DEV), lr=0.1,
                      scales=[s[2] for s in states], seed=3, **kw)
        return [s[0].cpu() for s in states]

    plain, moved = call(), call(numbers=[2, 7, 0])
    assert torch.equal(moved[0], plain[2]) and torch.equal(moved[2], plain[0])
    low = ref.adamw_random(n, 3, 1, 7)[0]
    want, _ = ref.adamw_encode((grad * float(torch.tensor(1 - 0.9))).double(), low, True)
    assert torch.equal(moved[1], want)
    for bad in ([0, 1], [0, 1, -1], [0, 1, 2 ** 31]):
        with pytest.raises((RuntimeError, ValueError)):
            call(numbers=bad)
