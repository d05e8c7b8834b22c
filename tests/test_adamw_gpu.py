"""The AdamW step on the GPU against its formulas in 64 bits on the CPU."""
import math

import pytest
import torch

import train_ref as ref
import paraconv2d_b200 as pc
from paraconv2d_b200.optim import ParaboloidAdamW

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def case(sizes, ptype, gtype, bits, masters, seed=0, spread=1e3):
    g = gen(seed)
    c = dict(params=[], grads=[], m=[], v=[], masters=[] if masters else None, scales=[] if bits == 8 else None)
    for n in sizes:
        w = torch.randn(n, generator=g) * 0.1
        size = torch.exp(torch.rand(n, generator=g) * math.log(spread) - math.log(spread)) * 0.1
        c["params"].append(w.to(ptype))
        if masters:
            c["masters"].append(w.clone())
        c["grads"].append((torch.randn(n, generator=g) * size).to(gtype))
        m, v = torch.randn(n, generator=g) * size, (size * torch.rand(n, generator=g)) ** 2
        if bits == 8:
            mc, ms = ref.adamw_encode(m.double(), [128] * n, True)
            vc, vs = ref.adamw_encode(v.double(), [128] * n, False)
            m, v = mc, vc
            c["scales"].append(torch.stack([ms, vs], 1))
        c["m"].append(m)
        c["v"].append(v)
    return c


def to(c, dev):
    return {k: None if v is None else [t.to(dev, copy=True) for t in v] for k, v in c.items()}


HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.2)


def step_both(c, t0, seed, factors=None, grad_scale=None, lr=None):
    """The call on the GPU, and the formulas' values for the same inputs."""
    d = to(c, DEV)
    step = torch.tensor([t0], device=DEV)
    scale = None if grad_scale is None else torch.tensor([grad_scale], device=DEV)
    hyper = dict(HYPER)
    want = ref.adamw(c, t0 + 1, seed=seed, factors=factors, grad_scale=grad_scale, **hyper)
    if lr is not None:
        hyper["lr"] = lr
    pc.adamw_step(d["params"], d["grads"], d["m"], d["v"], step, masters=d["masters"], scales=d["scales"],
                  factors=factors, grad_scale=scale, seed=seed, **hyper)
    assert step.tolist() == [t0 + 1]
    return {k: None if v is None else [t.cpu() for t in v] for k, v in d.items()}, want


def close(got, want, magnitude, roundings):
    """Off by at most so many roundings of 32 bits of the magnitude, and one of the type."""
    tol = magnitude * roundings * 2.0 ** -24
    if got.dtype != torch.float32:
        tol = tol + want.abs() * (torch.finfo(got.dtype).eps / 2 + 2.0 ** -20)
        tol = tol + (2.0 ** -25 if got.dtype == torch.float16 else 0)  # half a step of its subnormal numbers
    bad = (got.double() - want).abs() > tol + 1e-38
    assert not bad.any(), (got[bad][:4], want[bad][:4], tol[bad][:4])


def check(got, want, c):
    for i in range(len(c["params"])):
        w = want[i]
        held = got["masters"][i] if got["masters"] else got["params"][i]
        # weight and step: the decay's product, the step's quotient, root and factors (8) and the last difference
        close(held, w["param"], w["param_size"], 12)
        if got["masters"]:
            assert torch.equal(got["params"][i], held.to(got["params"][i].dtype))
        if got["scales"] is None:
            close(got["m"][i], w["m"], w["m_size"], 3)
            close(got["v"][i], w["v"], w["v_size"], 4)
        else:
            # the codes are those of 32-bit products and sums: whole numbers
            assert torch.equal(got["scales"][i], w["scales"])
            assert torch.equal(got["m"][i], w["m_code"]) and torch.equal(got["v"][i], w["v_code"])


SIZES = [1, 3, 255, 256, 257, 0, 1000, 8192, 8193, 20000]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("ptype,gtype,masters", [
    (torch.float32, torch.float32, False), (torch.bfloat16, torch.bfloat16, False),
    (torch.bfloat16, torch.float32, True), (torch.float16, torch.float16, True), (torch.float16, torch.float32, False)])
def test_step(bits, ptype, gtype, masters):
    c = case(SIZES, ptype, gtype, bits, masters, seed=1)
    got, want = step_both(c, 6, 123456789012345, grad_scale=0.7)
    check(got, want, c)


@pytest.mark.parametrize("bits", [32, 8])
def test_first_step_from_nothing(bits):
    c = case([300, 7], torch.float32, torch.float32, bits, False, seed=2)
    for i, n in enumerate((300, 7)):
        m, v, s = pc.optim.adamw_new_state(torch.empty(n), bits)
        c["m"][i], c["v"][i] = m, v
        if s is not None:
            c["scales"][i] = s
    got, want = step_both(c, 0, -5)
    check(got, want, c)


@pytest.mark.parametrize("bits", [32, 8])
def test_factors_and_device_rate(bits):
    c = case([100, 513, 40], torch.float32, torch.float32, bits, False, seed=3)
    got, want = step_both(c, 2, 7, factors=[(33, 1.0, 0.25, 0.0), None, (0, 5.0, 2.0, 0.5)],
                          lr=torch.tensor([3e-3], device=DEV))
    check(got, want, c)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_of_mixed_types(bits):
    """More tensors than a launch takes, of all types in one call."""
    parts = [case([5 + i % 300 for i in range(260)], t, t, bits, False, seed=4 + k) for k, t in enumerate(TYPES)]
    c = {}
    for k in parts[0]:
        c[k] = None if parts[0][k] is None else [t for three in zip(*(p[k] for p in parts)) for t in three]
    got, want = step_both(c, 1, 11)
    check(got, want, c)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("shift", [1, 2, 3])
def test_views_off_a_boundary(bits, shift):
    c = case([700], torch.bfloat16, torch.bfloat16, bits, False, seed=5)
    d = to(c, DEV)

    def moved(t):
        base = torch.zeros(t.numel() + shift, dtype=t.dtype, device=DEV)
        base[shift:] = t
        return base[shift:]

    for k in ("params", "grads", "m", "v"):
        d[k] = [moved(t) for t in d[k]]
    step = torch.tensor([4], device=DEV)
    pc.adamw_step(d["params"], d["grads"], d["m"], d["v"], step, scales=d["scales"], seed=1, **HYPER)
    want = ref.adamw(c, 5, seed=1, **HYPER)
    check({k: None if v is None else [t.cpu() for t in v] for k, v in d.items()}, want, c)


def test_orders_of_dimensions():
    """A channels-last parameter, its state in the same order and a gradient in the usual one."""
    g = gen(6)
    w, gr = torch.randn(4, 6, 3, 3, generator=g), torch.randn(4, 6, 3, 3, generator=g)
    p = w.to(DEV).to(memory_format=torch.channels_last)
    m, v, _ = pc.optim.adamw_new_state(p)
    assert m.stride() == p.stride()
    pc.adamw_step([p], [gr.to(DEV)], [m], [v], torch.zeros(1, dtype=torch.int64, device=DEV), **HYPER)
    c = dict(params=[w.flatten()], grads=[gr.flatten()], m=[torch.zeros(w.numel())], v=[torch.zeros(w.numel())],
             masters=None, scales=None)
    want = ref.adamw(c, 1, **HYPER)[0]
    close(p.cpu().flatten(), want["param"], want["param_size"], 12)
    close(m.cpu().flatten(), want["m"], want["m_size"], 3)


@pytest.mark.parametrize("bits", [32, 8])
def test_values_that_are_not_finite(bits):
    """They reach their own element, and in 8 bits the states of their 256."""
    c = case([600], torch.float32, torch.float32, bits, False, seed=8)
    c["grads"][0][300] = float("inf")
    c["grads"][0][520] = float("nan")
    got, want = step_both(c, 3, 9)
    fine = torch.ones(600, dtype=torch.bool)
    fine[[300, 520]] = False
    close(got["params"][0][fine], want[0]["param"][fine], want[0]["param_size"][fine], 12)
    assert got["params"][0][520].isnan()
    if bits == 32:
        assert got["m"][0][300].isinf() and got["v"][0][520].isnan()
        assert got["m"][0][fine].isfinite().all()
    else:
        assert got["scales"][0][:, 0].tolist()[1:] == [255, 255] and got["scales"][0][0, 0] < 255
        m, v = pc.adamw_state_values(*([t.to(DEV) for t in got[k]] for k in ("m", "v", "scales")))
        assert m[0][:256].isfinite().all() and m[0][256:].isnan().all() and v[0][256:].isnan().all()


def test_values_of_8_bit_states():
    """Every code under several exponents, in both types."""
    codes = torch.arange(256, dtype=torch.uint8).repeat(5)
    E = torch.tensor([1, 2, 100, 220, 255], dtype=torch.uint8)
    scales = torch.stack([E, E], 1)
    want_m, want_v = ref.adamw_decode(codes, E, True), ref.adamw_decode(codes, E, False)
    for dtype in (torch.float32, torch.bfloat16):
        m, v = pc.adamw_state_values([codes.to(DEV)], [codes.to(DEV)], [scales.to(DEV)], dtype=dtype)
        assert m[0].dtype == dtype
        # (exponents that a block's largest value cannot have give infinities)
        assert torch.equal(m[0].cpu().double().nan_to_num(7.0), want_m.to(dtype).double().nan_to_num(7.0))
        ok = want_v < 1e38
        assert torch.equal(v[0].cpu().double()[ok], want_v[ok])


def test_rounding_is_unbiased_and_moves_on():
    """A second moment of 8 bits follows a gradient that a rounding to nearest would not let it."""
    n = 256 * 64
    m, v, s = (t.to(DEV) for t in pc.optim.adamw_new_state(torch.empty(n), 8))
    p, g = torch.zeros(n, device=DEV), torch.full((n,), 0.5, device=DEV)
    step = torch.zeros(1, dtype=torch.int64, device=DEV)
    for _ in range(200):
        pc.adamw_step([p], [g], [m], [v], step, lr=0.0, betas=(0.9, 0.999), scales=[s], seed=3)
    values = pc.adamw_state_values([m], [v], [s])
    want = 0.25 * (1 - 0.999 ** 200)
    # the mean of n values, each off by a walk of 200 roundings with a spread below 2^-4 of it: six times that of the mean
    assert abs(float(values[1][0].double().mean()) / want - 1) < 6 * (2 ** -4) * 200 ** 0.5 / n ** 0.5
    assert abs(float(values[0][0].double().mean()) / 0.5 - 1) < 6 * (2 ** -4) * 200 ** 0.5 / n ** 0.5


def test_refusals():
    p = torch.zeros(512, device=DEV)
    g, m, v = torch.zeros_like(p), torch.zeros_like(p), torch.zeros_like(p)
    step = torch.zeros(1, dtype=torch.int64, device=DEV)

    def call(params=None, grads=None, ms=None, vs=None, st=step, **kw):
        pc.adamw_step([p] if params is None else params, [g] if grads is None else grads, [m] if ms is None else ms,
                      [v] if vs is None else vs, st, **{"lr": 1e-3, **kw})

    call()
    for bad in (dict(grads=[g, g]), dict(grads=[g.double()]), dict(grads=[g[:100]]), dict(ms=[m.bfloat16()]),
                dict(params=[p.double()]), dict(params=[p[::2]], grads=[g[::2]], ms=[m[::2]], vs=[v[::2]]),
                dict(grads=[p]), dict(ms=[v]), dict(params=[p, p], grads=[g, g], ms=[m, m.clone()], vs=[v, v.clone()]),
                dict(st=step.int()), dict(st=step.cpu()), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0),
                dict(weight_decay=float("nan")), dict(masters=[p.clone()]), dict(scales=[p]),
                dict(lr=torch.tensor(1e-3)), dict(grad_scale=torch.ones(2, device=DEV)),
                dict(factors=[(0, float("inf"), 1.0, 1.0)]), dict(factors=[None, (1, 1.0, 1.0, 1.0)]),
                dict(factors=[(-1, 1.0, 1.0, 1.0)]), dict(ms=[m.view(2, 256)])):
        with pytest.raises((RuntimeError, ValueError, NotImplementedError)):
            call(**bad)
    assert step.tolist() == [1]
    codes = [torch.zeros(512, dtype=torch.uint8, device=DEV) for _ in range(2)]
    with pytest.raises(RuntimeError):
        call(ms=codes[:1], vs=codes[1:])
    with pytest.raises(RuntimeError):
        call(ms=codes[:1], vs=codes[1:], scales=[torch.zeros(1, 2, dtype=torch.uint8, device=DEV)])
    call(params=[p.bfloat16()], grads=[g], masters=[p], ms=[m], vs=[v])
    pc.adamw_step([], [], [], [], step, lr=1e-3)


# ------------------------------------------------------------------ optimizer

def small_model(seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(pc.ParaConv2d(3, 8, 3, padding=1, h_lr_factor=0.5, p_lr_factor=2.0, wd_factor=0.25),
                               torch.nn.Flatten(1), torch.nn.Linear(8 * 36, 5)).to(DEV)


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_against_formulas(bits):
    model = small_model()
    opt = ParaboloidAdamW(model.parameters(), lr=1e-2, weight_decay=0.3, state_bits=bits, seed=5)
    x = torch.randn(4, 3, 6, 6, device=DEV)
    tags = next(p for p in model.parameters() if getattr(p, "isParaboloid", False))
    m, d = pc.optim.paraboloid_split(tags)
    for t in range(1, 4):
        opt.zero_grad()
        model(x).square().sum().backward()
        params = list(model.parameters())
        c = dict(params=[p.detach().cpu().flatten() for p in params], grads=[p.grad.cpu().flatten() for p in params],
                 masters=None, scales=None)
        for k, name in (("m", "exp_avg"), ("v", "exp_avg_sq")):
            c[k] = [(opt.state[p][name].cpu() if t > 1 else pc.optim.adamw_new_state(p.cpu().detach(), bits)[k == "v"])
                    .flatten() for p in params]
        if bits == 8:
            c["scales"] = [opt.state[p]["scales"].cpu() if t > 1 else
                           pc.optim.adamw_new_state(p.cpu().detach(), bits)[2] for p in params]
        factors = [(m * (1 + d), 0.5, 2.0, 0.25) if p is tags else None for p in params]
        opt.step()
        want = ref.adamw(c, t, lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.3, factors=factors, seed=5)
        for p, w in zip(params, want):
            close(p.detach().cpu().flatten(), w["param"], w["param_size"], 12)


@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoint_goes_on(bits):
    """A reloaded optimizer takes the same steps, 16-bit parameters with masters among them."""
    def build():
        torch.manual_seed(1)
        net = torch.nn.Sequential(torch.nn.Linear(40, 300), torch.nn.Linear(300, 7).bfloat16()).to(DEV)
        return net, ParaboloidAdamW(net.parameters(), lr=1e-2, state_bits=bits, masters=True, seed=2)

    def train(net, opt, seeds):
        for s in seeds:
            torch.manual_seed(s)
            for p in net.parameters():
                p.grad = torch.randn_like(p)
            opt.step()

    net, opt = build()
    train(net, opt, range(3))
    kept = {k: v.clone() for k, v in net.state_dict().items()}, opt.state_dict()
    import copy
    kept = copy.deepcopy(kept)
    train(net, opt, range(3, 6))
    net2, opt2 = build()
    net2.load_state_dict(kept[0])
    opt2.load_state_dict(kept[1])
    states = [opt2.state[p] for p in net2.parameters()]
    assert all(s["step"] is states[0]["step"] for s in states)
    assert states[2]["master"].dtype == torch.float32
    train(net2, opt2, range(3, 6))
    for a, b in zip(net.parameters(), net2.parameters()):
        assert torch.equal(a, b)
        for k in opt.state[a]:
            assert torch.equal(opt.state[a][k], opt2.state[b][k]), k


def test_parameters_without_gradients_keep_their_own_count():
    a, b = (torch.nn.Parameter(torch.ones(10, device=DEV)) for _ in range(2))
    opt = ParaboloidAdamW([a, b], lr=1e-2)
    for grads in ((1, 1), (1, 0), (1, 1), (0, 1)):
        for p, on in zip((a, b), grads):
            p.grad = torch.ones_like(p) if on else None
        opt.step()
    assert opt.state[a]["step"].tolist() == [3] and opt.state[b]["step"].tolist() == [3]
    assert torch.equal(a, b)  # the same three steps


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step(bits):
    """A replayed step counts on, follows a rate on the GPU, and equals eager steps."""
    def build():
        torch.manual_seed(3)
        p = torch.nn.Parameter(torch.randn(1000, device=DEV))
        p.grad = torch.randn(1000, device=DEV)
        lr = torch.tensor([1e-2], device=DEV)
        return p, lr, ParaboloidAdamW([p], lr=lr, state_bits=bits)

    p, lr, opt = build()
    q, lr2, opt2 = build()
    opt.step()
    opt2.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for i in range(3):
        for r in (lr, lr2):
            r.fill_(1e-2 / (i + 1))
        graph.replay()
        opt2.step()
    assert torch.equal(p, q) and opt.state[p]["step"].tolist() == [4]


def test_other_stream_and_closed_over_version():
    p = torch.nn.Parameter(torch.randn(5000, device=DEV))
    p.grad = torch.randn_like(p)
    opt = ParaboloidAdamW([p], lr=1e-2)
    y = (p * p).sum()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        opt.step()
    torch.cuda.current_stream().wait_stream(stream)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
