"""Linear attention on the GPU against its recurrence in 64 bits on the CPU."""
import math

import pytest
import torch

import train_ref as ref
import paraconv2d_b200 as pc

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16

# Scores and states meet the inputs as one number of 8 bits of mantissa (off by 2^-8 of itself at most) for
# bfloat16, two (2^-16, and the states' part likewise) for float16, three for float32.
PARTS = {BF16: 2.0 ** -8, F16: 2.0 ** -15, F32: 2.0 ** -22}
# The decays' gradients take the states as two or three of them.
DECAY_PARTS = {BF16: 2.0 ** -15, F16: 2.0 ** -14, F32: 2.0 ** -22}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def inputs(B, H, G, dk, dv, L, dtype, tokens, seed, low=1e-3, high=2.0, init=False):
    g = gen(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = dict(q=r(B, G, dk, L).to(dtype), k=(r(B, G, dk, L) * dk ** -0.5).to(dtype), v=r(B, H, dv, L).to(dtype))
    u = torch.rand(*((B, H, L) if tokens else (H,)), generator=g)
    t["g"] = -torch.exp(math.log(low) + u * math.log(high / low))
    t["init"] = r(B, H, dk, dv) if init else None
    return t, r(B, H, dv, L).to(dtype), r(B, H, dk, dv)


def close(got, want, size, part, steps, what):
    # beside the parts: 32-bit roundings of a chunk's products and exponentials, and one a chunk of the states
    tol = size * (part + (64 + steps) * 2.0 ** -24)
    if got.dtype != F32:
        tol = tol + want.abs() * torch.finfo(got.dtype).eps / 2 + (2.0 ** -25 if got.dtype == F16 else 0)
    bad = (got.detach().cpu().double() - want).abs() > tol + 1e-30
    assert not bad.any(), (what, int(bad.sum()), got.detach().cpu()[bad][:3], want[bad][:3], tol[bad][:3])


def check(B, H, G, dk, dv, L, dtype, tokens=True, init=False, lengths=None, seed=0, train=True, scale=None, low=1e-3,
          high=2.0, nan_behind=True):
    t, go, gf = inputs(B, H, G, dk, dv, L, dtype, tokens, seed, low, high, init)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    d = {k: None if x is None else x.to(DEV) for k, x in t.items()}
    god = go.to(DEV)
    if n is not None and nan_behind:  # what lies behind the tokens is not read
        for i, m in enumerate(lengths):
            for x in (d["q"], d["k"], d["v"], god) + ((d["g"],) if tokens else ()):
                x[i, ..., max(m, 0):] = float("nan")
    leaves = [x for x in d.values() if x is not None]
    if train:
        for x in leaves:
            x.requires_grad_(True)
    out, final = pc.linear_attention(d["q"], d["k"], d["v"], d["g"], scale=scale, initial_state=d["init"],
                                     lengths=None if n is None else n.to(DEV), return_final_state=True)
    chunk = 64 if dtype == BF16 else 32
    v, m = ref.attention(**t, scale=scale, lengths=lengths, grad=go if train else None, grad_final=gf, chunk=chunk)
    steps = L // chunk
    close(out, v["out"], m["out"], PARTS[dtype], steps, "out")
    close(final, v["final"], m["final"], 2.0 ** -22, steps, "final")
    if not train:
        return
    grads = dict(zip([k for k, x in d.items() if x is not None],
                     torch.autograd.grad([out, final], leaves, [god, gf.to(DEV)])))
    # a gradient meets a score and a state, each in parts
    for name, key in (("q", "dq"), ("k", "dk"), ("v", "dv")):
        close(grads[name], v[key], m[key], PARTS[dtype], steps, key)
    if init:
        close(grads["init"], v["dinit"], m["dinit"], 2.0 ** -22, steps, "dinit")
    dg, mg = (v["dg"], m["dg"]) if tokens else (v["dg"].sum((0, 2)), m["dg"].sum((0, 2)))
    close(grads["g"], dg, mg, DECAY_PARTS[dtype], steps, "dg")
    if n is not None:
        for i, m in enumerate(lengths):
            for x in (out, grads["q"], grads["k"], grads["v"]) + ((grads["g"],) if tokens else ()):
                assert not x[i, ..., max(m, 0):].any()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dims", [(1, 1, 1, 1, 1, 1), (1, 2, 2, 16, 16, 64), (2, 2, 1, 8, 24, 65), (1, 3, 3, 64, 64, 130),
                                  (1, 2, 1, 128, 128, 96), (2, 4, 2, 33, 65, 40), (1, 2, 2, 100, 17, 200),
                                  (1, 1, 1, 15, 128, 31), (3, 2, 1, 48, 80, 77)])
def test_shapes(dims, dtype):
    check(*dims, dtype, tokens=True, init=sum(dims) % 2 == 0, seed=sum(dims))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens", [False, True])
def test_decays_and_scale(tokens, dtype):
    check(2, 3, 3, 32, 32, 150, dtype, tokens=tokens, init=True, seed=1, scale=0.3)
    check(1, 2, 2, 32, 32, 150, dtype, tokens=tokens, seed=2, low=2.0, high=30.0)   # strong ones
    check(1, 2, 2, 32, 32, 150, dtype, tokens=tokens, seed=3, low=1e-6, high=1e-4)  # hardly any


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lengths", [[70, 0, 1, 64, 65], [0, 0, 0, 0, 0], [-3, 1000, 70, 33, 2]])
def test_lengths(lengths, dtype):
    check(5, 2, 1, 24, 40, 70, dtype, init=True, lengths=lengths, seed=4)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("train", [False, True])
def test_few_heads_by_segments(dtype, train):
    """A long sequence of few heads goes by segments, whose states are carried."""
    check(1, 2, 1, 32, 48, 1111, dtype, init=True, seed=5, train=train, low=1e-4, high=1e-1)
    check(2, 1, 1, 16, 16, 1024, dtype, init=True, seed=6, train=train, lengths=[1024, 300], tokens=False)


def test_forgetting():
    """Decays of -inf: a token sees nothing from before it, itself in full."""
    t, go, gf = inputs(1, 2, 2, 16, 16, 100, F32, True, 7, init=True)
    at = [0, 5, 31, 32, 70, 71, 99]
    t["g"][:, 1, at] = float("-inf")
    t["g"][:, 0, 40:60] = float("-inf")
    v, m = ref.attention(**t, grad=go, grad_final=gf, chunk=32)
    d = {k: x.to(DEV).requires_grad_(True) for k, x in t.items()}
    out, final = pc.linear_attention(d["q"], d["k"], d["v"], d["g"], initial_state=d["init"], return_final_state=True)
    grads = torch.autograd.grad([out, final], list(d.values()), [go.to(DEV), gf.to(DEV)])
    close(out, v["out"], m["out"], PARTS[F32], 4, "out")
    close(final, v["final"], m["final"], 2.0 ** -22, 4, "final")
    for x, key in zip(grads, ("dq", "dk", "dv", "dg", "dinit")):
        close(x, v[key], m[key], PARTS[F32], 4, key)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_large_states(dtype):
    """States beyond float16's range."""
    t, go, gf = inputs(1, 1, 1, 16, 16, 200, dtype, False, 8, low=1e-6, high=1e-5)
    t["k"], t["v"] = (torch.full_like(t[n], 100.0) for n in "kv")
    t["q"] = t["q"] * 2 ** -10
    v, m = ref.attention(**t)
    assert float(v["final"].max()) > 1e6
    d = {k: None if x is None else x.to(DEV) for k, x in t.items()}
    out, final = pc.linear_attention(d["q"], d["k"], d["v"], d["g"], return_final_state=True)
    close(out, v["out"], m["out"], PARTS[dtype], 6, "out")
    close(final, v["final"], m["final"], 2.0 ** -22, 6, "final")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("name", ["q", "k", "v", "g"])
def test_values_that_are_not_finite_reach_no_earlier_token(name, value, dtype):
    t, _, _ = inputs(1, 2, 2, 32, 32, 150, dtype, True, 9)
    v, m = ref.attention(**t)  # of the finite values; the sums near the value go by another order: not the same bits
    d = {k: None if x is None else x.to(DEV) for k, x in t.items()}
    if name == "g":
        d["g"][0, 1, 90] = float("nan")
    else:
        d[name][0, 1, 3, 90] = value
    out = pc.linear_attention(d["q"], d["k"], d["v"], d["g"])
    fine = torch.ones(v["out"].shape, dtype=torch.bool)
    fine[0, 1, 3 if name == "v" else slice(None), 90:] = False  # (an infinity in v: nor another of the values)
    close(out.cpu()[fine], v["out"][fine], m["out"][fine], PARTS[dtype], 4, name)
    assert not out[0, 1, 3, 90].isfinite()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradients_that_are_not_finite_reach_no_later_token(dtype):
    """The gradient of a token's output reaches the keys and values up to it, and its own query."""
    t, go, _ = inputs(1, 1, 1, 32, 32, 150, dtype, True, 10)
    v, m = ref.attention(**t, grad=go, chunk=64 if dtype == BF16 else 32)
    d = {k: None if x is None else x.to(DEV).requires_grad_(True) for k, x in t.items()}
    leaves = [d[n] for n in ("q", "k", "v", "g")]
    god = go.to(DEV)
    god[0, 0, 3, 90] = float("inf")
    grads = torch.autograd.grad(pc.linear_attention(*leaves), leaves, god)
    for g, key in zip(grads, ("dq", "dk", "dv", "dg")):
        fine = torch.ones(v[key].shape, dtype=torch.bool)
        if key == "dq":
            fine[..., 90] = False
        elif key == "dv":
            fine[0, 0, 3, :91] = False
        else:
            fine[..., :91] = False
        close(g.cpu()[fine], v[key][fine], m[key][fine], (DECAY_PARTS if key == "dg" else PARTS)[dtype], 4, key)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_steps_go_on_from_a_prompt(dtype):
    """A prompt and then single tokens equal the whole sequence."""
    t, _, _ = inputs(3, 4, 2, 40, 24, 90, dtype, True, 11, init=True)
    v, m = ref.attention(**t)
    d = {k: x.to(DEV) for k, x in t.items()}
    out, state = pc.linear_attention(d["q"][..., :70], d["k"][..., :70], d["v"][..., :70], d["g"][..., :70],
                                     initial_state=d["init"], return_final_state=True)
    places = torch.zeros(5, 4, 40, 24, device=DEV)
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device=DEV)
    places[slots.long()] = state
    for i in range(70, 90):
        o = pc.linear_attention_step(d["q"][..., i], d["k"][..., i], d["v"][..., i], d["g"][..., i], places, slots=slots)
        close(o, v["out"][..., i], m["out"][..., i], 2.0 ** -22, 24, i)
    close(places[slots.long()], v["final"], m["final"], 2.0 ** -22, 24, "final")
    assert not places[[1, 3]].any()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dims", [(1, 1, 1, 1, 1), (2, 3, 3, 64, 64), (4, 4, 2, 128, 128), (3, 2, 1, 33, 65), (2, 2, 2, 100, 12),
                                  (1, 12, 4, 7, 128)])
def test_step(dims, dtype):
    B, H, G, dk, dv = dims
    t, _, _ = inputs(B, H, G, dk, dv, 1, dtype, B % 2 == 0, 12, init=True)
    v, m = ref.attention(**t)
    d = {k: x.to(DEV) for k, x in t.items()}
    g = d["g"][..., 0] if B % 2 == 0 else d["g"]
    out = pc.linear_attention_step(d["q"][..., 0], d["k"][..., 0], d["v"][..., 0], g, d["init"])
    close(out, v["out"][..., 0], m["out"][..., 0], 0, 0, "out")
    close(d["init"], v["final"], m["final"], 0, 0, "state")


def test_step_places():
    """Padding, places outside the array, and a place that an earlier row has."""
    B, H, dk, dv = 6, 2, 8, 8
    g = torch.zeros(H, device=DEV)
    q, k, v = (torch.ones(B, H, n, device=DEV) for n in (dk, dk, dv))
    state = torch.zeros(3, H, dk, dv, device=DEV)
    slots = torch.tensor([1, -1, 3, 1, -7, 0], dtype=torch.int32, device=DEV)
    out = pc.linear_attention_step(q, k, v, g, state, slots=slots)
    assert not out[1].any() and out[[2, 3, 4]].isnan().all() and out[[0, 5]].isfinite().all()
    assert state[0].eq(1).all() and state[1].eq(1).all() and not state[2].any()


def test_refusals():
    B, H, G, dk, dv, L = 2, 4, 2, 8, 16, 10
    z = lambda *s, **k: torch.zeros(*s, device=DEV, **k)  # noqa: E731
    good = dict(q=z(B, G, dk, L), k=z(B, G, dk, L), v=z(B, H, dv, L), log_decay=z(H))
    pc.linear_attention(**good)
    for bad in (dict(q=z(B, 3, dk, L), k=z(B, 3, dk, L)), dict(k=z(B, G, dk + 1, L)), dict(v=z(B, H, dv, L + 1)),
                dict(q=z(B, G, dk, L, dtype=F16)), dict(log_decay=z(H + 1)), dict(log_decay=z(B, H, L, dtype=BF16)),
                dict(log_decay=z(B, H)), dict(initial_state=z(B, H, dv, dk)), dict(lengths=z(B)), dict(scale=math.inf),
                dict(q=z(B, G, 129, L), k=z(B, G, 129, L)), dict(v=z(B, H, 129, L)), dict(v=z(B, H, 0, L)),
                dict(v=z(B, H, dv, L).double()), dict(k=torch.zeros(B, G, dk, L))):
        with pytest.raises((RuntimeError, NotImplementedError)):
            pc.linear_attention(**{**good, **bad})
    step = dict(q=z(B, G, dk), k=z(B, G, dk), v=z(B, H, dv), log_decay=z(H), state=z(B, H, dk, dv))
    pc.linear_attention_step(**step)
    for bad in (dict(state=z(1, H, dk, dv)), dict(state=z(B, H, dk, dv, dtype=F16)), dict(state=z(B, H, dv, dk).transpose(2, 3)),
                dict(slots=z(B)), dict(log_decay=z(B, H, 1)), dict(v=step["state"].view(-1)[:B * H * dv].view(B, H, dv)),
                dict(q=z(B, G, dk).requires_grad_(True))):
        with pytest.raises(RuntimeError):
            pc.linear_attention_step(**{**step, **bad})
    leaf = z(H).requires_grad_(True)
    (dg,) = torch.autograd.grad(pc.linear_attention(**{**good, "log_decay": leaf}).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        dg.sum().backward()


def test_empty():
    q = torch.zeros(0, 2, 8, 5, device=DEV)
    assert pc.linear_attention(q, q, q, torch.zeros(2, device=DEV)).shape == q.shape
    q = torch.zeros(3, 2, 8, 0, device=DEV, requires_grad=True)
    g = torch.zeros(2, device=DEV, requires_grad=True)
    init = torch.randn(3, 2, 8, 8, device=DEV, requires_grad=True)
    out, state = pc.linear_attention(q, q, q, g, initial_state=init, return_final_state=True)
    assert out.shape == q.shape and torch.equal(state, init)
    state.sum().backward()
    assert init.grad.eq(1).all() and not g.grad.any()


def test_strides_and_views():
    """[batch, length, heads, dim] tensors as views, and one off a vector's boundary."""
    t, _, _ = inputs(2, 2, 2, 32, 32, 72, BF16, True, 13)
    d = {k: None if x is None else x.to(DEV) for k, x in t.items()}
    want = pc.linear_attention(d["q"], d["k"], d["v"], d["g"])
    v = [d[n].permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1) for n in "qkv"]
    assert torch.equal(pc.linear_attention(*v, d["g"].transpose(1, 2).contiguous().transpose(1, 2)), want)
    base = torch.zeros(d["v"].numel() + 1, dtype=BF16, device=DEV)
    base[1:] = d["v"].flatten()
    assert torch.equal(pc.linear_attention(d["q"], d["k"], base[1:].view(d["v"].shape), d["g"]), want)


def test_gradient_against_differences():
    t, go, gf = inputs(1, 2, 1, 8, 8, 40, F32, True, 14, init=True)
    d = {k: x.to(DEV).requires_grad_(True) for k, x in t.items()}
    god, gfd = go.to(DEV), gf.to(DEV)

    def loss(d):
        out, final = pc.linear_attention(d["q"], d["k"], d["v"], d["g"], initial_state=d["init"], return_final_state=True)
        return (out * god).double().sum() + (final * gfd).double().sum()

    grads = dict(zip(d, torch.autograd.grad(loss(d), list(d.values()))))
    h = 2.0 ** -8
    for n, gr in grads.items():
        way = torch.randn(t[n].shape, generator=gen(15)).to(DEV)
        with torch.no_grad():
            ends = [loss({**d, n: d[n] + s * h * way}) for s in (1, -1)]
        slope = float(ends[0] - ends[1]) / (2 * h)
        # linear in all but the decays, whose third derivative along `way` is of the order of its gradient's terms
        assert abs(slope - float((gr * way).double().sum())) <= (4 * h * h + 2.0 ** -20 / h) * float((gr * way).abs().sum() + 10), n


@pytest.mark.parametrize("dims", [(2, 4, 2, 32, 32, 100), (1, 2, 2, 64, 64, 2048)])
def test_captured_on_another_stream(dims):
    """Two graphs of forward and backward passes that are replayed in turn equal eager calls."""
    stream = torch.cuda.Stream()
    graphs = []
    for seed in range(2):
        t, go, gf = inputs(*dims, BF16, True, 16 + seed, init=True)
        d = {k: x.to(DEV) for k, x in t.items()}
        god, gfd = go.to(DEV), gf.to(DEV)

        def both(d, god=god, gfd=gfd):
            leaves = [x.requires_grad_(True) for x in d.values()]
            outs = pc.linear_attention(*leaves[:4], initial_state=leaves[4], return_final_state=True)
            return [x.detach() for x in outs] + list(torch.autograd.grad(outs, leaves, [god, gfd]))

        want = [x.clone() for x in both({k: x.clone() for k, x in d.items()})]
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = both(d)
        graphs.append((graph, got, want, d, god, gfd))
    for _ in range(2):
        for graph, got, want, *_ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for graph, got, want, *_ in graphs:
        for a, b in zip(got, want):
            assert torch.equal(a, b)
