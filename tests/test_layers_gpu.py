"""The layers beside ParaConv2d on the GPU, against the 64-bit references of
layers_ref.py.

Tolerances.  An output is off by the one rounding to its type (half a unit in
the last place) plus `units` 32-bit roundings (2^-24) of the value's magnitude:

* dropout: scale, product, residual sum: 3.
* convolution: K products and sums (K + 1); silu adds exp (its argument's
  rounding and 3 units, at |pre| < 20: 23) and a division (4), and carries the
  sum's error with a slope of at most 1.1: 1.1 (K + 1) + 27 < 40 for K <= 8.
  Gradients use silu' with the same parts: 64.  dw sums up to 64 products in
  a lane, then 5 levels, then in 64 bits: 64 + 64 + 5 < 160.
* scan: a step's d is off by 4 units and what its argument's rounding makes of
  it (`weight`, taken from the case); a decay exp(d A) by 3 + |d A| e^-|dA|
  (2 + 4 weight) < 5 + 2 weight, d u B by 6 + 4 weight.  Each of L steps adds
  one such error to a state, and a backward chain a second one of L steps, the
  sums over states and channels (added pairwise, in order, by at most 12
  levels of up to 64 terms) 2 log and 64, gate and softplus' 40: for the
  forward pass (L + 4) (8 + 4 weight) + 64, twice that for gradients.
"""
import math

import pytest
import torch

import layers_ref as ref
import paraconv2d_b200 as pc
from paraconv2d_b200 import _lib

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def dev(t):
    return None if t is None else t.to(DEV)


def check(got, value, mag, units, what):
    e = ref.excess(got, value, mag, units)
    assert e <= 1, f"{what}: {e:.3g} times what is allowed"


# ------------------------------------------------------------------- dropout

@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 255, 4096, 5003])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout_and_its_gradients(dtype, n, residual):
    g = gen(n)
    p, seed, offset = 0.3, -(2 ** 61) + n, 2 ** 40 + 5
    x = ref.rand(g, n, dtype=dtype)
    res = ref.rand(g, n, dtype=dtype) if residual else None
    grad = ref.rand(g, n, dtype=dtype)
    keep, scale = ref.kept_mask(n, p, seed, offset), ref.keep_scale(p)
    key = torch.tensor([seed, offset], device=DEV)
    xd = dev(x).requires_grad_()
    rd = dev(res).requires_grad_() if residual else None
    out = pc.dropout(xd, p, key, residual=rd)
    want = torch.where(keep, x.double() * scale, 0.0)
    mag = want.abs()
    if residual:
        want, mag = want + res.double(), mag + res.double().abs()
    units = 3 if dtype != torch.float64 else 2.0 ** -27
    check(out, want, mag, units, "out")
    if not residual:
        assert torch.equal(out.detach().cpu() != 0, keep & (x != 0))
    grads = torch.autograd.grad(out, [xd, rd] if residual else [xd], dev(grad))
    dwant = torch.where(keep, grad.double() * scale, 0.0)
    check(grads[0], dwant, dwant.abs(), units, "dx")
    if residual:
        assert torch.equal(grads[1].cpu(), grad)


def test_dropout_drops_nan_and_infinity_and_keeps_the_ends_of_p():
    n = 4096
    keep = ref.kept_mask(n, 0.5, 3, 4)
    x = torch.where(keep, 1.0, torch.tensor([math.nan, math.inf, -math.inf, 7.0]).repeat(n // 4))
    key = torch.tensor([3, 4], device=DEV)
    out = pc.dropout(dev(x), 0.5, key).cpu()
    assert torch.equal(out, torch.where(keep, 2.0, 0.0))
    y = torch.randn(1001, device=DEV)
    assert torch.equal(pc.dropout(y, 0.0, key), y)
    assert torch.equal(pc.dropout(y, 1.0, key), torch.zeros_like(y))
    assert torch.equal(pc.dropout(y, 1.0, key, residual=y), y)
    assert pc.dropout(y[:0], 0.5, key).numel() == 0


def test_dropout_mask_is_the_same_for_all_types_and_layouts():
    key = torch.tensor([11, 12], device=DEV)
    ones = torch.ones(33, 65, device=DEV)
    want = pc.dropout(ones, 0.4, key) != 0
    for dtype in (torch.float64, torch.bfloat16, torch.float16):
        assert torch.equal(pc.dropout(ones.to(dtype), 0.4, key) != 0, want)
    # strided, and a view that starts off a vector boundary
    assert torch.equal(pc.dropout(torch.ones(65, 33, device=DEV).t(), 0.4, key) != 0, want)
    off = torch.ones(33 * 65 + 1, device=DEV, dtype=torch.float16)[1:].view(33, 65)
    assert torch.equal(pc.dropout(off, 0.4, key) != 0, want)
    # the share of kept elements: within 6 standard deviations
    n = 1 << 22
    share = (pc.dropout(torch.ones(n, device=DEV), 0.4, key) != 0).double().mean().item()
    q = 1 - round(0.4 * 65536) / 65536
    assert abs(share - q) < 6 * math.sqrt(q * (1 - q) / n)


def test_dropout_beyond_32_bit_offsets():
    n = (1 << 32) + 11
    x = torch.ones(n, dtype=torch.float16, device=DEV)
    out = pc.dropout(x, 0.25, torch.tensor([5, 6], device=DEV))
    for group in (0, (1 << 29) - 1, 1 << 29):  # of eight elements
        bits = [h >= round(0.25 * 65536) for h in ref.halves(group, 5, 6)][:n - 8 * group]
        assert (out[8 * group:8 * group + 8] != 0).tolist() == bits
    assert (out[8 * ((1 << 29) + 1):] != 0).tolist() == [h >= 16384 for h in ref.halves((1 << 29) + 1, 5, 6)][:3]


def test_dropout_module_counts_its_calls():
    m = pc.Dropout(0.5, seed=9).to(DEV)
    x = torch.ones(512, device=DEV)
    first, second = m(x), m(x)
    assert not torch.equal(first, second) and m.state.tolist() == [9, 2]
    assert torch.equal(first, pc.dropout(x, 0.5, torch.tensor([9, 0], device=DEV)))
    again = pc.Dropout(0.5).to(DEV)
    again.load_state_dict({"state": torch.tensor([9, 1])})
    assert torch.equal(again(x), second)
    # replays of a captured call go on counting
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = m(x)
    seen = []
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        seen.append(y.clone())
        assert torch.equal(y, pc.dropout(x, 0.5, torch.tensor([9, 3 + i], device=DEV)))
    assert not torch.equal(seen[0], seen[1]) and m.state.tolist() == [9, 6]


def test_dropout_refuses():
    x = torch.ones(4, device=DEV)
    key = torch.zeros(2, dtype=torch.int64, device=DEV)
    for bad in (lambda: pc.dropout(x, 0.5, key.cpu()), lambda: pc.dropout(x, 0.5, key[:1]),
                lambda: pc.dropout(x, 0.5, key.int()), lambda: pc.dropout(x, 2.0, key),
                lambda: pc.dropout(x, 0.5, key, residual=x[:3]), lambda: pc.dropout(x, 0.5, key, residual=x.half()),
                lambda: pc.dropout(x.int(), 0.5, key)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            bad()


# -------------------------------------------------------- causal convolution

def conv_case(seed, B, D, L, K, dtype, wdtype=None, bias=True, carried=True, lengths=None):
    g = gen(seed)
    wdtype = wdtype or dtype
    c = dict(x=ref.rand(g, B, D, L, dtype=dtype), w=ref.rand(g, D, K, dtype=wdtype, scale=0.7),
             bias=ref.rand(g, D, dtype=wdtype) if bias else None,
             init=ref.rand(g, B, D, K - 1, dtype=dtype) if carried else None)
    go, gf = ref.rand(g, B, D, L, dtype=dtype), ref.rand(g, B, D, K - 1, dtype=dtype)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    return c, go, gf, lens


def conv_check(c, go, gf, lens, silu):
    K = c["w"].shape[1]
    v, m = ref.conv(c["x"], c["w"], c["bias"], silu, c["init"], lens, go, gf)
    t = {k: dev(a) for k, a in c.items()}
    if lens is not None:  # what lies behind a row's tokens may be anything
        for b, n in enumerate(lens.tolist()):
            t["x"][b, :, max(0, n):] = math.nan
    leaves = {k: a.requires_grad_() for k, a in t.items() if a is not None}
    out, final = pc.causal_conv(t["x"], t["w"], t["bias"], activation="silu" if silu else None,
                                initial_state=t["init"], lengths=dev(lens), return_final_state=True)
    check(out, v["out"], m["out"], 40, "out")
    assert torch.equal(final.detach().cpu().double(), v["final"])
    grads = dict(zip(leaves, torch.autograd.grad([out, final], list(leaves.values()), [dev(go), dev(gf)])))
    names = dict(x="dx", w="dw", bias="db", init="dinit")
    for k, gr in grads.items():
        if gr.numel():
            check(gr, v[names[k]], m[names[k]], 64 if k in ("x", "init") else 160, names[k])
    assert grads["w"].dtype == c["w"].dtype
    with torch.no_grad():  # without autograd: the same values
        alone = pc.causal_conv(t["x"], t["w"], t["bias"], activation="silu" if silu else None,
                               initial_state=t["init"], lengths=dev(lens))
    assert torch.equal(alone, out)
    return grads


@pytest.mark.parametrize("K", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("L", [1, 2, 5, 8, 31, 264])
def test_conv_taps_and_lengths(K, L):
    conv_check(*conv_case(100 * K + L, 2, 3, L, K, torch.float32), silu=True)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("L", [3, 64, 257, 600, 2049])
@pytest.mark.parametrize("silu", [False, True])
def test_conv_types(dtype, L, silu):
    conv_check(*conv_case(L, 3, 5, L, 4, TYPES[dtype], bias=L != 64, carried=L != 257), silu=silu)


def test_conv_32_bit_weights_beside_16_bit_inputs():
    conv_check(*conv_case(5, 2, 9, 77, 4, torch.bfloat16, wdtype=torch.float32), silu=True)


@pytest.mark.parametrize("L,lengths", [(20, [20, 0, 1, 2, 3, 19]), (300, [0, 300, 257, 8, 256, 1000, -5]),
                                       (1, [0, 1])])
@pytest.mark.parametrize("K", [1, 2, 4, 8])
@pytest.mark.parametrize("carried", [False, True])
def test_conv_ragged_rows(L, lengths, K, carried):
    conv_check(*conv_case(L + K, len(lengths), 3, L, K, torch.float16, carried=carried, lengths=lengths), silu=True)


def test_conv_empty():
    w = torch.randn(3, 4, device=DEV, requires_grad=True)
    init = torch.randn(2, 3, 3, device=DEV, requires_grad=True)
    out, final = pc.causal_conv(torch.zeros(2, 3, 0, device=DEV), w, initial_state=init, return_final_state=True)
    assert out.shape == (2, 3, 0) and torch.equal(final, init)
    gf = torch.randn_like(init)
    dw, di = torch.autograd.grad(final, [w, init], gf, allow_unused=True)
    assert torch.equal(di, gf) and torch.equal(dw, torch.zeros_like(w))
    out, final = pc.causal_conv(torch.zeros(0, 3, 5, device=DEV), w, return_final_state=True)
    assert out.shape == (0, 3, 5) and final.shape == (0, 3, 3)
    dw, = torch.autograd.grad(out.sum(), w)
    assert torch.equal(dw, torch.zeros_like(w))


def test_conv_strided_inputs_and_expanded_gradients():
    g = gen(3)
    x = torch.randn(2, 50, 6, generator=g).to(DEV).transpose(1, 2).requires_grad_()  # [2, 6, 50], not contiguous
    w = torch.randn(4, 6, generator=g).to(DEV).t().requires_grad_()
    out = pc.causal_conv(x, w, activation="silu")
    same = pc.causal_conv(x.detach().contiguous(), w.detach().contiguous(), activation="silu")
    assert torch.equal(out, same)
    got = torch.autograd.grad(out.sum(), [x, w])
    v, m = ref.conv(x, w, None, True, grad=torch.ones(2, 6, 50))
    check(got[0], v["dx"], m["dx"], 64, "dx")
    check(got[1], v["dw"], m["dw"], 160, "dw")


def test_conv_differences():
    """The gradient of a sum against central differences of the same sum, in
    fp32: the step's truncation is below 1e-4 of the sum of the terms, and the
    values' roundings, 2^-24 * 40 each over the step 2^-6, below another."""
    c, go, _, _ = conv_case(8, 2, 4, 40, 4, torch.float32)
    t = {k: dev(a).requires_grad_() for k, a in c.items()}
    run = lambda t: pc.causal_conv(t["x"], t["w"], t["bias"], "silu", t["init"])  # noqa: E731
    grads = dict(zip(t, torch.autograd.grad(run(t), list(t.values()), dev(go))))
    step = 2.0 ** -6
    for k in t:
        way = ref.rand(gen(9), *t[k].shape).to(DEV)
        way /= way.abs().max()
        with torch.no_grad():
            hi = run({**t, k: t[k] + step * way}).double()
            lo = run({**t, k: t[k] - step * way}).double()
        terms = (hi - lo) / (2 * step) * dev(go).double()
        a, b = float(terms.sum()), float((grads[k].double() * way.double()).sum())
        assert abs(a - b) <= 2e-4 * float(terms.abs().sum()) + 1e-4, k


@pytest.mark.parametrize("K", [1, 2, 4, 8])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_conv_step_goes_on_where_a_prompt_ends(K, dtype):
    """Single tokens from a prompt's final state give what the whole row
    gives, bit for bit: the same sums in the same order."""
    B, D, L, n = 3, 70, 13, 9
    c, _, _, _ = conv_case(K, B, D, L, K, TYPES[dtype])
    t = {k: dev(a) for k, a in c.items()}
    whole, final = pc.causal_conv(t["x"], t["w"], t["bias"], "silu", t["init"], return_final_state=True)
    head, state = pc.causal_conv(t["x"][..., :n].contiguous(), t["w"], t["bias"], "silu", t["init"],
                                 return_final_state=True)
    assert torch.equal(head, whole[..., :n])
    for i in range(n, L):
        out = pc.causal_conv_step(t["x"][..., i], state, t["w"], t["bias"], "silu")
        assert torch.equal(out, whole[..., i])
    assert torch.equal(state, final)


def test_conv_step_places():
    D, K, places = 300, 4, 7
    g = gen(1)
    w = torch.randn(D, K, generator=g).to(DEV)
    state = torch.randn(places, D, K - 1, generator=g).to(DEV)
    x = torch.randn(6, D, generator=g).to(DEV)
    slots = torch.tensor([5, -1, 0, 5, 7, -3], dtype=torch.int32, device=DEV)
    before = state.clone()
    out = pc.causal_conv_step(x, state, w, slots=slots)
    alone = before[[5, 0]].contiguous()
    good = pc.causal_conv_step(x[[0, 2]], alone, w)
    assert torch.equal(out[[0, 2]], good) and torch.equal(state[[5, 0]], alone)
    assert torch.equal(out[1], torch.zeros(D, device=DEV))
    assert torch.isnan(out[[3, 4, 5]]).all()  # twice the same place; none such; none such
    rest = [1, 2, 3, 4, 6]
    assert torch.equal(state[rest], before[rest])


def test_conv_infinite_and_nan_tokens_stay_in_their_windows():
    x = torch.zeros(2, 2, 40, device=DEV)
    x[0, 0, 10], x[0, 1, 39], x[1, 0, 0] = math.inf, math.nan, math.nan
    w = torch.ones(2, 4, device=DEV)
    out = pc.causal_conv(x, w).cpu()
    want = torch.zeros(2, 2, 40)
    want[0, 0, 10:14], want[0, 1, 39], want[1, 0, :4] = math.inf, math.nan, math.nan
    assert torch.equal(torch.nan_to_num(out, nan=7.0, posinf=8.0), torch.nan_to_num(want, nan=7.0, posinf=8.0))


def test_conv_beyond_32_bit_offsets():
    """Rows whose elements lie beyond 2^31 of the array, forwards and backwards."""
    L = (1 << 30) - 3
    x = torch.zeros(1, 3, L, dtype=torch.float16, device=DEV)
    x[0, 2, -5:] = 1.0
    x.requires_grad_()
    w = torch.tensor([[1.0, 2.0]], device=DEV).expand(3, 2).contiguous().half().requires_grad_()
    out = pc.causal_conv(x, w)
    assert out[0, 2, -7:].tolist() == [0, 0, 2, 3, 3, 3, 3] and not out[0, :2].any()
    grad = torch.zeros_like(x)
    grad[0, 2, -1] = 1.0
    dx, dw = torch.autograd.grad(out, [x, w], grad)
    assert dx[0, 2, -3:].tolist() == [0, 1, 2] and not dx[0, :2].any()
    assert dw.tolist() == [[0, 0], [0, 0], [1, 1]]


def test_conv_refuses():
    x, w = torch.zeros(2, 3, 5, device=DEV), torch.zeros(3, 4, device=DEV)
    state = torch.zeros(2, 3, 3, device=DEV)
    bad = [lambda: pc.causal_conv(x[0], w), lambda: pc.causal_conv(x, w[:2]), lambda: pc.causal_conv(x, w.half()),
           lambda: pc.causal_conv(x.double(), w.double()), lambda: pc.causal_conv(x, torch.zeros(3, 9, device=DEV)),
           lambda: pc.causal_conv(x, w, bias=torch.zeros(2, device=DEV)), lambda: pc.causal_conv(x, w.cpu()),
           lambda: pc.causal_conv(x, w, initial_state=state[:1]),
           lambda: pc.causal_conv(x, w, lengths=torch.tensor([1, 2], device=DEV)),
           lambda: pc.causal_conv(x, w, lengths=torch.tensor([1, 2], dtype=torch.int32)),
           lambda: pc.causal_conv(x, torch.zeros(3, 0, device=DEV)),
           lambda: pc.causal_conv_step(x[..., 0], state[..., :2], w),
           lambda: pc.causal_conv_step(x[..., 0], state.transpose(0, 1).contiguous().transpose(0, 1), w),
           lambda: pc.causal_conv_step(x[..., 0], state[:1], w),
           lambda: pc.causal_conv_step(x[..., 0], state.half(), w),
           lambda: pc.causal_conv_step(x[..., 0], state, w, slots=torch.zeros(2, device=DEV, dtype=torch.int64))]
    for i, f in enumerate(bad):
        with pytest.raises((RuntimeError, NotImplementedError)):
            f()
            pytest.fail(f"call {i} was not refused")


# ---------------------------------------------------------- state space scan

def scan_case(seed, nb, ch, L, N, G, dtype, gate=True, skip=True, bias=True, carried=True, lengths=None):
    g = gen(seed)
    c = dict(u=ref.rand(g, nb, ch, L, dtype=dtype), delta=ref.rand(g, nb, ch, L, dtype=dtype, scale=0.5),
             A=-(torch.rand(ch, N, generator=g) * N + 0.05), B=ref.rand(g, nb, G, N, L, dtype=dtype),
             C=ref.rand(g, nb, G, N, L, dtype=dtype), D=ref.rand(g, ch) if skip else None,
             z=ref.rand(g, nb, ch, L, dtype=dtype) if gate else None,
             bias=ref.rand(g, ch, shift=-2.5) if bias else None,
             init=ref.rand(g, nb, ch, N) if carried else None)
    go, gf = ref.rand(g, nb, ch, L, dtype=dtype), ref.rand(g, nb, ch, N)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    return c, go, gf, lens


SCAN_GRADS = dict(u="du", delta="dd", A="dA", B="dB", C="dC", D="dD", z="dz", bias="dbias", init="dinit")


def scan_call(t, softplus, lens, **kw):
    return pc.ssm_scan(t["u"], t["delta"], t["A"], t["B"], t["C"], D=t["D"], z=t["z"], delta_bias=t["bias"],
                       delta_softplus=softplus, initial_state=t["init"], lengths=lens, **kw)


def scan_check(c, go, gf, lens, softplus=True):
    v, m = ref.scan(**{k: c[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")}, softplus=softplus,
                    init=c["init"], lengths=lens, grad=go, grad_final=gf)
    units = (c["u"].shape[2] + 4) * (8 + 4 * float(v["weight"])) + 64
    t = {k: dev(a) for k, a in c.items()}
    if lens is not None:
        for b, n in enumerate(lens.tolist()):
            for k in ("u", "delta", "z", "B", "C"):
                if t[k] is not None:
                    t[k][b, ..., max(0, n):] = math.nan
    leaves = {k: a.requires_grad_() for k, a in t.items() if a is not None}
    out, final = scan_call(t, softplus, dev(lens), return_final_state=True)
    check(out, v["out"], m["out"], units, "out")
    check(final, v["final"], m["final"], units, "final")
    dgo = dev(go)
    if lens is not None:
        for b, n in enumerate(lens.tolist()):
            dgo[b, ..., max(0, n):] = math.nan
    grads = dict(zip(leaves, torch.autograd.grad([out, final], list(leaves.values()), [dgo, dev(gf)])))
    for k, gr in grads.items():
        check(gr, v[SCAN_GRADS[k]], m[SCAN_GRADS[k]], 2 * units, SCAN_GRADS[k])
    with torch.no_grad():
        alone = scan_call(t, softplus, dev(lens))
    assert torch.equal(alone, out)
    return grads


@pytest.mark.parametrize("N", [1, 3, 4, 5, 8, 16, 24, 33, 64, 100, 128])
@pytest.mark.parametrize("L", [1, 2, 17, 33, 70])
def test_scan_states_and_lengths(N, L):
    scan_check(*scan_case(N * 7 + L, 2, 6, L, N, 2, torch.float32))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("ch,G,L", [(1, 1, 40), (35, 1, 64), (66, 2, 129), (130, 1, 31)])
def test_scan_types_and_channels(dtype, ch, G, L):
    scan_check(*scan_case(ch + L, 2, ch, L, 16, G, TYPES[dtype]))


@pytest.mark.parametrize("gate,skip,bias,carried,softplus", [
    (False, False, False, False, False), (True, False, False, False, True), (False, True, False, True, True),
    (False, False, True, False, True), (True, True, True, True, False)])
def test_scan_optional_inputs(gate, skip, bias, carried, softplus):
    c, go, gf, lens = scan_case(5, 2, 9, 50, 8, 1, torch.float32, gate, skip, bias, carried)
    if not softplus:
        c["delta"] = c["delta"].abs() * 0.2
        if c["bias"] is not None:
            c["bias"] = c["bias"].abs() * 0.02
    scan_check(c, go, gf, lens, softplus)


@pytest.mark.parametrize("N", [2, 8, 16, 40, 128])
@pytest.mark.parametrize("L,lengths", [(40, [40, 0, 1, 33, 2]), (130, [64, 0, 130, 65, 500, -1, 16])])
def test_scan_ragged_rows(N, L, lengths):
    scan_check(*scan_case(N + L, len(lengths), 5, L, N, 1, torch.float16, lengths=lengths))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("N,L,lengths", [(16, 1000, None), (16, 515, [515, 0]), (6, 640, [130, 1]), (30, 700, None)])
def test_scan_in_segments(dtype, N, L, lengths):
    """Few rows and a long axis: the length is cut into segments that run at
    the same time."""
    nb = 1 if lengths is None else len(lengths)
    scan_check(*scan_case(N + L, nb, 40, L, N, 1, TYPES[dtype], lengths=lengths))


def test_scan_large_steps_and_growing_states():
    """softplus above its threshold, decays that vanish, and A > 0."""
    c, go, gf, lens = scan_case(12, 1, 5, 20, 4, 1, torch.float32)
    c["delta"][..., ::3] = 25.0
    c["A"][0] = -300.0
    c["A"][1] = 0.01
    c["A"][2] = 0.0
    c["delta"][:, 1] = -3.0
    scan_check(c, go, gf, lens)


def test_scan_empty():
    init = torch.randn(2, 6, 4, device=DEV, requires_grad=True)
    A = torch.randn(6, 4, device=DEV, requires_grad=True)
    z = torch.zeros
    out, final = pc.ssm_scan(z(2, 6, 0, device=DEV), z(2, 6, 0, device=DEV), A, z(2, 1, 4, 0, device=DEV),
                             z(2, 1, 4, 0, device=DEV), initial_state=init, return_final_state=True)
    assert out.shape == (2, 6, 0) and torch.equal(final, init)
    gf = torch.randn_like(init)
    dA, di = torch.autograd.grad(final, [A, init], gf)
    assert torch.equal(di, gf) and torch.equal(dA, torch.zeros_like(A))
    u = z(0, 6, 5, device=DEV)
    out = pc.ssm_scan(u, u, A, z(0, 1, 4, 5, device=DEV), z(0, 1, 4, 5, device=DEV))
    dA, = torch.autograd.grad(out.sum(), A)
    assert out.shape == (0, 6, 5) and torch.equal(dA, torch.zeros_like(A))


def test_scan_without_channels():
    z = lambda *s: torch.zeros(*s, device=DEV, requires_grad=True)  # noqa: E731
    B, C = z(2, 1, 4, 9), z(2, 1, 4, 9)
    out, final = pc.ssm_scan(z(2, 0, 9), z(2, 0, 9), z(0, 4), B, C, return_final_state=True)
    assert out.shape == (2, 0, 9) and final.shape == (2, 0, 4)
    dB, dC = torch.autograd.grad(out.sum(), [B, C])
    assert not dB.any() and not dC.any()


@pytest.mark.parametrize("L", [5, 40, 700])
def test_scan_infinite_states(L):
    """A state that is infinite stays so, decaying, growing or kept; the other
    states of its channel and the other channels are what they are without."""
    c, _, _, _ = scan_case(L, 1, 40, L, 4, 1, torch.float32)
    c["A"][1, 2], c["A"][2, 2] = 0.01, 0.0
    t = {k: dev(a) for k, a in c.items()}
    want_out, want = scan_call(t, True, None, return_final_state=True)
    for ch in range(3):
        t["init"][0, ch, 2] = -math.inf
    out, final = scan_call(t, True, None, return_final_state=True)
    far = torch.zeros(40, 4, dtype=torch.bool)
    far[:3, 2] = True
    assert (final[0].cpu()[far] == -math.inf).all() and torch.equal(final[0].cpu()[~far], want[0].cpu()[~far])
    assert torch.equal(out[0, 3:], want_out[0, 3:]) and not torch.isfinite(out[0, :3]).any()


def test_scan_strided_inputs_and_partial_gradients():
    c, go, _, _ = scan_case(4, 2, 6, 37, 5, 2, torch.float32)
    t = {k: dev(a) for k, a in c.items()}
    want = scan_call(t, True, None)
    s = dict(t)
    for k in ("u", "delta", "z", "B", "C"):
        s[k] = t[k].transpose(-1, -2).contiguous().transpose(-1, -2)
    off = torch.empty(t["u"].numel() + 1, device=DEV)[1:].view(t["u"].shape)
    s["u"] = off.copy_(t["u"])
    assert torch.equal(scan_call(s, True, None), want)
    # only some inputs need a gradient; the final state alone is used
    s["B"] = t["B"].clone().requires_grad_()
    out, final = scan_call(s, True, None, return_final_state=True)
    gf = torch.randn_like(final)
    dB, = torch.autograd.grad(final, s["B"], gf)
    v, m = ref.scan(**{k: c[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")}, softplus=True,
                    init=c["init"], grad=torch.zeros_like(go), grad_final=gf.cpu())
    check(dB, v["dB"], m["dB"], 2 * (41 * (8 + 4 * float(v["weight"])) + 64), "dB")


def test_scan_differences():
    """As for the convolution; the recurrence is smooth in all its inputs, and
    a sum over 60 tokens has errors of up to 1300 roundings a term."""
    c, go, _, _ = scan_case(8, 2, 5, 60, 6, 1, torch.float32)
    t = {k: dev(a).requires_grad_() for k, a in c.items()}
    grads = dict(zip(t, torch.autograd.grad(scan_call(t, True, None), list(t.values()), dev(go))))
    step = 2.0 ** -7
    for k in t:
        way = ref.rand(gen(9), *t[k].shape).to(DEV)
        way /= way.abs().max()
        with torch.no_grad():
            hi = scan_call({**t, k: t[k] + step * way}, True, None).double()
            lo = scan_call({**t, k: t[k] - step * way}, True, None).double()
        terms = (hi - lo) / (2 * step) * dev(go).double()
        a, b = float(terms.sum()), float((grads[k].double() * way.double()).sum())
        assert abs(a - b) <= 1e-3 * float(terms.abs().sum()) + 1e-2, k


@pytest.mark.parametrize("N", [1, 4, 6, 16, 64, 128])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_scan_step_goes_on_where_a_prompt_ends(N, dtype):
    nb, ch, G, L, n = 2, 70, 2, 9, 5
    c, _, _, _ = scan_case(N, nb, ch, L, N, G, TYPES[dtype])
    v, m = ref.scan(**{k: c[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")}, softplus=True, init=c["init"])
    units = (L + 4) * (8 + 4 * float(v["weight"])) + 64
    t = {k: dev(a) for k, a in c.items()}
    head = {k: (t[k][..., :n].contiguous() if k in ("u", "delta", "z", "B", "C") else t[k]) for k in t}
    out, state = scan_call(head, True, None, return_final_state=True)
    check(out, v["out"][..., :n], m["out"][..., :n], units, "prompt")
    for i in range(n, L):
        got = pc.ssm_scan_step(t["u"][..., i], t["delta"][..., i], state, t["A"], t["B"][..., i], t["C"][..., i],
                               D=t["D"], z=t["z"][..., i], delta_bias=t["bias"], delta_softplus=True)
        check(got, v["out"][..., i], m["out"][..., i], units, f"token {i}")
    check(state, v["final"], m["final"], units, "state")


def test_scan_step_places():
    ch, N, places = 40, 16, 7
    c, _, _, _ = scan_case(3, 6, ch, 1, N, 1, torch.bfloat16)
    t = {k: dev(a) for k, a in c.items()}
    state = torch.randn(places, ch, N, device=DEV)
    before = state.clone()
    slots = torch.tensor([5, -1, 0, 5, 7, -3], dtype=torch.int32, device=DEV)

    def step(rows, st, slots=None):
        return pc.ssm_scan_step(t["u"][rows, :, 0], t["delta"][rows, :, 0], st, t["A"], t["B"][rows, ..., 0],
                                t["C"][rows, ..., 0], D=t["D"], z=t["z"][rows, :, 0], delta_bias=t["bias"],
                                delta_softplus=True, slots=slots)

    out = step(list(range(6)), state, slots)
    alone = before[[5, 0]].contiguous()
    good = step([0, 2], alone)
    assert torch.equal(out[[0, 2]], good) and torch.equal(state[[5, 0]], alone)
    assert torch.equal(out[1], torch.zeros_like(out[1])) and torch.isnan(out[[3, 4, 5]]).all()
    rest = [1, 2, 3, 4, 6]
    assert torch.equal(state[rest], before[rest])


def test_scan_step_beyond_32_bit_offsets():
    ch, N = 2048, 16
    places = (1 << 31) // (ch * N) + 3
    state = torch.zeros(places, ch, N, device=DEV)  # 8.6 GB
    state[-1] = 1.0
    c, _, _, _ = scan_case(3, 1, ch, 1, N, 1, torch.float32)
    t = {k: dev(a) for k, a in c.items()}
    args = [t["u"][..., 0], t["delta"][..., 0]]
    rest = dict(D=t["D"], z=t["z"][..., 0], delta_bias=t["bias"], delta_softplus=True)
    last = torch.tensor([places - 1], dtype=torch.int32, device=DEV)
    out = pc.ssm_scan_step(*args, state, t["A"], t["B"][..., 0], t["C"][..., 0], slots=last, **rest)
    small = torch.ones(1, ch, N, device=DEV)
    want = pc.ssm_scan_step(*args, small, t["A"], t["B"][..., 0], t["C"][..., 0], **rest)
    assert torch.equal(out, want) and torch.equal(state[-1:], small)
    assert not state[:-1].any()


def test_scan_refuses():
    c, _, _, _ = scan_case(3, 2, 6, 8, 4, 2, torch.float32)
    t = {k: dev(a) for k, a in c.items()}
    lens = torch.tensor([1, 2], dtype=torch.int32, device=DEV)
    scan_call(t, True, lens)
    bad = [dict(u=t["u"].half()), dict(u=t["u"][..., :7]), dict(delta=t["delta"][:1]), dict(A=t["A"].double()),
           dict(A=t["A"][:5]), dict(A=torch.zeros(6, 129, device=DEV)), dict(B=t["B"][:, 0]), dict(B=t["B"].half()),
           dict(B=torch.zeros(2, 4, 4, 8, device=DEV), C=torch.zeros(2, 4, 4, 8, device=DEV)),
           dict(C=t["C"][:, :, :3]), dict(D=t["D"][:2]), dict(z=t["z"][:, :3]), dict(bias=t["bias"].cpu()),
           dict(init=t["init"][:1]), dict(init=t["init"].half())]
    for i, change in enumerate(bad):
        with pytest.raises((RuntimeError, NotImplementedError)):
            scan_call({**t, **change}, True, None)
            pytest.fail(f"call {i} was not refused")
    for wrong in (lens.long(), lens[:1], lens.cpu()):
        with pytest.raises(RuntimeError):
            scan_call(t, True, wrong)
    one = {k: (v[..., 0] if k in ("u", "delta", "z", "B", "C") else v) for k, v in t.items()}
    state = t["init"].clone()
    for st in (state[:1], state.half(), state[..., :3], state.transpose(0, 1).contiguous().transpose(0, 1)):
        with pytest.raises(RuntimeError):
            pc.ssm_scan_step(one["u"], one["delta"], st, t["A"], one["B"], one["C"])
    with pytest.raises(RuntimeError, match="once_differentiable|differentiable once"):
        u = t["u"].clone().requires_grad_()
        g, = torch.autograd.grad(scan_call({**t, "u": u}, True, None).square().sum(), u, create_graph=True)
        g.sum().backward()


# ------------------------------------------------- together, streams, graphs

class Block(torch.nn.Module):
    """The operators as they are used together, over the map of a ParaConv2d
    layer: convolution, projections of each token, gated scan, residual."""

    def __init__(self, ch, states, p):
        super().__init__()
        self.conv = pc.CausalConv(ch, 4, activation="silu")
        self.scan = pc.SSMScan(ch, states)
        self.drop = pc.Dropout(p, seed=21)
        self.proj = torch.nn.Parameter(torch.randn(ch + 2 * states + ch, ch) * ch ** -0.5)
        self.states = states

    def inputs(self, x):
        ch, n = x.shape[1], self.states
        w = self.proj.to(x.dtype)
        d, b, c, z = torch.einsum("oc,bc...->bo...", w, x).split([ch, n, n, ch], 1)
        return d.contiguous(), b.unsqueeze(1).contiguous(), c.unsqueeze(1).contiguous(), z.contiguous()

    def forward(self, x):
        h = self.conv(x)
        d, b, c, z = self.inputs(h)
        return self.drop(self.scan(h, d, b, c, z), residual=x)


def test_block_over_a_paraconv_map():
    """ParaConv2d -> block -> sum, with gradients to every parameter, against
    the same block computed by autograd in 64 bits from the layer's map."""
    torch.manual_seed(0)
    layer = pc.ParaConv2d(3, 8, 3, padding=1).to(DEV)
    block = Block(8, 4, 0.25).to(DEV)
    x = torch.randn(2, 3, 6, 7, generator=gen(1)).to(DEV)
    fmap = layer(x)
    seq = fmap.flatten(2)
    seq.retain_grad()
    out = block(seq)
    go = torch.randn(out.shape, generator=gen(2)).to(DEV)
    (out * go).sum().backward()
    assert layer.pars.grad is not None and torch.isfinite(layer.pars.grad).all()

    p = {n: v.detach().cpu().double().requires_grad_() for n, v in block.named_parameters()}
    s = seq.detach().cpu().double().requires_grad_()
    line = torch.cat([torch.zeros(2, 8, 3, dtype=torch.float64), s], -1)
    pre = sum(p["conv.weight"][:, k, None] * line[..., k:k + 42] for k in range(4)) + p["conv.bias"][:, None]
    h = torch.nn.functional.silu(pre)
    d, b, c, z = torch.einsum("oc,bcl->bol", p["proj"], h).split([8, 4, 4, 8], 1)
    dt = torch.nn.functional.softplus(d + p["scan.delta_bias"][:, None])
    A = -torch.exp(p["scan.A_log"])
    state, ys = torch.zeros(2, 8, 4, dtype=torch.float64), []
    for t in range(42):
        state = torch.exp(dt[..., t, None] * A) * state + (dt * h)[..., t, None] * b[:, None, :, t]
        ys.append((state * c[:, None, :, t]).sum(-1))
    y = (torch.stack(ys, -1) + p["scan.D"][:, None] * h) * torch.nn.functional.silu(z)
    keep = ref.kept_mask(y.numel(), 0.25, 21, 0).view(y.shape)
    want = s + torch.where(keep, y * ref.keep_scale(0.25), 0.0)
    (want * go.cpu().double()).sum().backward()
    # (each value passes at most 42 steps and two sums of 8 in fp32: 1e-4 of the largest)
    assert float((out.detach().cpu().double() - want.detach()).abs().max()) <= 1e-4 * float(want.detach().abs().max())
    for got, ref_ in [(seq.grad, s.grad)] + [(q.grad, p[n].grad) for n, q in block.named_parameters()]:
        assert float((got.cpu().double() - ref_).abs().max()) <= 2e-4 * float(ref_.abs().max())


def test_prompt_then_tokens_equals_the_whole():
    """Convolution and scan over a prompt, then token by token with states in
    places of a pool, against the whole sequence."""
    torch.manual_seed(3)
    ch, n, L, head = 24, 16, 50, 41
    block = Block(ch, n, 0.0).to(DEV).eval()
    x = torch.randn(3, ch, L, generator=gen(4)).to(DEV)
    with torch.no_grad():
        whole = block(x)
        h, cs = block.conv(x[..., :head].contiguous(), return_final_state=True)
        d, b, c, z = block.inputs(h)
        y, ss = block.scan(h, d, b, c, z, return_final_state=True)
        assert torch.allclose(x[..., :head] + y, whole[..., :head], rtol=1e-5, atol=1e-5)
        pool_c, pool_s = block.conv.new_state(5), block.scan.new_state(5)
        slots = torch.tensor([4, 0, 2], dtype=torch.int32, device=DEV)
        pool_c[slots.long()], pool_s[slots.long()] = cs, ss
        for t in range(head, L):
            h = block.conv.step(x[..., t], pool_c, slots=slots)
            d, b, c, z = block.inputs(h)
            y = block.scan.step(h, d, pool_s, b, c, z, slots=slots)
            assert torch.allclose(x[..., t] + y, whole[..., t], rtol=1e-5, atol=1e-5), t
    assert not pool_s[[1, 3]].any()


def _train_step(block, x, go):
    return torch.autograd.grad(block(x), [x] + list(block.parameters()), go)


def test_same_results_again_and_on_another_stream():
    torch.manual_seed(5)
    block = Block(96, 16, 0.0).to(DEV)
    x = torch.randn(2, 96, 700, generator=gen(6)).to(DEV).requires_grad_()
    go = torch.randn(2, 96, 700, generator=gen(7)).to(DEV)
    first = _train_step(block, x, go)
    again = _train_step(block, x, go)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _train_step(block, x, go)
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(first, again, other):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_two_captured_steps_replayed_together():
    """Forward and backward captured twice and replayed at the same time on two
    streams: the graphs' workspaces are their own."""
    torch.manual_seed(8)
    blocks = [Block(64, 16, 0.0).to(DEV) for _ in range(2)]
    xs = [torch.randn(1, 64, 900, generator=gen(9 + i)).to(DEV).requires_grad_() for i in range(2)]
    go = torch.randn(1, 64, 900, generator=gen(11)).to(DEV)
    want = [[g.clone() for g in _train_step(b, x, go)] for b, x in zip(blocks, xs)]
    graphs, outs = [], []
    for b, x in zip(blocks, xs):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _train_step(b, x, go)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_train_step(b, x, go))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for o in outs:
        for g in o:
            g.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for got, w in zip(outs, want):
        for a, b in zip(got, w):
            assert torch.equal(a, b)


def test_captured_tokens():
    """Steps of a captured graph move the states on as eager steps do, with
    the slots as they are at each replay."""
    ch, N = 64, 16
    c, _, _, _ = scan_case(3, 2, ch, 1, N, 1, torch.bfloat16)
    t = {k: dev(a) for k, a in c.items()}
    w = torch.randn(ch, 4, device=DEV, dtype=torch.bfloat16)
    slots = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    cs, ss = torch.zeros(4, ch, 3, device=DEV, dtype=torch.bfloat16), torch.zeros(4, ch, N, device=DEV)

    def step(cs, ss, slots):
        h = pc.causal_conv_step(t["u"][..., 0], cs, w, activation="silu", slots=slots)
        return pc.ssm_scan_step(h, t["delta"][..., 0], ss, t["A"], t["B"][..., 0], t["C"][..., 0], D=t["D"],
                                z=t["z"][..., 0], delta_bias=t["bias"], delta_softplus=True, slots=slots)

    ec, es = cs.clone(), ss.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cs.clone(), ss.clone(), slots)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cs, ss, slots)
    for places in ([0, 1], [3, 0], [2, -1]):
        slots.copy_(torch.tensor(places, dtype=torch.int32))
        graph.replay()
        want = step(ec, es, torch.tensor(places, dtype=torch.int32, device=DEV))
        assert torch.equal(out, want) and torch.equal(cs, ec) and torch.equal(ss, es)


def test_no_device_error_was_recorded():
    torch.cuda.synchronize()
    assert _lib.cabi().pc2d_device_status() == 0
