"""The layers beside ParaConv2d on the GPU where a call or a value leaves the
ordinary.  Tolerances as in test_layers_gpu.py, unless said at the test.
"""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

import layers_ref as ref
import paraconv2d_b200 as pc
from test_layers_gpu import DEV, SCAN_GRADS, check, conv_case, dev, gen, scan_call, scan_case

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------- steps

def test_steps_refuse_inputs_within_their_state():
    """A view of the state as a token: other rows' places would be written
    while it is read.  Neighbours of the state in one allocation are fine, and
    so are views that have to be copied first."""
    w = torch.randn(16, 2, device=DEV)
    pool = torch.randn(6, 16, 1, device=DEV)
    slots = torch.tensor([2, 3], dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="shares memory with the state"):
        pc.causal_conv_step(pool[:2, :, 0], pool, w, slots=slots)
    with pytest.raises(RuntimeError, match="shares memory with the state"):
        pc.causal_conv_step(torch.zeros(2, 16, device=DEV), pool, w, bias=pool[5, :, 0], slots=slots)
    before = pool.clone()
    got = pc.causal_conv_step(pool[:2, :, 0], pool[2:4], w)
    assert torch.equal(got, pc.causal_conv_step(before[:2, :, 0], before[2:4].clone(), w))
    u, B = torch.randn(2, 16, device=DEV), torch.randn(2, 1, 16, device=DEV)
    A = -torch.rand(16, 16, device=DEV)
    pool = torch.randn(6, 16, 16, device=DEV)
    names = dict(u=u, delta=u.abs(), A=A, B=B, C=B, D=u[0].clone(), z=u.clone(), delta_bias=u[1].clone())

    def step(state, **kw):
        t = {**names, **kw}
        return pc.ssm_scan_step(t["u"], t["delta"], state, t["A"], t["B"], t["C"], D=t["D"], z=t["z"],
                                delta_bias=t["delta_bias"], slots=slots)

    step(pool)
    within = dict(u=pool[0, :2], delta=pool[5, 14:], A=pool[1], B=pool[0, :2].view(2, 1, 16), C=pool[5, 14:].view(2, 1, 16),
                  D=pool[0, 0], z=pool[0, :2], delta_bias=pool[5, 15])
    for k, v in within.items():
        with pytest.raises(RuntimeError, match="shares memory with the state"):
            step(pool, **{k: v})
    # a strided view is copied before anything is written
    views, whole = pool.clone(), pool.clone()
    got = step(views, u=views[:2, :, 3])
    assert torch.equal(got, step(whole, u=pool[:2, :, 3].contiguous())) and torch.equal(views, whole)


# ------------------------------------------------------------------ autograd

def test_forward_mode_is_refused():
    """An input with a tangent: no derivative rather than one of zero."""
    c, _, _, _ = scan_case(1, 2, 6, 8, 4, 1, torch.float32)
    t = {k: dev(a) for k, a in c.items()}
    key = torch.tensor([1, 2], device=DEV)
    one = {k: (v[..., 0].contiguous() if k in ("u", "delta", "z", "B", "C") else v) for k, v in t.items()}
    w = torch.randn(6, 4, device=DEV)
    with fwd.dual_level():
        dual = {k: fwd.make_dual(v, torch.ones_like(v)) for k, v in t.items()}
        for k in dual:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                scan_call({**t, k: dual[k]}, True, None)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            pc.dropout(dual["u"], 0.5, key)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            pc.dropout(t["u"], 0.5, key, residual=dual["u"])
        with pytest.raises(NotImplementedError, match="forward-mode"):
            pc.causal_conv(t["u"], fwd.make_dual(w, w))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            pc.causal_conv_step(fwd.make_dual(one["u"], one["u"]), torch.zeros(2, 6, 3, device=DEV), w)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            pc.ssm_scan_step(one["u"], one["delta"], fwd.make_dual(t["init"].clone(), t["init"]), one["A"], one["B"], one["C"])
    assert torch.equal(scan_call(t, True, None), scan_call(t, True, None))


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_what_autograd_saved_and_a_call_changed_is_noticed(mode):
    """A key that is counted on, and kept inputs that a step moves on, between
    a call that saved them and its backward pass."""
    x = torch.randn(2, 6, 9, device=DEV, requires_grad=True)
    w = torch.randn(6, 4, device=DEV)
    state = torch.tensor([5, 0], device=DEV)
    out = pc.dropout(x, 0.5, state)
    with mode():
        torch.ops.paraconv2d_b200.dropout_next_key(state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    kept = torch.randn(2, 6, 3, device=DEV)
    out = pc.causal_conv(x, w, initial_state=kept)
    with mode():
        pc.causal_conv_step(x.detach()[..., 0], kept, w)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    h = torch.randn(2, 6, 4, device=DEV)
    before = h._version
    with mode():
        pc.ssm_scan_step(x.detach()[..., 0], x.detach()[..., 0], h, -torch.ones(6, 4, device=DEV),
                         torch.ones(2, 1, 4, device=DEV), torch.ones(2, 1, 4, device=DEV))
    assert h._version > before
    with torch.inference_mode():  # (an inference tensor has no version to count)
        pc.causal_conv_step(x.detach()[..., 0], torch.zeros(2, 6, 3, device=DEV), w)


def test_dispatch_modes_see_the_calls():
    from torch.utils._python_dispatch import TorchDispatchMode

    class Log(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(func.name())
            return func(*args, **(kwargs or {}))

    c, go, _, _ = scan_case(1, 2, 6, 8, 4, 1, torch.float32)
    t = {k: dev(a).requires_grad_() for k, a in c.items()}
    w = torch.randn(6, 4, device=DEV, requires_grad=True)
    with Log() as log:
        y = pc.dropout(scan_call({**t, "u": pc.causal_conv(t["u"], w)}, True, None), 0.5, torch.tensor([1, 2], device=DEV))
        torch.autograd.grad(y, [t["u"], w], dev(go))
        with torch.no_grad():
            pc.causal_conv_step(t["u"][..., 0], torch.zeros(2, 6, 3, device=DEV), w)
    own = [n.split("::")[1] for n in log.names if n.startswith("paraconv2d_b200")]
    assert own == ["causal_conv_forward", "ssm_scan_forward", "dropout", "dropout", "ssm_scan_backward",
                   "causal_conv_backward", "causal_conv_step"]


# ---------------------------------------------- infinities in the convolution

def finite_part(t):
    """What a finite value can contain."""
    return torch.where(torch.isfinite(t), t, 0.0)


def same_or_both_not_finite(got, value, mag, units, what):
    """Finite where the formula's value is, and then within the tolerance."""
    g = got.detach().cpu()
    ok = torch.isfinite(value)
    assert torch.equal(torch.isfinite(g), ok), (what, g, value)
    check(torch.where(ok, g, 0.0), torch.where(ok, value, 0.0), torch.where(ok, mag, 0.0), units, what)


@pytest.mark.parametrize("L", [5, 8, 13, 16, 21, 300, 523])
@pytest.mark.parametrize("K", [2, 4, 8])
def test_conv_weight_gradients_leave_out_what_taps_do_not_meet(L, K):
    """A row's last tokens meet its last taps only, the kept inputs its first:
    an infinity there makes those taps' gradients infinite and no others."""
    c, go, gf, _ = conv_case(L + K, 2, 5, L, K, torch.float32, bias=False)
    for b in range(2):
        c["x"][b, 0, -1] = math.inf
        c["x"][b, 1, -min(2, L)] = math.nan
        c["init"][b, 2, 0] = -math.inf
        c["init"][b, 3, -1] = math.inf
    v, _ = ref.conv(c["x"], c["w"], None, False, c["init"], None, go, gf)
    _, m = ref.conv(finite_part(c["x"]), c["w"], None, False, finite_part(c["init"]), None, go, gf)
    assert torch.isfinite(v["dw"]).any() and not torch.isfinite(v["dw"]).all()
    x, w, init = (dev(c[k]).requires_grad_() for k in ("x", "w", "init"))
    out, final = pc.causal_conv(x, w, initial_state=init, return_final_state=True)
    got = torch.autograd.grad([out, final], [x, w, init], [dev(go), dev(gf)])
    for g, n in zip(got, ("dx", "dw", "dinit")):
        same_or_both_not_finite(g, v[n], m[n], 160, n)
    # the same rows within a padded batch
    pad = torch.full((2, 5, L + 11), math.nan, device=DEV)
    pad[..., :L] = x.detach()
    pad.requires_grad_()
    lens = torch.full((2,), L, dtype=torch.int32, device=DEV)
    out, final = pc.causal_conv(pad, w, initial_state=init, lengths=lens, return_final_state=True)
    pgo = torch.full((2, 5, L + 11), math.nan, device=DEV)
    pgo[..., :L] = dev(go)
    got = torch.autograd.grad([out, final], [pad, w, init], [pgo, dev(gf)])
    assert not got[0][..., L:].any() and not out[..., L:].any()
    for g, n in zip((got[0][..., :L], *got[1:]), ("dx", "dw", "dinit")):
        same_or_both_not_finite(g, v[n], m[n], 160, n)


@pytest.mark.parametrize("n", [1, 2, 13, 16, 290])
@pytest.mark.parametrize("K", [1, 2, 4, 8])
def test_conv_infinite_weights_reach_their_windows_only(n, K):
    """An infinite weight: the gradient of an input that its tap does not meet
    stays finite, and behind a row's tokens everything stays 0."""
    L = n + 13
    c, go, _, _ = conv_case(n + K, 2, 4, n, K, torch.float32, bias=False)
    c["w"][0, 0], c["w"][1, -1], c["w"][2, K // 2] = math.inf, -math.inf, math.nan
    go[:, :, n // 2] = 0.0
    v, _ = ref.conv(c["x"], c["w"], None, False, c["init"], None, go, torch.zeros(2, 4, K - 1))
    _, m = ref.conv(c["x"], finite_part(c["w"]), None, False, c["init"], None, go, torch.zeros(2, 4, K - 1))
    x, pgo = (torch.full((2, 4, L), math.nan, device=DEV) for _ in range(2))
    x[..., :n], pgo[..., :n] = dev(c["x"]), dev(go)
    x.requires_grad_()
    init = dev(c["init"]).requires_grad_()
    out = pc.causal_conv(x, dev(c["w"]), initial_state=init, lengths=torch.full((2,), n, dtype=torch.int32, device=DEV))
    dx, di = torch.autograd.grad(out, [x, init], pgo)
    assert not out[..., n:].any() and not dx[..., n:].any()
    same_or_both_not_finite(out[..., :n], v["out"], m["out"], 40, "out")
    same_or_both_not_finite(dx[..., :n], v["dx"], m["dx"], 64, "dx")
    same_or_both_not_finite(di, v["dinit"], m["dinit"], 64, "dinit")


# ------------------------------------------- the scan's states, beyond bounds

def test_scan_segments_keep_infinite_states_that_decay_fast():
    """700 tokens of one row are cut into segments, over each of which these
    states decay by more than 32 bits hold: an infinite one stays infinite."""
    c, _, _, _ = scan_case(1, 1, 40, 700, 4, 1, torch.float32)
    c["A"][:3, 2] = -100.0
    t = {k: dev(a) for k, a in c.items()}
    _, want = scan_call(t, True, None, return_final_state=True)
    t["init"][0, :3, 2] = -math.inf
    _, final = scan_call(t, True, None, return_final_state=True)
    far = torch.zeros(40, 4, dtype=torch.bool)
    far[:3, 2] = True
    assert (final[0].cpu()[far] == -math.inf).all() and torch.equal(final[0].cpu()[~far], want[0].cpu()[~far])
    # backwards: an infinite gradient of the final state reaches the first one
    t["init"] = dev(c["init"]).requires_grad_()
    gf = torch.zeros(1, 40, 4, device=DEV)
    gf[0, :3, 2] = math.inf
    _, final = scan_call(t, True, None, return_final_state=True)
    di, = torch.autograd.grad(final, t["init"], gf)
    assert (di[0].cpu()[far] == math.inf).all() and not di[0].cpu()[~far].any()


def test_scan_segments_of_growing_states_that_are_zero_or_small():
    """Growth over a segment that overflows 32 bits by itself, of states that
    are still 0, or small enough to stay within them."""
    c, go, _, _ = scan_case(2, 1, 40, 700, 4, 1, torch.float32, gate=False, carried=False)
    c["delta"][:] = -2.3  # d = 0.095
    c["bias"][:] = 0.0
    c["A"][:] = 20.0
    c["u"][..., :-5] = 0.0   # the states stay 0 up to the last tokens,
    go[..., 5:] = 0.0        # their gradients from the first ones on
    v, m = ref.scan(**{k: c[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")}, softplus=True,
                    grad=torch.zeros_like(go), grad_final=None)
    t = {k: dev(a) for k, a in c.items()}
    units = 704 * (8 + 4 * float(v["weight"])) + 64
    out, final = scan_call(t, True, None, return_final_state=True)
    check(out, v["out"], m["out"], units, "out")
    check(final, v["final"], m["final"], units, "final")
    c["u"] = ref.rand(gen(3), 1, 40, 700)
    c["u"][..., 5:] = 0.0
    c["A"][:] = torch.where(torch.arange(40)[:, None] < 20, 20.0, -20.0)
    t = {k: dev(a) for k, a in c.items()}
    leaves = {k: t[k].requires_grad_() for k in ("u", "B")}
    out = scan_call(t, True, None)
    du, dB = torch.autograd.grad(out, list(leaves.values()), dev(go))
    assert torch.isfinite(du).all() and not du[..., 5:].any()
    assert torch.isfinite(dB).all()


@pytest.mark.parametrize("A,init", [(8.0, 1e-30), (-8.0, 1e30)])
def test_scan_segment_factor_out_of_range_beside_a_state_that_is_not(A, init):
    """exp of 128 tokens' sum overflows (underflows); times the state that it
    meets, it does not.  The rest of the row changes nothing (d = 0)."""
    c, _, _, _ = scan_case(4, 1, 40, 300, 4, 1, torch.float32, gate=False)
    c["bias"][:] = 0.0
    c["delta"][..., :128] = -2.3
    c["delta"][..., 128:] = -200.0
    c["u"][:] = 0.0
    c["A"][:], c["init"][:] = A, init
    v, m = ref.scan(**{k: c[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")}, softplus=True, init=c["init"])
    t = {k: dev(a) for k, a in c.items()}
    _, final = scan_call(t, True, None, return_final_state=True)
    # (the exponent, 102, is off by its d's 4 roundings and its sum's 128 at most: 132 * 102 of them)
    check(final, v["final"], m["final"], 132 * 102 + 304 * 12, "final")


@pytest.mark.parametrize("L,lengths", [(5, None), (37, None), (64, None), (45, [45, 7, 0]), (700, None)])
@pytest.mark.parametrize("N", [3, 16])
def test_scan_infinite_decay_rates(L, lengths, N):
    """A = -inf forgets at every token, and only at tokens: what a lowest
    finite rate gives, bit for bit, gradients too."""
    nb = 1 if lengths is None else len(lengths)
    c, go, gf, lens = scan_case(L + N, nb, 10, L, N, 1, torch.float32, lengths=lengths)
    results = []
    for low in (-math.inf, -1e38):
        t = {k: dev(a) for k, a in c.items()}
        t["A"][::2, 1] = low
        leaves = [t[k].requires_grad_() for k in t]
        out, final = scan_call(t, True, dev(lens), return_final_state=True)
        results.append([out, final, *torch.autograd.grad([out, final], leaves, [dev(go), dev(gf)])])
    for a, b in zip(*results):
        assert torch.isfinite(b).all() and torch.equal(a, b)


def test_scan_step_infinite_decay_rates():
    c, _, _, _ = scan_case(2, 2, 10, 1, 16, 1, torch.float32)
    c["delta"][0] = -200.0  # d = 0: nothing is forgotten
    results = []
    for low in (-math.inf, -1e38):
        t = {k: dev(a[..., 0].contiguous() if k in ("u", "delta", "z", "B", "C") else a) for k, a in c.items()}
        t["A"][:, 1] = low
        state = t["init"].clone()
        out = pc.ssm_scan_step(t["u"], t["delta"], state, t["A"], t["B"], t["C"], D=t["D"], z=t["z"],
                               delta_bias=t["bias"], delta_softplus=True)
        results.append((out, state))
    assert torch.isfinite(results[0][1]).all()
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])


@pytest.mark.parametrize("L,n", [(13, 13), (40, 13), (32, 32), (700, 655)])
@pytest.mark.parametrize("N,channel", [(4, 0), (16, 0), (16, 9)])
def test_scan_state_that_overflows_at_the_last_token(L, n, N, channel):
    """The last token makes a state infinite: its own output and dC are so,
    and nothing else; not the gradients behind it, nor the sums that pass
    over the rest of its tile, nor those over lanes without a channel."""
    c, go, _, _ = scan_case(L + N, 1, 10, n, N, 1, torch.float32, gate=False)
    c["u"][0, channel, -1] = 1e38
    c["B"][0, 0, 2, -1] = 1e5
    go[0, :, -1] *= 1e-12
    v, m = ref.scan(**{k: c[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")}, softplus=True,
                    init=c["init"], grad=go)
    t = {k: dev(a) for k, a in c.items()}
    pgo = torch.full((1, 10, L), math.nan, device=DEV)
    pgo[..., :n] = dev(go)
    for k in ("u", "delta", "B", "C"):
        t[k] = torch.nn.functional.pad(t[k], (0, L - n), value=math.nan)
    leaves = {k: a.requires_grad_() for k, a in t.items() if a is not None}
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    out, final = scan_call(t, True, lens, return_final_state=True)
    assert torch.isinf(final[0, channel, 2]) and torch.isfinite(final).sum() == 10 * N - 1
    assert not torch.isfinite(out[0, channel, n - 1]) and torch.isfinite(out).sum() == 10 * L - 1
    grads = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), pgo)))
    units = 2 * ((n + 4) * (8 + 4 * float(v["weight"])) + 64)
    assert torch.isinf(grads["C"][0, 0, 2, n - 1])
    grads["C"][0, 0, 2, n - 1] = 0.0
    v["dC"][0, 0, 2, n - 1] = 0.0
    for k, gr in grads.items():
        if k in ("u", "delta", "B", "C"):
            assert not gr[..., n:].any(), k
            gr = gr[..., :n]
        check(gr, v[SCAN_GRADS[k]], m[SCAN_GRADS[k]], units, SCAN_GRADS[k])


@pytest.mark.parametrize("L,n", [(40, 13), (700, 655), (64, 33)])
@pytest.mark.parametrize("N", [4, 16, 40])
def test_scan_infinite_skip_and_final_gradient_leave_padding_at_0(L, n, N):
    c, go, gf, lens = scan_case(L + N, 1, 10, L, N, 1, torch.float32, lengths=[n])
    c["D"][0], gf[0, 1, 0] = math.inf, -math.inf
    t = {k: dev(a).requires_grad_() for k, a in c.items()}
    out, final = scan_call(t, True, dev(lens), return_final_state=True)
    grads = dict(zip(t, torch.autograd.grad([out, final], list(t.values()), [dev(go), dev(gf)])))
    for k in ("u", "delta", "z", "B", "C"):
        assert not grads[k][..., n:].any(), k
    for k in ("u", "delta", "z"):
        assert torch.isfinite(grads[k][0, 2:]).all(), k
    assert torch.isfinite(grads["A"][2:]).all() and torch.isfinite(grads["bias"][2:]).all()
    assert torch.isinf(grads["u"][0, 0, :n]).all() and torch.isinf(grads["init"][0, 1, 0])


def test_scan_states_that_grow_and_decay_within_a_tile():
    """Growth over a few tokens whose product overflows 32 bits, taken back
    within the same 16 tokens: zero states stay 0 and small ones come back."""
    c, go, _, _ = scan_case(6, 1, 8, 20, 4, 1, torch.float32, gate=False, bias=False)
    c["A"][:] = -1.0
    c["delta"][:] = 0.1
    c["delta"][..., 0:2], c["delta"][..., 2:4] = -70.0, 75.0
    c["u"][..., :4] = 0.0
    c["init"][:, ::2], c["init"][:, 1::2] = 0.0, 1e-30
    v, m = ref.scan(**{k: c[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")}, init=c["init"])
    t = {k: dev(a) for k, a in c.items()}
    out, final = scan_call(t, False, None, return_final_state=True)
    # (decays of exponents up to 75: each off by 75 roundings more than the general bound has)
    units = 24 * (8 + 4 * float(v["weight"]) + 75) + 64
    check(out, v["out"], m["out"], units, "out")
    check(final, v["final"], m["final"], units, "final")


@pytest.mark.parametrize("N", [1, 16])
def test_scan_long_sums_of_parameter_gradients(N):
    """dD of rows that are not cut (256 groups of a channel each): 65536 terms
    of one sign, the same in 32 bits here and in 64 there.  A lane adds at most
    16 terms of a tile in 32 bits, the tiles in 64, and at most 4 lanes are
    joined: 16 + 2 + 2 roundings of the sum.  One running sum in 32 bits would
    be off by about 256, as its roundings add up like a random walk."""
    ch, L = 256, 65536
    g = torch.Generator(device=DEV).manual_seed(1)
    u = torch.rand(1, ch, L, generator=g, device=DEV) + 0.5
    go = torch.rand(1, ch, L, generator=g, device=DEV) + 0.5
    D = torch.ones(ch, device=DEV, requires_grad=True)
    B = torch.zeros(1, ch, N, L, device=DEV)
    delta = torch.ones(1, ch, L, device=DEV)
    bias = torch.zeros(ch, device=DEV, requires_grad=True)
    out = pc.ssm_scan(u, delta, -torch.ones(ch, N, device=DEV), B, B + 1.0, D=D, delta_bias=bias,
                      initial_state=torch.zeros(1, ch, N, device=DEV))
    dD, db = torch.autograd.grad(out, [D, bias], go)
    exact = (go.double() * u.double()).sum((0, 2)).cpu()
    check(dD, exact, exact.abs(), 20, "dD")
    assert not db.any()  # (B and the states are 0)

