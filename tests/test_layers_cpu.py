"""The layers beside ParaConv2d without a GPU: refusals, registration, and the
64-bit references that the GPU tests compare with, against autograd and
against differences."""
import pytest
import torch

import layers_ref as ref
import paraconv2d_b200 as pc
from paraconv2d_b200 import _lib

lib = _lib.cabi()
INVALID, UNSUPPORTED, WORKSPACE = _lib.PC2D_ERR_INVALID_ARGUMENT, _lib.PC2D_ERR_UNSUPPORTED, _lib.PC2D_ERR_WORKSPACE


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------ the references

def test_philox_known_answers():
    """The generator's published known answers (zeros; all ones)."""
    assert ref.philox((0, 0, 0, 0), (0, 0)) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    ones = 0xFFFFFFFF
    assert ref.philox((ones,) * 4, (ones,) * 2) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]


def _autograd_conv(x, w, b, silu, init, lengths):
    K = w.shape[1]
    outs, finals = [], []
    for i in range(x.shape[0]):
        n = x.shape[2] if lengths is None else int(lengths[i])
        line = torch.cat([init[i], x[i, :, :n]], -1)
        pre = sum(w[:, k, None] * line[:, k:k + n] for k in range(K)) + b[:, None]
        out = torch.nn.functional.silu(pre) if silu else pre
        outs.append(torch.nn.functional.pad(out, (0, x.shape[2] - n)))
        finals.append(line[:, n:])
    return torch.stack(outs), torch.stack(finals)


@pytest.mark.parametrize("K", [1, 2, 4])
@pytest.mark.parametrize("silu", [False, True])
def test_conv_reference_against_autograd(K, silu):
    g = gen(1)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True) for s in ((3, 2, 7), (2, K), (2,)))
    init = torch.randn(3, 2, K - 1, generator=g, dtype=torch.float64, requires_grad=True)
    lengths = torch.tensor([7, 0, 2])
    go, gf = torch.randn(3, 2, 7, generator=g, dtype=torch.float64), torch.randn(3, 2, K - 1, generator=g, dtype=torch.float64)
    out, final = _autograd_conv(x, w, b, silu, init, lengths)
    loss = (out * go).sum() + (final * gf).sum()
    want = torch.autograd.grad(loss, [x, w, b, init], allow_unused=True)
    v, _ = ref.conv(x, w, b, silu, init, lengths, go, gf)
    assert torch.allclose(v["out"], out, atol=1e-13) and torch.allclose(v["final"], final, atol=1e-13)
    for n, t in zip(("dx", "dw", "db", "dinit"), want):
        assert torch.allclose(v[n], t if t is not None else torch.zeros_like(v[n]), atol=1e-12), n


def _scan_case(g, dtype=torch.float64):
    nb, ch, L, N, G = 3, 4, 9, 3, 2
    r = lambda *s: torch.randn(*s, generator=g, dtype=dtype)  # noqa: E731
    t = dict(u=r(nb, ch, L), delta=r(nb, ch, L), A=-torch.rand(ch, N, generator=g, dtype=dtype) - 0.1, B=r(nb, G, N, L),
             C=r(nb, G, N, L), D=r(ch), z=r(nb, ch, L), bias=r(ch), init=r(nb, ch, N))
    return t, r(nb, ch, L), r(nb, ch, N), torch.tensor([9, 0, 4])


def _forward_scan(t, lengths):
    """The forward pass alone, for autograd and for differences."""
    nb, ch, L = t["u"].shape
    G, N = t["B"].shape[1:3]
    d = torch.nn.functional.softplus(t["delta"] + t["bias"][:, None], threshold=1e9)
    owner = torch.arange(ch) // (ch // G)
    h, outs = t["init"], []
    for s in range(L):
        new = torch.exp(d[:, :, s, None] * t["A"]) * h + (d * t["u"])[:, :, s, None] * t["B"][:, owner, :, s]
        on = s < lengths
        h = torch.where(on[:, None, None], new, h)
        y = (h * t["C"][:, owner, :, s]).sum(-1) + t["D"] * t["u"][..., s]
        outs.append(torch.where(on[:, None], y * torch.nn.functional.silu(t["z"][..., s]), 0.0))
    return torch.stack(outs, -1), h


GRADS = dict(u="du", delta="dd", A="dA", B="dB", C="dC", D="dD", z="dz", bias="dbias", init="dinit")


def test_scan_reference_against_autograd_and_differences():
    g = gen(2)
    t, go, gf, lengths = _scan_case(g)
    leaves = {k: v.clone().requires_grad_(True) for k, v in t.items()}
    out, final = _forward_scan(leaves, lengths)
    loss = (out * go).sum() + (final * gf).sum()
    want = dict(zip(leaves, torch.autograd.grad(loss, list(leaves.values()))))
    v, _ = ref.scan(**{k: t[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")}, softplus=True,
                    init=t["init"], lengths=lengths, grad=go, grad_final=gf)
    assert torch.allclose(v["out"], out, atol=1e-12) and torch.allclose(v["final"], final, atol=1e-12)
    for name, key in GRADS.items():
        assert torch.allclose(v[key], want[name], atol=1e-11), name
    # central differences along a direction: the error is of the order of step^2
    step = 1e-5
    for name, key in GRADS.items():
        way = torch.randn(t[name].shape, generator=g, dtype=torch.float64)
        ends = []
        for sign in (1, -1):
            o, f = _forward_scan({**t, name: t[name] + sign * step * way}, lengths)
            ends.append((o * go).sum() + (f * gf).sum())
        slope = float(ends[0] - ends[1]) / (2 * step)
        assert abs(slope - float((v[key] * way).sum())) <= 1e-6 * (1 + float((v[key] * way).abs().sum())), name


# ------------------------------------------------------------------ refusals

def test_layer_ops_are_registered_without_a_cpu_kernel():
    x = torch.zeros(2, 3, 4)
    with pytest.raises(NotImplementedError):
        pc.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(NotImplementedError):
        pc.causal_conv(x, torch.zeros(3, 4))
    with pytest.raises(NotImplementedError):
        pc.ssm_scan(x, x, torch.zeros(3, 1), torch.zeros(2, 1, 1, 4), torch.zeros(2, 1, 1, 4))
    assert "Tensor(a!) state" in str(torch.ops.paraconv2d_b200.ssm_scan_step.default._schema)
    assert "Tensor(a!) state" in str(torch.ops.paraconv2d_b200.causal_conv_step.default._schema)


def test_python_refusals():
    x = torch.zeros(2, 3, 4)
    with pytest.raises(ValueError):
        pc.causal_conv(x, torch.zeros(3, 4), activation="relu")
    with pytest.raises(ValueError):
        pc.Dropout(1.5)
    with pytest.raises(ValueError):
        pc.CausalConv(4, taps=9)
    with pytest.raises(ValueError):
        pc.SSMScan(4, states=129)
    state = torch.zeros(2, 3, 3)
    with pytest.raises(RuntimeError, match="no backward"):
        pc.causal_conv_step(x[..., 0], state, torch.zeros(3, 4, requires_grad=True))


@pytest.mark.parametrize("args,code", [
    (dict(dtype=7), INVALID), (dict(dtype=-1), INVALID), (dict(p=-0.1), INVALID), (dict(p=1.1), INVALID),
    (dict(p=float("nan")), INVALID), (dict(n=-1), INVALID), (dict(), INVALID), (dict(n=0), 0),
])
def test_dropout_refusals(args, code):
    a = dict(dtype=0, p=0.5, n=8)
    a.update(args)
    assert lib.pc2d_dropout(a["dtype"], None, None, None, a["p"], a["n"], None, None) == code


CONV = dict(dtype=0, wdtype=0, batch=2, channels=3, length=5, taps=4)


@pytest.mark.parametrize("args,code", [
    (dict(dtype=1, wdtype=1), INVALID), (dict(wdtype=2), INVALID), (dict(dtype=3, wdtype=2), INVALID),
    (dict(taps=0), INVALID), (dict(taps=9), UNSUPPORTED), (dict(batch=-1), INVALID), (dict(length=-1), INVALID),
    (dict(length=2 ** 31 - 1), UNSUPPORTED), (dict(), INVALID), (dict(batch=0), 0),
])
def test_conv_refusals(args, code):
    a = {**CONV, **args}
    sizes = (a["batch"], a["channels"], a["length"], a["taps"], 1)
    assert lib.pc2d_causal_conv_forward(a["dtype"], a["wdtype"], None, None, None, None, None, *sizes, None, None,
                                        None) == code
    if "length" not in args:
        places = max(0, a["batch"])
        assert lib.pc2d_causal_conv_step(a["dtype"], a["wdtype"], None, None, None, None, None, a["batch"], places,
                                         a["channels"], a["taps"], 1, None, None) == code


def test_conv_backward_refuses_a_short_workspace():
    need = lib.pc2d_causal_conv_backward_workspace_size(2, 3, 5, 4)
    assert need >= 2 * 3 * 5 * 4  # a share for each row, tap and bias
    one = 256  # any aligned address: nothing is launched
    st = lib.pc2d_causal_conv_backward(0, 0, one, None, one, one, None, None, None, 2, 3, 5, 4, 1, one, one, None, None,
                                       one, need - 1, None)
    assert st == WORKSPACE
    st = lib.pc2d_causal_conv_backward(0, 0, one + 4, None, one, one, None, None, None, 2, 3, 5, 4, 1, one, one, None,
                                       None, one, need, None)
    assert st == INVALID  # not on a 16-byte boundary


SCAN = dict(dtype=0, batch=2, channels=4, length=5, states=16, groups=2)


@pytest.mark.parametrize("args,code", [
    (dict(dtype=1), INVALID), (dict(states=0), INVALID), (dict(states=129), UNSUPPORTED), (dict(groups=3), INVALID),
    (dict(groups=0), INVALID), (dict(batch=-1), INVALID), (dict(length=2 ** 31 - 1), UNSUPPORTED), (dict(), INVALID),
    (dict(batch=0), 0),
])
def test_scan_refusals(args, code):
    a = {**SCAN, **args}
    sizes = (a["batch"], a["channels"], a["length"], a["states"], a["groups"])
    n = None
    assert lib.pc2d_ssm_scan_forward(a["dtype"], n, n, n, n, n, n, n, n, n, n, 1, *sizes, n, n, n, n, 0, n) == code
    if "length" not in args:
        assert lib.pc2d_ssm_scan_step(a["dtype"], n, n, n, n, n, n, n, n, n, n, 1, a["batch"], max(0, a["batch"]),
                                      a["channels"], a["states"], a["groups"], n, n) == code


def test_step_refuses_more_rows_than_states():
    one = 256
    assert lib.pc2d_ssm_scan_step(0, one, one, one, one, one, one, None, None, None, None, 1, 3, 2, 4, 16, 1, one,
                                  None) == INVALID
    assert lib.pc2d_causal_conv_step(0, 0, one, one, one, None, None, 3, 2, 4, 4, 1, one, None) == INVALID
    # (one tap keeps nothing, but a row still needs its place)
    assert lib.pc2d_causal_conv_step(0, 0, one, None, one, None, None, 3, 2, 4, 1, 1, one, None) == INVALID


def test_scan_backward_refuses_a_short_workspace():
    need = lib.pc2d_ssm_scan_backward_workspace_size(2, 4, 5, 16, 2)
    one = 256
    p = [one] * 40
    st = lib.pc2d_ssm_scan_backward(0, one, None, one, one, one, one, one, None, None, None, None, one, 1, 2, 4, 5, 16,
                                    2, one, one, one, one, one, None, None, None, None, one, need - 1, None)
    assert st == WORKSPACE and p
    # without the checkpoints of a forward pass
    st = lib.pc2d_ssm_scan_backward(0, one, None, one, one, one, one, one, None, None, None, None, None, 1, 2, 4, 5,
                                    16, 2, one, one, one, one, one, None, None, None, None, one, need, None)
    assert st == INVALID


def test_other_entry_points_refuse_the_layers_types():
    """float16 and bfloat16 exist for the sequence operators only."""
    for dtype in (2, 3):
        assert lib.pc2d_pad_scale(dtype, None, 1, 1, 1, 1, 0, 0, 0, 0, 1.0, None, None) == INVALID
        assert lib.pc2d_param_step(dtype, None, None, None, 1, 1, 0.1, 1.0, 1.0, 0.0, 1.0, 0.0, 1, None) == INVALID
        assert lib.pc2d_forward(dtype, None, None, 1.0, 3, 3, 1, 1, 1, 1, 1, 3, 8, 8, 2, None, None, None, 0,
                                None) == INVALID


def test_module_parameters():
    m = pc.SSMScan(6, states=5)
    steps = torch.nn.functional.softplus(m.delta_bias.detach())
    assert float(steps.min()) >= 0.00099 and float(steps.max()) <= 0.101
    assert torch.allclose(torch.exp(m.A_log.detach()), torch.arange(1, 6).float().expand(6, 5), rtol=1e-6)
    assert m.new_state(3).shape == (3, 6, 5)
    c = pc.CausalConv(6, taps=3, activation="silu")
    assert c.weight.shape == (6, 3) and c.new_state(2).shape == (2, 6, 2)
    d = pc.Dropout(0.3, seed=-4).eval()
    x = torch.randn(3)
    assert d(x) is x and torch.equal(d(x, residual=x), x + x)
    assert d.state_dict()["state"].tolist() == [-4, 0]
