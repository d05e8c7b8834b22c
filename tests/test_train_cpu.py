"""Group norm, linear attention and the AdamW step without a GPU: refusals,
registration, and the 64-bit references that the GPU tests compare with,
against autograd and against differences."""
import ctypes

import pytest
import torch

import train_ref as ref
import paraconv2d_b200 as pc
from paraconv2d_b200 import _lib

lib = _lib.cabi()
INVALID, UNSUPPORTED, WORKSPACE = _lib.PC2D_ERR_INVALID_ARGUMENT, _lib.PC2D_ERR_UNSUPPORTED, _lib.PC2D_ERR_WORKSPACE
ONE = 256  # any aligned address: nothing is launched


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------ the references

@pytest.mark.parametrize("silu", [False, True])
def test_norm_reference_against_autograd(silu):
    g = gen(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True)  # noqa: E731
    x, w, b = r(3, 6, 7), r(6), r(6)
    d = torch.randn(3, 6, 7, generator=g, dtype=torch.float64)
    lengths = [7, 0, 4]
    v, m = ref.norm(x, 2, w, b, 1e-3, silu, lengths, d)
    rows = []
    for i, n in enumerate(lengths):
        y = torch.zeros(1, 6, 7, dtype=torch.float64)
        if n:
            y = torch.nn.functional.group_norm(x[i:i + 1, :, :n], 2, w, b, 1e-3)
            y = torch.nn.functional.pad(torch.nn.functional.silu(y) if silu else y, (0, 7 - n))
        rows.append(y)
    out = torch.cat(rows)
    want = torch.autograd.grad((out * d).sum(), [x, w, b])
    assert torch.allclose(v["out"], out, atol=1e-12)
    for k, t in zip(("dx", "dw", "db"), want):
        assert torch.allclose(v[k], t, atol=1e-11), k
    for k in v:
        assert (m[k] >= v[k].abs() - 1e-12).all(), k


def _attention_case(g):
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    t = dict(q=r(2, 2, 3, 9), k=r(2, 2, 3, 9), v=r(2, 4, 5, 9), g=-r(2, 4, 9).abs(), init=r(2, 4, 3, 5))
    return t, r(2, 4, 5, 9), r(2, 4, 3, 5), [9, 4]


def _forward_attention(t, lengths):
    own, S, outs = torch.arange(4) // 2, t["init"], []
    for i in range(9):
        new = torch.exp(t["g"][:, :, i])[..., None, None] * S
        new = new + t["k"][:, own, :, i][..., None] * t["v"][:, :, None, :, i]
        on = torch.tensor(lengths)[:, None, None, None] > i
        S = torch.where(on, new, S)
        o = torch.einsum("bhk,bhkv->bhv", t["q"][:, own, :, i], S) * 3 ** -0.5
        outs.append(torch.where(on[..., 0], o, 0.0))
    return torch.stack(outs, -1), S


def test_attention_reference_against_autograd_and_differences():
    g = gen(2)
    t, go, gf, lengths = _attention_case(g)
    leaves = {k: x.clone().requires_grad_(True) for k, x in t.items()}
    out, final = _forward_attention(leaves, lengths)
    want = torch.autograd.grad((out * go).sum() + (final * gf).sum(), list(leaves.values()))
    v, m = ref.attention(**t, lengths=lengths, grad=go, grad_final=gf, chunk=4)
    assert torch.allclose(v["out"], out, atol=1e-12) and torch.allclose(v["final"], final, atol=1e-12)
    keys = ("dq", "dk", "dv", "dg", "dinit")
    for k, x in zip(keys, want):
        assert torch.allclose(v[k], x, atol=1e-11), k
    for k in v:
        assert (m[k] >= v[k].abs() - 1e-12).all(), k
    step = 1e-5
    for name, key in zip(t, keys):
        way = torch.randn(t[name].shape, generator=g, dtype=torch.float64)
        ends = []
        for s in (1, -1):
            o, f = _forward_attention({**t, name: t[name] + s * step * way}, lengths)
            ends.append((o * go).sum() + (f * gf).sum())
        slope = float(ends[0] - ends[1]) / (2 * step)
        assert abs(slope - float((v[key] * way).sum())) <= 1e-6 * (1 + float((v[key] * way).abs().sum())), name


def test_adamw_reference_against_torch():
    g = gen(3)
    p = torch.nn.Parameter(torch.randn(50, generator=g, dtype=torch.float64))
    opt = torch.optim.AdamW([p], lr=1e-2, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.3)
    c = dict(params=[p.detach().clone()], masters=None, scales=None, m=[torch.zeros(50).double()], v=[torch.zeros(50).double()])
    for t in range(1, 4):
        p.grad = torch.randn(50, generator=g).double()
        opt.step()
        o = ref.adamw({**c, "grads": [p.grad]}, t, 1e-2, (0.8, 0.95), 1e-6, 0.3)[0]
        c.update(params=[o["param"]], m=[o["m"]], v=[o["v"]])
        assert torch.allclose(o["param"], p.detach(), atol=1e-13)


@pytest.mark.parametrize("signed", [True, False])
@pytest.mark.parametrize("size", [1.0, 1e-37, 1e30, 1e-41, 0.0])
def test_8_bit_values(signed, size):
    """A code's value is within a step of what it stands for, and the codes keep their order."""
    g = gen(4)
    x = torch.randn(700, generator=g) * torch.exp(4 * torch.randn(700, generator=g)) * size
    x = x if signed else x.abs()
    low = torch.randint(0, 256, (700,), generator=g)
    code, scale = ref.adamw_encode(x, low, signed)
    back = ref.adamw_decode(code, scale, signed)
    least = torch.exp2(scale.double() - 127).repeat_interleave(256)[:700]
    step = torch.maximum(x.double().abs(), least) / 8
    assert ((back - x.double()).abs() <= step).all()
    if not signed:
        assert ((back > 0) == (x > 0)).all()
        whole = torch.arange(256, dtype=torch.uint8)
        values = ref.adamw_decode(whole, torch.tensor([100], dtype=torch.uint8), False)
        assert (values[1:] > values[:-1]).all()


# ------------------------------------------------------------------ refusals

def test_ops_are_registered_without_a_cpu_kernel():
    x = torch.zeros(2, 4, 3)
    with pytest.raises(NotImplementedError):
        pc.group_norm(x, 2)
    q = torch.zeros(2, 2, 4, 3)
    with pytest.raises(NotImplementedError):
        pc.linear_attention(q, q, q, torch.zeros(2))
    with pytest.raises(NotImplementedError):
        pc.linear_attention_step(q[..., 0], q[..., 0], q[..., 0], torch.zeros(2), torch.zeros(2, 2, 4, 4))
    with pytest.raises(NotImplementedError):
        pc.adamw_step([x], [x], [x], [x], torch.zeros(1, dtype=torch.int64), lr=0.1)
    p = torch.nn.Parameter(x)
    p.grad = x
    with pytest.raises(NotImplementedError):
        pc.ParaboloidAdamW([p]).step()
    ops = torch.ops.paraconv2d_b200
    assert "Tensor(a!) state" in str(ops.linear_attention_step.default._schema)
    assert "Tensor(a!)[] params" in str(ops.adamw_step.default._schema)


def test_python_refusals():
    with pytest.raises(ValueError):
        pc.group_norm(torch.zeros(2, 4, 3), 2, activation="gelu")
    with pytest.raises(ValueError):
        pc.GroupNorm(3, 4)
    with pytest.raises(ValueError):
        pc.LinearAttention(2, 129, 4)
    with pytest.raises(RuntimeError, match="no backward"):
        q = torch.zeros(2, 2, 4)
        pc.linear_attention_step(q, q, q, torch.zeros(2, requires_grad=True), torch.zeros(2, 2, 4, 4))
    p = [torch.nn.Parameter(torch.zeros(3))]
    for bad in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0), dict(weight_decay=-0.1), dict(state_bits=16)):
        with pytest.raises(ValueError):
            pc.ParaboloidAdamW(p, **bad)
    with pytest.raises(ValueError):
        pc.adamw_new_state(torch.zeros(3), bits=4)
    m, v, s = pc.adamw_new_state(torch.zeros(3, 100), bits=8)
    assert m.shape == v.shape == (300,) and s.shape == (2, 2) and m.dtype == s.dtype == torch.uint8


NORM = dict(dtype=0, wdtype=0, batch=2, channels=6, length=5, groups=3)


@pytest.mark.parametrize("args,code", [
    (dict(dtype=1, wdtype=1), INVALID), (dict(wdtype=3), INVALID), (dict(dtype=2, wdtype=3), INVALID),
    (dict(groups=4), INVALID), (dict(groups=0), INVALID), (dict(channels=0), INVALID), (dict(batch=-1), INVALID),
    (dict(length=2 ** 31 - 1), UNSUPPORTED), (dict(channels=8193, groups=1), UNSUPPORTED),
    (dict(batch=2 ** 24), UNSUPPORTED), (dict(), INVALID), (dict(batch=0), 0), (dict(length=0), 0),
])
def test_norm_refusals(args, code):
    a = {**NORM, **args}
    sizes = (a["batch"], a["channels"], a["length"], a["groups"])
    n = None
    assert lib.pc2d_group_norm_forward(a["dtype"], a["wdtype"], 0, n, n, n, n, *sizes, 1e-5, 1, n, n, n, 0, n) == code
    if code:  # (an empty backward pass clears the weights' gradients)
        assert lib.pc2d_group_norm_backward(a["dtype"], a["wdtype"], 0, n, n, n, n, n, n, *sizes, 1, n, n, n, n, 0, n) == code


def test_norm_workspaces():
    # one group for the whole GPU: two launches that share sums in the workspace
    need = lib.pc2d_group_norm_workspace_size(0, 0, 1, 64, 1 << 16, 1, 0)
    assert need > 0
    st = lib.pc2d_group_norm_forward(0, 0, 0, ONE, ONE, ONE, None, 1, 64, 1 << 16, 1, 1e-5, 0, ONE, None, ONE, need - 256,
                                     None)
    assert st == WORKSPACE
    need = lib.pc2d_group_norm_workspace_size(0, 1, 2, 6, 5, 3, 1)
    assert need >= 2 * 6 * 8  # a sum of each kind for each channel of a row
    st = lib.pc2d_group_norm_backward(0, 0, 1, ONE, ONE, ONE, ONE, None, ONE, 2, 6, 5, 3, 1, ONE, ONE, ONE, ONE, need - 1,
                                      None)
    assert st == WORKSPACE
    assert lib.pc2d_group_norm_forward(0, 0, 0, ONE, ONE, ONE, None, 2, 6, 5, 3, -1.0, 0, ONE, None, None, 0, None) == INVALID
    # arrays off their elements' boundary
    assert lib.pc2d_group_norm_forward(0, 0, 0, ONE + 2, ONE, ONE, None, 2, 6, 5, 3, 1e-5, 0, ONE, None, None, 0,
                                       None) == INVALID


ATTENTION = dict(dtype=0, batch=2, heads=4, groups=2, length=5, dk=8, dv=16, scale=1.0)


@pytest.mark.parametrize("args,code", [
    (dict(dtype=1), INVALID), (dict(heads=0), INVALID), (dict(groups=3), INVALID), (dict(groups=0), INVALID),
    (dict(dk=0), INVALID), (dict(dv=0), INVALID), (dict(dk=129), UNSUPPORTED), (dict(dv=129), UNSUPPORTED),
    (dict(batch=-1), INVALID), (dict(length=-1), INVALID), (dict(length=2 ** 31 - 1), UNSUPPORTED),
    (dict(batch=2 ** 20), UNSUPPORTED), (dict(scale=float("nan")), INVALID), (dict(), INVALID), (dict(batch=0), 0),
])
def test_attention_refusals(args, code):
    a = {**ATTENTION, **args}
    n = None
    sizes = (a["batch"], a["heads"], a["groups"], a["length"], a["dk"], a["dv"])
    assert lib.pc2d_linear_attention_forward(a["dtype"], n, n, n, n, 0, n, n, *sizes, a["scale"], n, n, n, n, 0, n) == code
    if "length" not in args:
        assert lib.pc2d_linear_attention_step(a["dtype"], n, n, n, n, 0, n, n, a["batch"], max(0, a["batch"]), a["heads"],
                                              a["groups"], a["dk"], a["dv"], a["scale"], n, n) == code


def test_attention_workspaces():
    long = (0, ONE, ONE, ONE, ONE, 0, None, None, 1, 1, 1, 4096, 16, 16, 1.0)
    need = lib.pc2d_linear_attention_workspace_size(0, 1, 1, 1, 4096, 16, 16, 0)
    assert need > 0  # a sequence of one head goes by segments, whose states are in the workspace
    assert lib.pc2d_linear_attention_forward(*long, ONE, None, None, ONE, need - 256, None) == WORKSPACE
    assert lib.pc2d_linear_attention_forward(*long, ONE, None, ONE + 4, ONE, need, None) == INVALID  # kept states off 16 bytes
    need = lib.pc2d_linear_attention_workspace_size(0, 2, 4, 2, 5, 8, 16, 1)
    assert need >= lib.pc2d_linear_attention_states_size(0, 2, 4, 5, 8, 16) == 2 * 4 * 8 * 16 * 4
    back = (0, ONE, None, ONE, ONE, ONE, ONE, 0, ONE, None, 2, 4, 2, 5, 8, 16, 1.0, ONE, ONE, ONE, ONE, None)
    assert lib.pc2d_linear_attention_backward(*back, ONE, need - 1, None) == WORKSPACE
    none = back[:8] + (None,) + back[9:]
    assert lib.pc2d_linear_attention_backward(*none, ONE, need, None) == INVALID
    # a step of more rows than states, and a state off its boundary
    step = (0, ONE, ONE, ONE, ONE, 0)
    assert lib.pc2d_linear_attention_step(*step, ONE, None, 3, 2, 4, 2, 8, 16, 1.0, ONE, None) == INVALID
    assert lib.pc2d_linear_attention_step(*step, ONE + 4, None, 2, 2, 4, 2, 8, 16, 1.0, ONE, None) == INVALID


def _tensor(**kw):
    t = _lib.AdamWTensor(dtype=0, grad_dtype=0, param=ONE, grad=ONE, exp_avg=ONE, exp_avg_sq=ONE, n=8, split=8, rate_first=1.0,
                         rate_rest=1.0, decay=1.0)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


@pytest.mark.parametrize("bits,tensor,call,code", [
    (16, {}, {}, INVALID), (32, dict(dtype=1, grad_dtype=1), {}, INVALID), (32, dict(grad_dtype=2), {}, INVALID),
    (32, dict(n=-1), {}, INVALID), (32, dict(n=2 ** 35), {}, INVALID), (32, dict(split=-1), {}, INVALID),
    (32, dict(param=None), {}, INVALID), (32, dict(grad=None), {}, INVALID), (8, {}, {}, INVALID),
    (32, dict(param=ONE + 2), {}, INVALID), (32, dict(exp_avg=ONE + 1), {}, INVALID), (32, dict(master=ONE), {}, INVALID),
    (32, dict(rate_rest=float("inf")), {}, INVALID), (32, dict(decay=float("nan")), {}, INVALID),
    (32, {}, dict(lr=-1.0), INVALID), (32, {}, dict(beta1=1.0), INVALID), (32, {}, dict(beta2=-0.1), INVALID),
    (32, {}, dict(eps=float("nan")), INVALID), (32, {}, dict(step=None), INVALID), (32, {}, dict(bytes=8), WORKSPACE),
])
def test_adamw_refusals(bits, tensor, call, code):
    c = dict(step=ONE, lr=0.1, beta1=0.9, beta2=0.99, eps=1e-8, decay=0.1, bytes=64)
    c.update(call)
    st = lib.pc2d_adamw_step(bits, ctypes.byref(_tensor(**tensor)), 1, c["step"], None, c["lr"], c["beta1"], c["beta2"],
                             c["eps"], c["decay"], None, 0, ONE, c["bytes"], None)
    assert st == code
    assert lib.pc2d_adamw_workspace_size() <= 64


def test_adamw_values_refusals():
    ptrs = (ctypes.c_void_p * 1)(ONE)
    none = (ctypes.c_void_p * 1)(None)
    good = _tensor(scales=ONE)
    assert lib.pc2d_adamw_state_values(2, ctypes.byref(good), 1, ptrs, ptrs, None) == INVALID
    assert lib.pc2d_adamw_state_values(0, ctypes.byref(_tensor()), 1, ptrs, ptrs, None) == INVALID
    assert lib.pc2d_adamw_state_values(0, ctypes.byref(good), 1, none, ptrs, None) == INVALID
    assert lib.pc2d_adamw_state_values(0, None, 1, ptrs, ptrs, None) == INVALID


def test_module_parameters():
    m = pc.LinearAttention(8, 16, 32)
    keep = torch.exp(m._log_decay().detach())
    assert torch.allclose(1 - keep, torch.exp2(-torch.linspace(5, 12, 8)), rtol=1e-3)
    assert m.new_state(3).shape == (3, 8, 16, 32)
    n = pc.GroupNorm(2, 6)
    assert n.weight.eq(1).all() and not n.bias.any()
    assert pc.GroupNorm(2, 6, affine=False).weight is None
