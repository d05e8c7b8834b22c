"""Group norm, linear attention and the AdamW step on arrays whose offsets pass
32 bits: the end of each against the formulas in 64 bits."""
import pytest
import torch

import test_attention_gpu as attention
import train_ref as ref
import paraconv2d_b200 as pc
from strict import strictly

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def room():
    free, _ = torch.cuda.mem_get_info()
    if free < 80 << 30:
        pytest.skip("needs 80 GB")
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("last", [False, True])
def test_norm(last):
    B, C, L, groups = 9, 8, (1 << 26) + 3, 4
    assert B * C * L > 1 << 32
    torch.manual_seed(0)
    shape = (B, L, C) if last else (B, C, L)
    x, d = (torch.randn(shape, device=DEV, dtype=BF16) for _ in range(2))
    if last:
        x, d = x.transpose(1, 2), d.transpose(1, 2)
    x.requires_grad_(True)
    out = pc.group_norm(x, groups, activation="silu")
    (dx,) = torch.autograd.grad(out, x, d)
    row = x.detach()[-1].double().reshape(groups, -1)  # (the whole last row is needed for its statistics)
    mean = row.mean(1, keepdim=True)
    rstd = 1 / ((row - mean).square().mean(1, keepdim=True) + 1e-5).sqrt()
    xhat = (row - mean) * rstd
    sig = torch.sigmoid(xhat)
    h = d[-1].double().reshape(groups, -1) * sig * (1 + xhat * (1 - sig))
    hw, hx = h.mean(1, keepdim=True), (h * xhat).mean(1, keepdim=True)
    for got, want, size in ((out[-1], xhat * sig, xhat.abs() + 1), (dx[-1], rstd * (h - hw - xhat * hx), h.abs() + 1)):
        # a rounding to bfloat16, and 32-bit roundings of the terms as for small arrays
        off = (got.detach().double().reshape(groups, -1) - want).abs()
        bad = ~(off <= want.abs() * 2.0 ** -8 * 1.001 + size * 256 * 2.0 ** -24)
        assert not bad.any(), int(bad.sum())


@pytest.mark.parametrize("last", [False, True])
def test_norm_of_long_rows(last):
    """1.3e8 values a group, 65,536 of them a thread: their sums are as good as short ones."""
    B, C, L = 20, 8, 1 << 24
    torch.manual_seed(3)
    shape = (B, L, C) if last else (B, C, L)
    x, d = (torch.randn(shape, device=DEV) for _ in range(2))
    if last:
        x, d = x.transpose(1, 2), d.transpose(1, 2)
    w, b = (torch.randn(C, device=DEV).requires_grad_(True) for _ in range(2))
    x.requires_grad_(True)
    out = pc.group_norm(x, 1, w, b)
    dx, dw, db = torch.autograd.grad(out, [x, w, b], d)
    sums = torch.zeros(4, C, device=DEV, dtype=torch.float64)
    w64, b64 = w.detach().double()[:, None], b.detach().double()[:, None]
    for i in range(B):
        row, h = x.detach()[i].double(), d[i].double()
        rstd = 1 / ((row - row.mean()).square().mean() + 1e-5).sqrt()
        xhat = (row - row.mean()) * rstd
        sums += torch.stack([(h * xhat).sum(1), h.sum(1), (h * xhat).abs().sum(1), h.abs().sum(1)])
        if i not in (0, B - 1):
            continue
        hw = h * w64
        pairs = [(out[i], xhat * w64 + b64, (xhat * w64).abs() + b64.abs()),
                 (dx[i], rstd * (hw - hw.mean() - xhat * (hw * xhat).mean()),
                  hw.abs() + hw.abs().mean() + xhat.abs() * (hw * xhat).abs().mean())]
        for got, want, size in pairs:  # 64 roundings of the terms' sizes, as for rows of any length
            bad = ~((got.detach().double() - want).abs() <= size * 64 * 2.0 ** -24)
            assert not bad.any(), (i, int(bad.sum()))
    for got, want, size in ((dw, sums[0], sums[2]), (db, sums[1], sums[3])):
        assert ((got.double() - want).abs() <= size * 64 * 2.0 ** -24).all()


def test_attention():
    H, dk, dv, L, tail = 2, 8, 128, (1 << 24) + 72, 1500
    assert H * dv * L > 1 << 32
    torch.manual_seed(1)
    q, k = (torch.randn(1, 1, dk, L, device=DEV, dtype=BF16) for _ in range(2))
    v, go = (torch.randn(1, H, dv, L, device=DEV, dtype=BF16) for _ in range(2))
    g = -0.1 - 0.1 * torch.rand(1, H, L, device=DEV)  # (what is 1000 tokens back weighs less than e^-100)
    leaves = [t.requires_grad_(True) for t in (q, k, v, g)]
    out = pc.linear_attention(*leaves)
    grads = torch.autograd.grad(out, leaves, go)
    cut = [t.detach()[..., -tail:] for t in leaves]
    want, size = ref.attention(*cut, grad=go[..., -tail:])
    close = strictly(attention.close)
    for got, key in zip((out, *grads), ("out", "dq", "dk", "dv", "dg")):
        part = attention.DECAY_PARTS[BF16] if key == "dg" else 2.0 ** -15
        close(got[..., -400:], want[key][..., -400:], size[key][..., -400:], part, 64, key)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw(bits):
    n, tail = (1 << 32) + 1000, 1000
    torch.manual_seed(2)
    p, g = (torch.randn(n, device=DEV, dtype=BF16) for _ in range(2))
    m, v, s = pc.adamw_new_state(p, bits)
    before = p[-tail:].cpu()
    pc.adamw_step([p], [g], [m], [v], torch.zeros(1, dtype=torch.int64, device=DEV), lr=0.1, weight_decay=0.1,
                  scales=None if s is None else [s])
    c = dict(params=[before], grads=[g[-tail:].cpu()], masters=None, scales=None, m=[torch.zeros(tail)], v=[torch.zeros(tail)])
    want = ref.adamw(c, 1, lr=0.1, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)[0]
    got = p[-tail:].cpu().double()
    tol = want["param"].abs() * 2.0 ** -8 * 1.001 + want["param_size"] * 12 * 2.0 ** -24
    assert ((got - want["param"]).abs() <= tol).all()
    if bits == 8:  # (the block that the tail begins in begins before it)
        first = (n - tail) // 256
        m, v = (t[0][-tail:].cpu().double() for t in
                pc.adamw_state_values([m[first * 256:]], [v[first * 256:]], [s[first:].contiguous()]))
    else:
        m, v = m[-tail:].cpu().double(), v[-tail:].cpu().double()
    # an 8-bit code is a step off at most, an eighth of a value or of the block's smallest normal number
    for got, name, binades in ((m, "m", 15), (v, "v", 31)):
        step = want[name].abs() / 8 + want[name].abs().max() * 2.0 ** -(binades - 2) / 8 if bits == 8 else 0
        assert ((got - want[name]).abs() <= step + want[name + "_size"] * 4 * 2.0 ** -24).all()
