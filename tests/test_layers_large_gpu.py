"""The layers beside ParaConv2d on the GPU in the forms that their kernels take
for many rows, long runs and many blocks, which the small cases of
test_layers_gpu.py do not reach, and errors in norm.

Which form a call takes goes by its sizes and by the GPU's 148 SMs; the sizes
here are beyond the rules' borders for that number.  Tolerances as in
test_layers_gpu.py, unless said at the test.
"""
import pytest
import torch

import layers_ref as ref
import paraconv2d_b200 as pc
from test_layers_gpu import DEV, SCAN_GRADS, TYPES, conv_case, conv_check, dev, scan_call, scan_case, scan_check

pytestmark = pytest.mark.gpu

U32 = ref.U32


# ------------------------------------------------- forms for many and for few

@pytest.mark.parametrize("L", [2048, 2049])
@pytest.mark.parametrize("K", [1, 2, 4, 8])
def test_conv_runs_of_many_vectors(L, K):
    """2400 rows: a warp goes through 160 vectors, forwards two of them a lane
    at a time without checks, backwards with its carry from 32 to 32."""
    conv_check(*conv_case(L + K, 4, 600, L, K, torch.bfloat16 if K == 4 else torch.float32), silu=K != 2)


@pytest.mark.parametrize("L", [2048, 2045])
def test_conv_runs_of_many_vectors_in_ragged_rows(L):
    conv_check(*conv_case(L, 6, 401, L, 4, torch.float16, lengths=[L, 0, 1287, 1280, 1281, 2047]), silu=True)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("nb,ch,L,N,G", [(5, 1920, 72, 16, 1), (5, 1920, 67, 16, 2), (4, 1200, 40, 24, 1),
                                         (4, 1201, 41, 24, 1), (3, 100, 70, 10, 100)])
def test_scan_many_blocks(dtype, nb, ch, L, N, G):
    """300 blocks and more: the forward pass's layout for four blocks per SM."""
    scan_check(*scan_case(ch + L, nb, ch, L, N, G, TYPES[dtype]))


@pytest.mark.parametrize("N", [16, 24])
@pytest.mark.parametrize("L", [72, 67])
def test_scan_many_blocks_of_ragged_rows(N, L):
    scan_check(*scan_case(N + L, 6, 1667, L, N, 1, torch.float16, lengths=[L, 0, 33, 1, 64, 40]))


@pytest.mark.parametrize("ch,L,N", [(256, 20, 16), (520, 21, 16), (1024, 21, 3), (2050, 21, 3), (64, 20, 128),
                                    (33, 17, 128), (130, 9, 33)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_scan_shares_of_many_blocks(ch, L, N, dtype):
    """dB and dC from 8 blocks of a group and more, which several threads of
    the sum share, by vectors of four and one by one."""
    scan_check(*scan_case(ch + L, 2, ch, L, N, 1, TYPES[dtype]))


@pytest.mark.parametrize("N,L,lengths", [(3, 700, None), (3, 701, [701, 300]), (64, 515, None), (128, 400, None),
                                         (128, 401, [401, 260, 1]), (40, 1024, None)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_scan_in_segments_of_other_layouts(N, L, lengths, dtype):
    nb = 1 if lengths is None else len(lengths)
    scan_check(*scan_case(N + L, nb, 40, L, N, 1, TYPES[dtype], lengths=lengths))


# -------------------------------------------------------------- errors in norm

@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("nb,ch,L,N,G,lengths", [
    (2, 40, 130, 16, 1, None), (1, 40, 1000, 16, 1, None), (2, 300, 64, 64, 2, None), (1, 35, 515, 6, 1, None),
    (3, 70, 300, 24, 1, [300, 129, 7]), (1, 2000, 128, 16, 1, None)])
def test_scan_errors_in_norm(dtype, nb, ch, L, N, G, lengths):
    """The bounds of the other tests are for the worst case and grow with the
    length.  Over a whole output roundings add up like squares: a value has
    about 30 of its own (4 of the step and what softplus' argument adds, those
    of the decay's exponent, gate, sums), and those of the few tokens that a
    state remembers here: 84 units of 2^-24 (5e-6) in norm, and half a step of
    the output's type."""
    c, go, gf, lens = scan_case(nb + ch + L, nb, ch, L, N, G, TYPES[dtype], lengths=lengths)
    v, _ = ref.scan(**{k: c[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")}, softplus=True,
                    init=c["init"], lengths=lens, grad=go, grad_final=gf)
    t = {k: dev(a).requires_grad_() for k, a in c.items()}
    out, final = scan_call(t, True, dev(lens), return_final_state=True)
    grads = torch.autograd.grad([out, final], list(t.values()), [dev(go), dev(gf)])
    got = dict(out=out, final=final, **{SCAN_GRADS[k]: g for k, g in zip(t, grads)})
    for name, g in got.items():
        own = torch.finfo(g.dtype).eps / 2 if g.dtype != torch.float32 else 0.0
        error = float((g.detach().cpu().double() - v[name]).norm() / v[name].norm())
        assert error <= own + 84 * U32, f"{name}: {error:.3g}"


@pytest.mark.parametrize("G", [1, 256], ids=["in segments", "uncut"])
@pytest.mark.parametrize("N", [4, 16])
@pytest.mark.parametrize("rate", [2e-4, 5e-5, 1e-5])
def test_scan_slow_decays_are_not_biased(G, N, rate):
    """States that remember 5000 tokens and more.  The hardware's exponential is low by
    up to 0.8 units of 2^-24 on average; without the tiles' correction the mean
    error of the states would be hundreds of them.  With it a token's share
    meets at most 31 uncorrected decays, 16 on average: 13 units.  The tiles'
    own factors (an interpolation that is off by 0.01 units and a coefficient's
    rounding by 0.02, over 160 tiles) add 5, what the states' roundings leave
    in the mean of 1024 states and more 4: 22 in all, 32 allowed; the gradient
    of the first state meets whole tiles only."""
    ch, L = 256, 16384
    g = torch.Generator(device=DEV).manual_seed(N)
    A = -(torch.rand(ch, N, generator=g, device=DEV) + 0.5) * rate
    d = torch.rand(1, ch, L, generator=g, device=DEV) + 0.5
    ones = torch.ones(1, ch, L, device=DEV)
    B = torch.ones(1, G, N, L, device=DEV)
    init = torch.zeros(1, ch, N, device=DEV, requires_grad=True)
    out, final = pc.ssm_scan(ones, d, A, B, B, initial_state=init, return_final_state=True)
    first, = torch.autograd.grad(final, init, torch.ones_like(final))
    total = d[0].double().cumsum(-1)
    rest = total[:, -1:] - total
    exact = torch.stack([(d[0].double() * torch.exp(A[:, n, None].double() * rest)).sum(-1) for n in range(N)], -1)
    mean = float(((final[0].detach().double() - exact) / exact).mean()) / U32
    assert abs(mean) <= 32, f"states off by {mean:.3g} units on average"
    exact = torch.exp(A.double() * total[:, -1:])
    mean = float(((first[0].double() - exact) / exact).mean()) / U32
    assert abs(mean) <= 32, f"gradients off by {mean:.3g} units on average"


@pytest.mark.parametrize("G", [1, 256], ids=["in segments", "uncut"])
@pytest.mark.parametrize("N", [4, 16])
@pytest.mark.parametrize("rate", [2e-4, 5e-5, 1e-5])
def test_scan_slow_growth_is_not_biased(G, N, rate):
    """The same with A > 0: states that grow by up to e^5 over the row, whose
    tokens all stay remembered.  The bounds are those of slow decays."""
    test_scan_slow_decays_are_not_biased(G, N, -rate)
