"""Group norm on the GPU against its formulas in 64 bits on the CPU."""
import pytest
import torch

import train_ref as ref
import paraconv2d_b200 as pc

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def close(got, want, size, what):
    # The sums behind a value run over chains of at most a few thousand terms per thread, whose roundings add up
    # like a walk: 64 roundings of the terms' size cover them with the joins, the root and the activation's functions.
    tol = size * 64 * 2.0 ** -24
    if got.dtype != F32:
        tol = tol + want.abs() * (torch.finfo(got.dtype).eps / 2) * 1.001 + (2.0 ** -25 if got.dtype == F16 else 0)
    bad = (got.detach().cpu().double() - want).abs() > tol
    assert not bad.any(), (what, int(bad.sum()), got.detach().cpu()[bad][:3], want[bad][:3], tol[bad][:3])


def run(x, groups, w, b, silu, lengths=None, eps=1e-5, grad=None):
    leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    out = pc.group_norm(x, groups, w, b, eps=eps, activation="silu" if silu else None, lengths=lengths)
    return out, torch.autograd.grad(out, leaves, grad)


def check(shape, groups, dtype, last, silu=True, wdtype=None, affine=True, lengths=None, seed=0, offset=3.0, eps=1e-5):
    g = gen(seed)
    C = shape[1]
    x = torch.randn(shape, generator=g) + offset * torch.randn(1, C, *[1] * (len(shape) - 2), generator=g)
    d = torch.randn(shape, generator=g)
    w, b = torch.randn(C, generator=g), torch.randn(C, generator=g)
    x, d = x.to(dtype), d.to(dtype)
    w, b = (t.to(wdtype or dtype) if affine else None for t in (w, b))
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)

    def place(t):
        t = t.to(DEV)
        return t.movedim(1, -1).contiguous().movedim(-1, 1) if last else t

    xd, dd = place(x), place(d)
    if n is not None:  # what lies behind the tokens is not read
        for i, k in enumerate(lengths):
            xd[i, :, max(k, 0):] = float("nan")
            dd[i, :, max(k, 0):] = float("nan")
    out, grads = run(xd, groups, None if w is None else w.to(DEV), None if b is None else b.to(DEV), silu,
                     None if n is None else n.to(DEV), eps, dd)
    assert out.stride() == xd.stride() and grads[0].stride() == xd.stride()
    v, m = ref.norm(x, groups, w, b, eps, silu, lengths, d)
    close(out, v["out"], m["out"], "out")
    for got, k in zip(grads, ("dx", "dw", "db")):
        close(got, v[k], m[k], k)
    if n is not None:
        for i, k in enumerate(lengths):
            assert not out[i, :, max(k, 0):].any() and not grads[0][i, :, max(k, 0):].any()


@pytest.mark.parametrize("last", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape,groups", [
    ((1, 1, 1), 1), ((2, 6, 1), 3), ((3, 8, 5), 2), ((2, 32, 64), 32), ((2, 33, 77), 11), ((1, 40, 9), 4),
    ((5, 320, 17, 31), 32), ((2, 64, 32, 32), 8), ((3, 12, 7, 5), 1), ((1, 96, 4, 6, 8), 6), ((4, 10, 300), 5),
    ((2, 16, 4096), 2), ((1, 512, 40), 16), ((2, 1000, 6), 1)])
def test_shapes(shape, groups, dtype, last):
    check(shape, groups, dtype, last, silu=(shape[1] + groups) % 2 == 0, seed=shape[1])


@pytest.mark.parametrize("last", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lengths", [[40, 0, 1, 39, 17], [0, 0, 0, 0, 0], [-3, 100, 40, 2, 7]])
def test_lengths(lengths, dtype, last):
    check((5, 24, 40), 3, dtype, last, lengths=lengths, seed=2)


@pytest.mark.parametrize("last", [False, True])
def test_long_ragged_rows(last):
    check((3, 16, 5003), 4, BF16, last, lengths=[5003, 4100, 3], seed=3)


@pytest.mark.parametrize("last", [False, True])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_one_group_of_many_blocks(dtype, last):
    """One slab for the whole GPU: the sums go through device memory."""
    check((1, 64, 128, 130), 1, dtype, last, seed=4)


@pytest.mark.parametrize("last", [False, True])
@pytest.mark.parametrize("shape,groups", [((2, 8192, 3), 1), ((1, 8190, 5), 2), ((1, 2049 * 8, 2), 8), ((2, 257 * 4, 9), 4)])
def test_wide_groups(shape, groups, last):
    check(shape, groups, BF16, last, seed=5)


@pytest.mark.parametrize("last", [False, True])
def test_many_rows(last):
    check((3000, 8, 12), 4, F32, last, seed=6)


@pytest.mark.parametrize("last", [False, True])
def test_weights_of_32_bits_and_none(last):
    check((2, 48, 50), 6, BF16, last, wdtype=F32, seed=7)
    check((2, 48, 50), 6, F16, last, affine=False, silu=False, seed=8)


@pytest.mark.parametrize("last", [False, True])
def test_large_means_and_outliers(last):
    """A mean of 1000 deviations, and one value of 10^4 of them."""
    check((2, 32, 900), 4, F32, last, offset=1000.0, silu=False, seed=9)
    g = gen(10)
    x = torch.randn(2, 8, 1111, generator=g)
    x[:, 0, 0] = 1e4
    v, m = ref.norm(x, 2)
    xd = x.to(DEV)
    if last:
        xd = xd.transpose(1, 2).contiguous().transpose(1, 2)
    close(pc.group_norm(xd, 2), v["out"], m["out"], "out")


@pytest.mark.parametrize("last", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape,lengths", [((5, 32, 1), None), ((3, 6, 1), None), ((2, 7, 9), [1, 0]), ((2, 8, 8), [1, 1])])
def test_groups_of_one_value_have_no_gradient(shape, lengths, dtype, last):
    """Their result is the bias whatever they hold."""
    g = gen(20)
    x, w, b, d = (torch.randn(s, generator=g).to(dtype).to(DEV) for s in (shape, shape[1], shape[1], shape))
    if last:
        x, d = (t.movedim(1, -1).contiguous().movedim(-1, 1) for t in (x, d))
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    out, grads = run(x, shape[1], w, b, True, lengths=n, grad=d)
    assert not grads[0].any() and not grads[1].any()


def test_constant_input():
    x = torch.full((2, 8, 30), 7.25, device=DEV)
    b = torch.arange(8, device=DEV, dtype=F32)
    assert torch.equal(pc.group_norm(x, 4, None, b), b[:, None].expand_as(x))


def test_values_that_are_not_finite_stay_in_their_group():
    x = torch.randn(2, 8, 30, device=DEV)
    clean = pc.group_norm(x, 4)
    x[0, 3, 7] = float("inf")
    out = pc.group_norm(x, 4)
    assert out[0, 2:4].isnan().any()
    out[0, 2:4] = clean[0, 2:4]
    assert torch.equal(out, clean)


def test_orders_of_dimensions():
    x = torch.randn(3, 16, 6, 5, device=DEV)
    want = pc.group_norm(x, 4)
    for y in (x.to(memory_format=torch.channels_last), x.transpose(2, 3).contiguous().transpose(2, 3),
              torch.stack([x, x], -1)[..., 0]):
        got = pc.group_norm(y, 4)
        assert (got - want).abs().max() <= 4e-6 * want.abs().max()
    # a view off a vector's boundary
    base = torch.zeros(x.numel() + 1, device=DEV)
    base[1:] = x.flatten()
    assert (pc.group_norm(base[1:].view(x.shape), 4) - want).abs().max() <= 4e-6 * want.abs().max()


def test_gradient_against_differences():
    g = gen(11)
    x = torch.randn(2, 6, 9, generator=g).to(DEV)
    w, b, d = torch.randn(6, generator=g).to(DEV), torch.randn(6, generator=g).to(DEV), torch.randn(2, 6, 9, generator=g).to(DEV)
    out, grads = run(x, 2, w, b, True, grad=d)
    for t, gr in zip((x, w, b), grads):
        way = torch.randn(t.shape, generator=g).to(DEV)
        h = 2.0 ** -7
        ends = []
        for s in (1, -1):
            args = [u.detach() + s * h * way if u is t else u.detach() for u in (x, w, b)]
            ends.append((pc.group_norm(args[0], 2, args[1], args[2], activation="silu") * d).double().sum())
        slope = float(ends[0] - ends[1]) / (2 * h)
        # third derivatives are of the order of one: h^2, beside the outputs' roundings over h
        assert abs(slope - float((gr * way).double().sum())) <= (h * h + 2.0 ** -20 / h) * float((gr * way).abs().sum() + 10)


def test_empty_and_refused():
    assert pc.group_norm(torch.zeros(0, 4, 5, device=DEV), 2).shape == (0, 4, 5)
    x = torch.zeros(2, 4, 0, device=DEV, requires_grad=True)
    w = torch.ones(4, device=DEV, requires_grad=True)
    pc.group_norm(x, 2, w).sum().backward()
    assert w.grad.tolist() == [0.0] * 4
    x = torch.zeros(2, 4, 5, device=DEV)
    for bad in (dict(groups=3), dict(groups=0), dict(weight=torch.ones(3, device=DEV)), dict(weight=torch.ones(4)),
                dict(weight=torch.ones(4, device=DEV, dtype=F16)), dict(eps=-1.0), dict(activation="relu"),
                dict(weight=torch.ones(4, device=DEV), bias=torch.ones(4, device=DEV, dtype=F16)),
                dict(lengths=torch.zeros(2, device=DEV)), dict(lengths=torch.zeros(3, device=DEV, dtype=torch.int32))):
        with pytest.raises((RuntimeError, ValueError, NotImplementedError)):
            pc.group_norm(x, **{"groups": 2, **bad})
    with pytest.raises(RuntimeError):
        pc.group_norm(x[..., None], 2, lengths=torch.zeros(2, device=DEV, dtype=torch.int32))
    with pytest.raises(NotImplementedError):
        pc.group_norm(x.double(), 2)
    with pytest.raises(RuntimeError):
        pc.group_norm(torch.zeros(1, 8193, 1, device=DEV), 1)
    y = torch.randn(2, 4, 5, device=DEV, requires_grad=True)
    (dx,) = torch.autograd.grad(pc.group_norm(y, 2).square().sum(), y, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        dx.sum().backward()


@pytest.mark.parametrize("shape,groups", [((4, 32, 16, 16), 8), ((1, 64, 128, 128), 1)])
def test_captured_on_another_stream(shape, groups):
    """Two graphs of forward and backward passes, replayed on new inputs, equal eager calls."""
    norm = pc.GroupNorm(groups, shape[1], activation="silu").to(DEV)
    stream = torch.cuda.Stream()
    graphs = []
    for seed in range(2):
        x, d = torch.randn(shape, device=DEV), torch.randn(shape, device=DEV)
        with torch.cuda.stream(stream):
            stream.wait_stream(torch.cuda.current_stream())
            leaf = x.clone().requires_grad_(True)
            torch.autograd.grad(norm(leaf), [leaf, norm.weight, norm.bias], d)
            del leaf
        torch.cuda.current_stream().wait_stream(stream)
        x.requires_grad_(True)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = norm(x)
            grads = torch.autograd.grad(out, [x, norm.weight, norm.bias], d)
        graphs.append((graph, x, d, out, grads))
    for graph, x, d, out, grads in graphs:
        with torch.no_grad():
            x.copy_(torch.randn(shape, device=DEV))
        graph.replay()
    for graph, x, d, out, grads in graphs:
        y = x.detach().clone().requires_grad_(True)
        want = norm(y)
        assert torch.equal(out, want)
        for a, b in zip(grads, torch.autograd.grad(want, [y, norm.weight, norm.bias], d)):
            assert torch.equal(a, b)
