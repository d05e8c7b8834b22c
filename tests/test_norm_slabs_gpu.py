"""Group norm, channels last, of few rows, where a slab's sums go through device
memory and the last slab has fewer groups than the others."""
import pytest
import torch

import test_norm_gpu as norm
import train_ref as ref
import paraconv2d_b200 as pc
from strict import strictly
from test_norm_gpu import BF16, DEV, F16, F32, gen, run

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def strict(monkeypatch):
    monkeypatch.setattr(norm, "close", strictly(norm.close))


# Channels of a token and of a group: slabs of 64 bytes or more of whole groups leave 16 of 80 bfloat16 channels in
# groups of 8, 16 of 48 in groups of 8 or 16, 8 of 24 float32 ones.
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("shape,groups,dtype", [
    ((1, 80, 64, 64), 10, BF16), ((1, 48, 64, 64), 6, F16), ((1, 48, 64, 64), 3, BF16), ((1, 24, 64, 64), 3, F32),
    ((1, 24, 128, 128), 3, F32), ((2, 80, 128, 128), 5, BF16), ((3, 72, 61, 67), 6, F16), ((1, 80, 64, 64), 20, BF16)])
def test_a_smaller_last_slab(shape, groups, dtype, silu):
    norm.check(shape, groups, dtype, True, silu=silu, seed=30)


@pytest.mark.parametrize("channels,groups,dtype", [(80, 10, BF16), (48, 6, F16), (24, 3, F32)])
@pytest.mark.parametrize("lengths", [[4096, 3001], [0, 4096], [1, 4095], [2048, 17]])
def test_a_smaller_last_slab_of_ragged_rows(channels, groups, dtype, lengths):
    norm.check((2, channels, 4096), groups, dtype, True, lengths=lengths, seed=31)


@pytest.mark.parametrize("shape,groups,dtype", [((1, 24, 64, 64), 6, F32), ((1, 48, 64, 64), 6, BF16)])
def test_a_smaller_last_slab_off_a_boundary(shape, groups, dtype):
    """Views that start off a vector's boundary, whose slabs are cut by single elements."""
    g = gen(32)
    C = shape[1]
    x, d = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    w, b = torch.randn(C, generator=g).to(dtype), torch.randn(C, generator=g).to(dtype)

    def place(t):
        base = torch.zeros(t.numel() + 1, dtype=dtype, device=DEV)
        view = base[1:].view(shape[0], *shape[2:], C).movedim(-1, 1)
        view.copy_(t)
        return view

    out, grads = run(place(x), groups, w.to(DEV), b.to(DEV), True, grad=place(d))
    v, m = ref.norm(x, groups, w, b, silu=True, grad=d)
    norm.close(out, v["out"], m["out"], "out")
    for got, k in zip(grads, ("dx", "dw", "db")):
        norm.close(got, v[k], m[k], k)


def test_slabs_repeat_themselves():
    """The same call gives the same bits: no two blocks write the same numbers."""
    x = torch.randn(1, 80, 64, 64, device=DEV, dtype=BF16).to(memory_format=torch.channels_last).requires_grad_(True)
    d = torch.randn_like(x)
    first = None
    for _ in range(8):
        out = pc.group_norm(x, 10, activation="silu")
        both = [out.detach(), *torch.autograd.grad(out, x, d)]
        first = first or both
        assert all(torch.equal(a, b) for a, b in zip(first, both))
