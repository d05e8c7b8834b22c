"""A training step of a small network as it would be used: a ParaConv2d layer,
group norm with SiLU, linear attention over the map, and AdamW honouring the
layer's tags; eagerly, and captured into a CUDA graph."""
import pytest
import torch
import torch.nn as nn

import paraconv2d_b200 as pc

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Net(nn.Module):
    def __init__(self, heads=2, keys=8, values=8):
        super().__init__()
        self.conv = pc.ParaConv2d(3, 16, 3, padding=1, h_lr_factor=0.5, p_lr_factor=2.0, wd_factor=0.0)
        self.norm = pc.GroupNorm(4, 16, activation="silu")
        self.project = nn.Conv1d(16, heads * (2 * keys + values), 1)
        self.mix = pc.LinearAttention(heads, keys, values)
        self.out = nn.Linear(heads * values, 4)
        self.split = (heads, keys, values)

    def tail(self, x, mix):
        """Behind the normalisation: [batch, 16, length] to logits."""
        heads, keys, values = self.split
        b, _, n = x.shape
        q, k, v = self.project(x).split([heads * keys, heads * keys, heads * values], 1)
        y = mix(q.reshape(b, heads, keys, n), k.reshape(b, heads, keys, n), v.reshape(b, heads, values, n))
        return self.out(y.flatten(1, 2).mean(-1))

    def forward(self, images):
        return self.tail(self.norm(self.conv(images).flatten(2)), self.mix)


def recurrence(q, k, v, log_decay):
    state, outs = 0.0, []
    for t in range(q.shape[-1]):
        state = torch.exp(log_decay)[:, None, None] * state + k[..., t, None] * v[:, :, None, :, t]
        outs.append((q[..., t, None] * state).sum(2) * q.shape[2] ** -0.5)
    return torch.stack(outs, -1)


def build(seed=0):
    torch.manual_seed(seed)
    net = Net().to(DEV)
    return net, torch.randn(5, 3, 7, 9, device=DEV), torch.randn(5, 4, device=DEV)


def test_step_against_64_bits(monkeypatch):
    monkeypatch.setattr(torch.backends.cudnn, "allow_tf32", False)  # the projection is torch's own
    net, images, target = build()
    maps = net.conv(images).flatten(2)
    maps.retain_grad()
    loss = (net.tail(net.norm(maps), net.mix) - target).square().sum()
    loss.backward()
    # the same from the maps on, by torch's own operations in 64 bits
    ref = Net().double()
    ref.load_state_dict({k: v.double().cpu() for k, v in net.state_dict().items()})
    x = maps.detach().double().cpu().requires_grad_(True)
    y = nn.functional.silu(nn.functional.group_norm(x, 4, ref.norm.weight, ref.norm.bias, 1e-5))
    mix = lambda q, k, v: recurrence(q, k, v, -torch.exp(ref.mix.rate))  # noqa: E731
    want = (ref.tail(y, mix) - target.double().cpu()).square().sum()
    want.backward()
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * float(want.detach())
    pairs = [(maps.grad, x.grad)] + [(a.grad, dict(ref.named_parameters())[n].grad)
                                     for n, a in net.named_parameters() if not n.startswith("conv")]
    for got, exact in pairs:
        # chains of 32-bit operations with a dozen roundings each, sums of some hundred terms in between
        assert (got.cpu().double() - exact).norm() <= 2e-5 * exact.norm() + 1e-9
    assert net.conv.pars.grad.isfinite().all()


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_training_equals_eager(bits):
    steps = 4
    data = [build(10 + i)[1:] for i in range(steps)]

    def setup():
        net, _, _ = build(1)
        return net, pc.ParaboloidAdamW(net.parameters(), lr=1e-2, weight_decay=0.1, state_bits=bits, seed=3)

    def step(net, opt, images, target):
        for p in net.parameters():
            p.grad = None
        loss = (net(images) - target).square().mean()
        loss.backward()
        opt.step()
        return loss.detach()

    net, opt = setup()
    eager = [step(net, opt, *d).item() for d in data]
    assert eager[0] != eager[1]

    other, opt2 = setup()
    images, target = (t.clone() for t in data[0])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        first = step(other, opt2, images, target)
    torch.cuda.current_stream().wait_stream(stream)
    assert first.item() == eager[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        loss = step(other, opt2, images, target)
    for i in range(1, steps):
        images.copy_(data[i][0])
        target.copy_(data[i][1])
        graph.replay()
        assert loss.item() == eager[i]
    for a, b in zip(net.parameters(), other.parameters()):
        assert torch.equal(a, b)


def test_autocast_projections_and_16_bit_maps():
    """bfloat16 maps through the layers: types go through, gradients come back in them."""
    net, images, _ = build(2)
    x = net.conv(images).flatten(2).detach().bfloat16().requires_grad_(True)
    y = net.norm(x)  # weights in float32
    assert y.dtype == torch.bfloat16
    q = y.reshape(5, 2, 8, 63)
    out = net.mix(q, q, q)
    assert out.dtype == torch.bfloat16
    out.float().square().sum().backward()
    assert x.grad.dtype == torch.bfloat16 and net.norm.weight.grad.dtype == torch.float32
    assert net.mix.rate.grad.isfinite().all() and x.grad.isfinite().all()
