"""Linear attention on the GPU: what its gradients, its outputs and its states
promise beside their values."""
import pytest
import torch

import test_attention_gpu
import train_ref as ref
import paraconv2d_b200 as pc
from strict import strictly
from test_attention_gpu import BF16, DECAY_PARTS, DEV, F16, F32, PARTS, inputs

pytestmark = pytest.mark.gpu
close = strictly(test_attention_gpu.close)
AT = 90  # a token that is neither the first nor the last of its chunk


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dims", [(1, 2, 1, 64, 64, 2048), (1, 2, 2, 128, 128, 1500), (2, 3, 3, 32, 48, 777)])
def test_outputs_do_not_depend_on_gradients(dims, dtype):
    """A prompt has the same outputs and the same final state under no_grad as in training."""
    t, _, _ = inputs(*dims, dtype, True, 21, low=1e-4, high=1e-1, init=True)
    d = {k: x.to(DEV) for k, x in t.items()}
    call = lambda: pc.linear_attention(d["q"], d["k"], d["v"], d["g"], initial_state=d["init"],  # noqa: E731
                                       return_final_state=True)
    with torch.no_grad():
        plain = call()
    d["g"].requires_grad_(True)
    kept = call()
    assert torch.equal(plain[1], kept[1])
    assert torch.equal(plain[0], kept[0])


@pytest.mark.parametrize("dims,train", [((1, 1, 1, 16, 16, 64), True), ((2, 4, 2, 64, 64, 200), True), ((1, 2, 1, 128, 128, 333), True),
                                        ((3, 2, 1, 48, 80, 77), True), ((1, 2, 2, 128, 96, 2048), False)])
def test_bfloat16_is_rounded_once(dims, train, monkeypatch):
    """Scores and states meet the inputs as two numbers of 8 bits of mantissa, the first cut off (its rest is below 2^-7)
    and the second rounded (2^-8 of the rest): 2^-15 of the terms' sizes, beside the rounding of the outputs and of the
    gradients of q, k and v themselves."""
    monkeypatch.setitem(test_attention_gpu.PARTS, BF16, 2.0 ** -15)
    monkeypatch.setattr(test_attention_gpu, "close", strictly(test_attention_gpu.close))
    test_attention_gpu.check(*dims, BF16, init=True, seed=22, train=train)
    test_attention_gpu.check(*dims, BF16, seed=23, train=train, low=1e-4, high=1e-2)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("name", ["q", "k", "v"])
def test_infinities_reach_only_the_gradients_of_what_they_meet(name, value, dtype):
    """A query is in the gradients of keys, values and decays up to its token; a key or value in those of queries from
    its token on and of decays behind it, and in its own token's value or key."""
    t, go, _ = inputs(1, 2, 1, 32, 32, 150, dtype, True, 20)
    v, m = ref.attention(**t, grad=go, chunk=64 if dtype == BF16 else 32)
    d = {k: None if x is None else x.to(DEV) for k, x in t.items()}
    head = slice(None)
    if name == "v":
        d["v"][0, 1, 3, AT] = value
        head = 1
    else:
        d[name][0, 0, 3, AT] = value
    leaves = [d[n].requires_grad_(True) for n in ("q", "k", "v", "g")]
    grads = torch.autograd.grad(pc.linear_attention(*leaves), leaves, go.to(DEV))
    upto, before, after, token = slice(AT + 1), slice(AT), slice(AT, None), slice(AT, AT + 1)
    reached = {"q": dict(dk=(0, 0, 3, upto), dv=(0, head, slice(None), upto), dg=(0, head, upto)),
               "k": dict(dq=(0, 0, slice(None), after), dv=(0, head, slice(None), token), dg=(0, head, slice(AT + 1, None))),
               "v": dict(dq=(0, 0, slice(None), after), dk=(0, 0, slice(None), token), dg=(0, head, slice(AT + 1, None)))}[name]
    for g, key in zip(grads, ("dq", "dk", "dv", "dg")):
        fine = torch.ones(v[key].shape, dtype=torch.bool)
        if key in reached:
            fine[reached[key]] = False
        close(g.cpu()[fine], v[key][fine], m[key][fine], (DECAY_PARTS if key == "dg" else PARTS)[dtype], 4, (name, key))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_gradients_of_strong_decays(dtype):
    """A decay's gradient is as exact as its own terms, however large the pairs of tokens are that it does not divide:
    beside the states' parts, each exponent is off by two roundings of itself."""
    t, go, _ = inputs(1, 2, 2, 32, 32, 150, dtype, True, 24, low=3.0, high=30.0)
    forgets = [0, 17, 63, 64, 90, 149]
    t["g"][0, 1, forgets] = float("-inf")
    v, m = ref.attention(**t, grad=go, chunk=1)
    size = m["dg"] - (t["q"].double().abs() * m["dq"]).sum(2)  # (less the pairs that the reference allows to cancel)
    d = {k: None if x is None else x.to(DEV) for k, x in t.items()}
    g = d["g"].requires_grad_(True)
    (dg,) = torch.autograd.grad(pc.linear_attention(d["q"], d["k"], d["v"], g), g, go.to(DEV))
    close(dg, v["dg"], size.clamp(min=0) * (1 + 1e-9) + 1e-18 * m["dg"], DECAY_PARTS[dtype] + 30 * 2.0 ** -23, 4, "dg")
    assert not dg[0, 1, forgets].any()
