"""Linear attention on the GPU: what its gradients, its outputs and its states
promise beside their values."""
import pytest
import torch

import test_attention_gpu
import paraconv2d_b200 as pc
from strict import strictly
from test_attention_gpu import BF16, DEV, F16, F32, inputs

pytestmark = pytest.mark.gpu


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
