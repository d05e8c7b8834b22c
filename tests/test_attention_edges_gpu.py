"""Linear attention on the GPU: what its gradients, its outputs and its states
promise beside their values."""
import pytest
import torch

import paraconv2d_b200 as pc
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
