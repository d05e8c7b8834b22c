"""Group norm, linear attention and the AdamW step at the sizes and lengths where
they can go wrong, with comparisons that nothing but finite values pass."""
import pytest
import torch

import test_adamw_gpu as adamw
import test_attention_gpu as attention
import test_norm_gpu as norm
from strict import strictly

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def strict(monkeypatch):
    for module in (adamw, attention, norm):
        monkeypatch.setattr(module, "close", strictly(module.close))


@pytest.mark.parametrize("last", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape,groups", [((1, 1, 1), 1), ((2, 33, 77), 11), ((5, 320, 17, 31), 32), ((4, 10, 300), 5),
                                          ((2, 16, 4096), 2), ((1, 512, 40), 16), ((1, 64, 128, 130), 1), ((1, 8190, 5), 2)])
def test_norm(shape, groups, dtype, last):
    norm.check(shape, groups, dtype, last, seed=40)


@pytest.mark.parametrize("last", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape,groups,lengths", [((5, 24, 40), 3, [40, 0, 1, 39, 17]), ((5, 24, 40), 3, [-3, 100, 40, 2, 7]),
                                                  ((3, 16, 5003), 4, [5003, 4100, 3]), ((2, 6, 9), 6, [0, 9])])
def test_norm_of_ragged_rows(shape, groups, lengths, dtype, last):
    norm.check(shape, groups, dtype, last, lengths=lengths, seed=41)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dims", [(1, 1, 1, 1, 1, 1), (2, 2, 1, 8, 24, 65), (1, 2, 1, 128, 128, 96), (2, 4, 2, 33, 65, 40),
                                  (1, 2, 2, 100, 17, 200), (3, 2, 1, 48, 80, 77), (1, 2, 1, 32, 48, 1111)])
def test_attention(dims, dtype):
    attention.check(*dims, dtype, tokens=sum(dims) % 2 == 0, init=True, seed=42)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("lengths", [[70, 0, 1, 64, 65], [-3, 1000, 70, 33, 2]])
def test_attention_of_ragged_rows(lengths, dtype):
    attention.check(5, 2, 1, 24, 40, 70, dtype, init=True, lengths=lengths, seed=43)
    attention.check(5, 1, 1, 16, 16, 1030, dtype, init=True, lengths=[1030, 0, 513, 1, 1029], seed=44, low=1e-4, high=1e-1)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("train", [False, True])
def test_attention_forgets(train, dtype):
    """Strong decays, whose products leave 32 bits' range within a chunk."""
    attention.check(1, 2, 2, 32, 32, 150, dtype, seed=45, low=2.0, high=200.0, train=train)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("ptype,gtype,masters", [(F32, F32, False), (BF16, BF16, False), (BF16, F32, True), (F16, F32, False)])
def test_adamw(bits, ptype, gtype, masters):
    c = adamw.case(adamw.SIZES, ptype, gtype, bits, masters, seed=46)
    got, want = adamw.step_both(c, 6, 99, grad_scale=0.7)
    adamw.check(got, want, c)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("name", ["q", "k", "v", "g"])
def test_attention_beside_infinities(name, value, dtype):
    attention.test_values_that_are_not_finite_reach_no_earlier_token(name, value, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_gradients_beside_infinities(dtype):
    attention.test_gradients_that_are_not_finite_reach_no_later_token(dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_attention_states(dtype):
    attention.test_large_states(dtype)
    attention.test_step((3, 2, 1, 33, 65), dtype)
    if dtype != F16:
        attention.test_steps_go_on_from_a_prompt(dtype)


def test_attention_forgets_all():
    attention.test_forgetting()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_beside_infinities(bits):
    adamw.test_values_that_are_not_finite(bits)


@pytest.mark.parametrize("last", [False, True])
def test_norm_of_large_means_and_outliers(last):
    norm.test_large_means_and_outliers(last)
