"""Log probabilities of tokens that a mask has set to their type's lowest value: large negative numbers, not -inf, where a float holds them."""
import pytest
import torch

from test_gpu_logprobs import TYPES, check, reference, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("temperature", [1.0, 1.7, 1000.0])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [50, 4099, 40003])
def test_tokens_of_the_lowest_value(dtype, v, temperature):
    low = torch.finfo(dtype).min
    x, tok = rows(4, v, dtype, v)
    x[0, 7:] = low                                       # seven tokens allowed
    x[1, :-1] = low                                      # the last one
    x[2, ::2] = low
    tok[0], tok[1], tok[2] = 11, 0, 4
    want = reference(x, tok, 20, temperature)
    assert bool((want[0][:3] < -30).all()) and bool((want[2].abs() <= torch.finfo(torch.float32).max).all())
    check(x, tok, 20, temperature)                       # rows 0 and 1 have masked tokens among their alternatives


def test_beyond_float_is_minus_infinity():
    """below a temperature of 1 the lowest float is beyond what a float holds"""
    from wf_bitnet import ops
    x, tok = rows(2, 1000, torch.float32, 1)
    x[:, 5] = torch.finfo(torch.float32).min
    tok[:] = 5
    assert bool((ops.token_logprobs(x, tok, 0, 0.5)[0] == -float("inf")).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [0.3, 1.0, 7.0])
def test_an_alternatives_number_is_that_of_the_token(dtype, temperature):
    from wf_bitnet import ops
    x, _ = rows(40, 32003, dtype, 5)
    ids = x.to(torch.float64).sort(dim=-1, descending=True, stable=True).indices[:, :8].to(torch.int32)
    tlp = ops.token_logprobs(x, ids[:, 0].contiguous(), 8, temperature)[2]
    for j in range(8):
        assert torch.equal(ops.token_logprobs(x, ids[:, j].contiguous(), 0, temperature)[0], tlp[:, j])
