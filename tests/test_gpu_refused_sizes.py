"""Sizes that an operator refuses are refused before any memory is asked for them: the error is the operator's own, whatever the device has room for."""
import pytest
import torch

pytestmark = pytest.mark.gpu
D = 128


@pytest.fixture(params=["native", "ctypes"])
def ops(request, monkeypatch):
    from wf_bitnet import _native, ops
    if request.param == "ctypes":
        monkeypatch.setattr(_native, "_ops", _native._Ctypes)
    elif not _native.is_native():
        pytest.skip("no libwf_torch.so")
    return ops


def refused(call, error):
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with pytest.raises(error) as e:
        call()
    assert not isinstance(e.value, torch.OutOfMemoryError)
    assert torch.cuda.max_memory_allocated() - before < 16 << 20


def i32(*s):
    return torch.zeros(*s, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("top", [1 << 24, (1 << 31) - 1])
def test_alternatives(ops, top):
    x = torch.zeros(3, 200, device="cuda")
    refused(lambda: ops.token_logprobs(x, i32(3), top), ValueError)          # more than there are columns


def test_alternatives_of_many_columns(ops):
    x = torch.zeros(1, 1 << 22, dtype=torch.bfloat16, device="cuda")
    refused(lambda: ops.token_logprobs(x, i32(1), 1 << 22), NotImplementedError)


@pytest.mark.parametrize("tokens", [(1 << 30) + 1, (1 << 31) - 1])
def test_plans(ops, tokens):
    refused(lambda: ops.paged_plan(i32(2), i32(2), i32(2, 3), i32(9), i32(1), 16, tokens), NotImplementedError)


def test_shared_prefix_attention(ops):
    kv = ops.PagedKV(4, 1, 1, 16, D)
    q = torch.zeros(65536, 8, D, dtype=torch.bfloat16, device="cuda")
    refused(lambda: ops.paged_prefix_attn(q, kv, 0, i32(1), 16, i32(65536, 40), i32(65536)), NotImplementedError)          # more sequences with keys of their own than a grid has
    long = i32((1 << 26) + 8)
    refused(lambda: ops.paged_prefix_attn(q[:2], kv, 0, long, (1 << 30) + 16, i32(2, 0), i32(2)), NotImplementedError)
    refused(lambda: ops.paged_prefix_attn(q[:2], kv, 0, long, (1 << 30) + 16, i32(2, 8), i32(2)), NotImplementedError)
