"""Logits of more columns than a block's bitmap has, and histories longer than its list: slices of the columns, the last one short."""
import pytest
import torch

from test_gpu_logits import TYPES, agree, case

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def used_memory():
    """what is allocated next has been written before, so that an entry that a kernel leaves out shows"""
    if torch.cuda.is_available():
        kept = [torch.full((n // 4,), float("nan"), device="cuda") for n in [1 << 28] + [1 << 19] * 64]
        del kept


def check(a):
    from wf_bitnet import ops
    out = ops.process_logits(**a)
    assert agree(out, a)
    end = int(a["offsets"][-1]) if "offsets" in a else out.shape[0]
    assert torch.equal(out[end:], a["logits"][end:])
    mine = a["logits"].clone()
    ops.process_logits(**{**a, "logits": mine}, out=mine)
    assert torch.equal(mine, out)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [131071, 131072, 131073, 131072 + 511, 151936, 262144, 262145, 300007])
def test_vocabularies(V, dtype):
    check(case([1] * 3, V, dtype, L=300, bias=9, seed=V, hot=V))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [131073, 151936, 262145])
@pytest.mark.parametrize("rows", [[60] * 2, [3, 0, 40]])
def test_trees(rows, V, dtype):
    check(case(rows, V, dtype, L=100, bias=9, seed=V, nodes=True, tail=2, hot=V))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [8191, 8192, 8193, 8704, 20001, 32000, 140001])
@pytest.mark.parametrize("L", [8190, 8192, 8193, 30000])
def test_histories(L, V, dtype):
    """every token of some slices is in the history"""
    a = case([1] * 2, V, dtype, L=L, bias=3, seed=L + V, hot=V)
    a["history_lens"][0] = L
    check(a)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [8192, 20001, 140001])
def test_histories_of_trees(V, dtype):
    a = case([50, 0, 3], V, dtype, L=9000, bias=1, seed=V, nodes=True, tail=1, hot=V)
    a["history_lens"][0] = 9000
    check(a)


def test_many_biases():
    check(case([1, 1], 40000, torch.float32, L=10, bias=20000, hot=40000))


@pytest.mark.parametrize("lead", [1, 3])
def test_rows_off_alignment(lead):
    from wf_bitnet import ops
    for dtype in TYPES:
        a = case([2, 2], 151936, dtype, L=50, nodes=True, hot=151936)
        want = ops.process_logits(**a)
        wide = torch.randn(4, 151936 + 20, device="cuda").to(dtype)
        wide[:, lead:lead + 151936] = a["logits"]
        assert torch.equal(ops.process_logits(**{**a, "logits": wide[:, lead:lead + 151936]}), want)
