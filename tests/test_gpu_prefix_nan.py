"""Decode attention behind a shared prefix: what is not a number, in a query or under a key, stays through the joining of groups, splits and own chunks, and nothing else changes."""
import math

import pytest
import torch

from test_gpu_prefix_attn import case

pytestmark = pytest.mark.gpu
PREFIXES = [64, 100, 1000, 5000, 33000]


def attn(a):
    from wf_bitnet import ops
    return ops.paged_prefix_attn(*a, None, torch.float32)


def same(x, y):
    return torch.equal(x.contiguous().view(torch.int32), y.contiguous().view(torch.int32))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("B", [3, 40])                   # rows of one group, and of two
@pytest.mark.parametrize("own", [0, 300])
@pytest.mark.parametrize("prefix", PREFIXES)
def test_a_query_that_is_not_a_number(prefix, own, B, int8):
    a = case(B, 8, 2, prefix, [own] * B, 16, int8, 1)
    clean = attn(a)
    a[0][1, 3, 50] = math.nan
    out = attn(a)
    rest = torch.ones(out.shape[:2], dtype=torch.bool, device="cuda")
    rest[1, 3] = False
    assert bool(clean.isfinite().all()) and bool(out[1, 3].isnan().all()) and same(out[rest], clean[rest])


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("B", [3, 40])
@pytest.mark.parametrize("own", [0, 300])
@pytest.mark.parametrize("where", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("prefix", PREFIXES)
def test_a_key_that_is_not_a_number(prefix, where, own, B, int8):
    a = case(B, 8, 2, prefix, [own] * B, 16, int8, 2)
    kv, layer, table = a[1], a[2], a[3]
    clean = attn(a)
    at = int(where * (prefix - 1))
    if int8:
        kv.scales[table[at // 16].long(), layer, 0, 1, at % 16] = math.nan
    else:
        kv.pool[table[at // 16].long(), layer, 0, 1, at % 16, 5] = math.nan
    out = attn(a)
    assert bool(out[:, 4:].isnan().all()) and same(out[:, :4], clean[:, :4])
