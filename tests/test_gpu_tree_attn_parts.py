"""Attention of drafted tokens where several blocks share a row's keys: what is not a number in one of their parts stays, and nothing else changes."""
import math

import pytest
import torch

from test_gpu_tree_attn import case

pytestmark = pytest.mark.gpu
F32 = torch.float32
# one row tile of keys for one block, for a few (each warp of the join has one part at most), and for many
CONTEXTS = [0, 100, 700, 1100, 1500, 2000, 3000, 9000, 40000]
HEADS = [(8, 2), (2, 2)]                                 # rows of two groups, and of one


def attn(a, **more):
    from wf_bitnet import ops
    return ops.paged_tree_attn(**{**a, **more}, out_dtype=F32)


def place(a, j, page=16):
    """page and slot of a sequence's token j (the first sequence's)"""
    return a["block_table"][0, j // page].long(), j % page


def same(x, y):
    return torch.equal(x.contiguous().view(torch.int32), y.contiguous().view(torch.int32))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("H, Hkv", HEADS)
@pytest.mark.parametrize("ctx", CONTEXTS)
def test_a_query_that_is_not_a_number(ctx, H, Hkv, int8):
    a, _ = case([ctx, 50], [33, 4], H, Hkv, 16, int8, 3)
    clean = attn(a)
    a["q"][11, 1, 77] = math.nan
    out = attn(a)
    assert bool(out[11, 1].isnan().all())
    rest = torch.ones(out.shape[:2], dtype=torch.bool, device="cuda")
    rest[11, 1] = False
    assert bool(clean.isfinite().all()) and same(out[rest], clean[rest])


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("H, Hkv", HEADS)
@pytest.mark.parametrize("where", ["first", "middle", "draft"])
@pytest.mark.parametrize("ctx", CONTEXTS)
def test_a_key_that_is_not_a_number(ctx, where, H, Hkv, int8):
    """a cached token's reaches all rows of its key/value head, a draft's those that see it"""
    if where != "draft" and not ctx:
        pytest.skip("no cached tokens")
    n, j = 33, 16
    a, bits = case([ctx, 50], [n, 4], H, Hkv, 16, int8, 4)
    clean = attn(a)
    at = {"first": 0, "middle": ctx // 2, "draft": ctx + j}[where]
    page, slot = place(a, at)
    if int8:
        a["kv"].scales[page, a["layer"], 0, 1, slot] = math.nan
    else:
        a["kv"].pool[page, a["layer"], 0, 1, slot, 5] = math.nan
    out = attn(a)
    hit = torch.zeros(out.shape[:2], dtype=torch.bool, device="cuda")
    hit[:n, H // Hkv:] = (bits[0][:, j] if where == "draft" else torch.ones(n, dtype=torch.bool)).cuda()[:, None]
    assert bool(hit.any()) and bool(out[hit].isnan().all()) and same(out[~hit], clean[~hit])


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("H, Hkv", HEADS)
@pytest.mark.parametrize("ctx", CONTEXTS)
def test_a_value_that_is_not_finite_reaches_the_rows_that_see_it(ctx, H, Hkv, value):
    """those rows have it in its columns (every weight here is a number above zero), all others the bits of the clean result, whose hidden value is zero"""
    n, j = 33, 16
    a, bits = case([ctx, 50], [n, 4], H, Hkv, 16, False, 5)
    page, slot = place(a, ctx + j)
    a["kv"].pool[page, a["layer"], 1, 1, slot] = 0.0
    clean = attn(a)
    a["kv"].pool[page, a["layer"], 1, 1, slot, 40:100] = value
    out = attn(a)
    hit = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    hit[:n, H // Hkv:, 40:100] = bits[0][:, j].cuda()[:, None, None]
    assert bool(hit.any()) and same(out[~hit], clean[~hit])
    assert bool((out[hit].isnan() if math.isnan(value) else out[hit] == value).all())


@pytest.mark.parametrize("H, Hkv", HEADS)
@pytest.mark.parametrize("ctx", CONTEXTS)
def test_an_infinite_score(ctx, H, Hkv):
    """+inf makes a row NaN, -inf is no weight: the bits of a row that does not see the key"""
    n, j = 33, 16
    a, bits = case([ctx, 50], [n, 4], H, Hkv, 16, False, 6)
    page, slot = place(a, ctx + j)
    less = a["mask"].clone()
    less[:n, 0] &= ~(1 << j)
    clean = attn(a)
    hidden = attn(a, mask=less)
    a["kv"].pool[page, a["layer"], 0, 1, slot, 9] = math.inf
    out = attn(a)
    q = a["q"][:n, H // Hkv:, 9].float()
    sees = bits[0][:, j].cuda()[:, None].expand_as(q)
    mine = out[:n, H // Hkv:]
    assert bool((q != 0).all()) and bool(mine[sees & (q > 0)].isnan().all())
    # a row that saw nothing else had weights of that key alone, and has zeros without it, here as there
    assert same(mine[sees & (q < 0)], hidden[:n, H // Hkv:][sees & (q < 0)])
    assert same(mine[~sees], clean[:n, H // Hkv:][~sees])
    assert same(out[:, :H // Hkv], clean[:, :H // Hkv]) and same(out[n:], clean[n:])


@pytest.mark.parametrize("n", [2, 40, 100])
@pytest.mark.parametrize("ctx", CONTEXTS[1:])
def test_a_score_that_is_not_a_number_beside_none_but_minus_infinity(ctx, n):
    """the two groups of a block have every other tile: in one of them a row has only scores of -inf, in the other only one that is not a number"""
    a, bits = case([ctx], [n], 1, 1, 16, False, 7, pad=0)
    a["q"] = a["q"].abs() + 0.1
    pool, layer = a["kv"].pool, a["layer"]
    for b in range(-(-(ctx + n) // 16)):
        pool[a["block_table"][0, b].long(), layer, 0] = -math.inf
    j = n - 1
    page, slot = place(a, ctx + j)
    pool[page, layer, 0, 0, slot] = math.nan
    bits[0][:, j] = torch.arange(n) % 3 != 0
    a["mask"][:, j // 64] &= ~(-2**63 if j % 64 == 63 else 1 << (j % 64))
    a["mask"][:, j // 64] |= torch.where(bits[0][:, j].cuda(), -2**63 if j % 64 == 63 else 1 << (j % 64), 0)
    out = attn(a)
    sees = bits[0][:, j].cuda()
    assert bool(out[sees].isnan().all()) and not out[~sees].any()
