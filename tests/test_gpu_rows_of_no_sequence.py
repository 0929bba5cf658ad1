"""Offsets that begin behind row 0: the rows in front of the first sequence are of no sequence, as those behind the last one are."""
import math

import numpy as np
import pytest
import torch

from test_gpu_logits import case as logits_case
from test_gpu_tree_plan import forest, i32

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def used_memory():
    """what is allocated next has been written before, so that an entry that a kernel leaves out shows"""
    if torch.cuda.is_available():
        kept = [torch.full((n // 4,), float("nan"), device="cuda") for n in [1 << 28] + [1 << 19] * 64]
        del kept


@pytest.mark.parametrize("max_nodes", [40, 200])
@pytest.mark.parametrize("lead", [1, 5, 3000])
def test_masks_and_positions(lead, max_nodes):
    from wf_bitnet import ops
    nodes = [40, 0, 7]
    parents = forest(np.random.default_rng(lead), nodes)
    offsets = np.concatenate([[0], np.cumsum(nodes)])
    lens = i32([100, 3, 9])
    want = ops.tree_plan(i32(parents), i32(offsets), lens, max_nodes)
    pad = np.full(lead, 2, np.int32)
    p = ops.tree_plan(i32(np.concatenate([pad, parents, pad])), i32(offsets + lead), lens, max_nodes)
    T = len(parents)
    assert torch.equal(p.mask[lead:lead + T], want.mask) and torch.equal(p.positions[lead:lead + T], want.positions)
    for rows in (slice(0, lead), slice(lead + T, None)):
        assert not p.mask[rows].any() and not p.positions[rows].any()
    p = ops.tree_plan(i32(pad), i32([lead + 9] * 4), lens, max_nodes)           # (beyond the rows: all of them)
    assert not p.mask.any() and not p.positions.any()


@pytest.mark.parametrize("lead", [1, 5, 3000])
def test_acceptance(lead):
    from wf_bitnet import ops
    B, n = 9, 6
    rng = np.random.default_rng(lead)
    parents = forest(rng, [n] * B, 2)
    tokens, targets = rng.integers(0, 3, B * n), rng.integers(0, 3, B * n)
    offsets = np.arange(B + 1) * n
    table = i32(np.arange(B * 2).reshape(B, 2))
    lens = i32(rng.integers(0, 20, B))

    def accept(pad):
        kv = ops.PagedKV(B * 2 + 1, 1, 1, 16, 128)
        kv.pool.copy_(torch.randn(kv.pool.shape, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda"))
        free = torch.full((B * 2 + 1,), -1, dtype=torch.int32, device="cuda")
        row = lambda x: i32(np.concatenate([np.zeros(pad, np.int32), x, np.zeros(pad, np.int32)]))  # noqa: E731
        return kv, free, ops.tree_accept(row(parents), row(tokens), row(targets), i32(offsets + pad), lens, kv, table, free, i32([0]))
    kv0, free0, want = accept(0)
    kv, free, a = accept(lead)
    assert torch.equal(a.path[lead:lead + B * n], want.path) and bool((a.path[:lead] == -1).all()) and bool((a.path[lead + B * n:] == -1).all())
    for x, y in zip((a.accepted, a.next_tokens, a.lens, a.free_count, a.status), (want.accepted, want.next_tokens, want.lens, want.free_count, want.status)):
        assert torch.equal(x, y)
    assert torch.equal(kv.pool, kv0.pool) and torch.equal(free, free0) and int(a.status) == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [1, 100, 1003, 32003, 140000])
@pytest.mark.parametrize("rows", [[3], [2, 0, 5], [60, 1, 9]])
@pytest.mark.parametrize("lead", [1, 7, 70])
def test_logits(lead, rows, V, dtype):
    """copied, whatever their masks say; in place left as they are"""
    from wf_bitnet import ops
    a = logits_case(rows, V, dtype, L=40, nodes=True, tail=2, seed=lead)
    want = ops.process_logits(**a)
    g = torch.Generator(device="cuda").manual_seed(lead)
    more = dict(a)
    more["logits"] = torch.cat([torch.randn(lead, V, generator=g, device="cuda").to(dtype), a["logits"]])
    more["allowed"] = torch.cat([torch.zeros(lead, a["allowed"].shape[1], dtype=torch.int32, device="cuda"), a["allowed"]])
    more["node_mask"] = torch.cat([torch.full((lead, a["node_mask"].shape[1]), -1, device="cuda"), a["node_mask"]])
    more["node_tokens"] = torch.cat([torch.zeros(lead, dtype=torch.int32, device="cuda"), a["node_tokens"]])
    more["offsets"] = a["offsets"] + lead
    out = ops.process_logits(**more)
    assert torch.equal(out[:lead], more["logits"][:lead]) and torch.equal(out[lead:], want)
    out = ops.process_logits(**more, out=torch.full_like(out, math.nan))
    assert torch.equal(out[:lead], more["logits"][:lead]) and torch.equal(out[lead:], want)
    mine = more["logits"].clone()
    ops.process_logits(**{**more, "logits": mine}, out=mine)
    assert torch.equal(mine, out)


def test_logits_of_no_sequence_at_all():
    from wf_bitnet import ops
    x = torch.randn(300, 999, device="cuda")
    for offsets in ([0], [300], [9], [1000, 1000]):
        assert torch.equal(ops.process_logits(x, offsets=i32(offsets), out=torch.full_like(x, math.nan)), x)


def test_attention():
    from test_gpu_tree_attn import case
    from wf_bitnet import ops
    a, _ = case([70, 3], [9, 30], 8, 2, 16, pad=0)
    want = ops.paged_tree_attn(**a)
    lead = 37
    a["q"] = torch.cat([torch.randn(lead, 8, 128, device="cuda").to(torch.bfloat16), a["q"]])
    a["mask"] = torch.cat([torch.full((lead, a["mask"].shape[1]), -1, device="cuda"), a["mask"]])
    a["offsets"] = a["offsets"] + lead
    out = ops.paged_tree_attn(**a)
    assert not out[:lead].any() and torch.equal(out[lead:], want)
