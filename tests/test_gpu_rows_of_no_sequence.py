"""Offsets that begin behind row 0: the rows in front of the first sequence are of no sequence, as those behind the last one are."""
import numpy as np
import pytest
import torch

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
