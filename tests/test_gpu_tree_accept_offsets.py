"""Acceptance with offsets that do not rise: sequences that share rows of the path.  The result means nothing, but every sequence's keys and values are still its own."""
import numpy as np
import pytest
import torch

from test_gpu_tree_plan import i32

pytestmark = pytest.mark.gpu
PAGE, BLOCKS = 16, 14


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("offsets, lens", [([0, 200, 10, 60], [3, 5, 150]), ([0, 200, 10, 60, 50, 200], [0, 1, 170, 2, 70]), ([150, 200, 0, 200, 190, 199], [100, 7, 20, 9, 214])])
def test_no_place_outside_the_sequence_is_read(offsets, lens, int8):
    """each page holds its sequence's number, one more table row than there are sequences stands behind them, and drafts are kept whole, or with jumps"""
    from wf_bitnet import ops
    B, T = len(lens), 200
    for seed in range(20):
        rng = np.random.default_rng(seed)
        pages = rng.permutation((B + 1) * BLOCKS + 2)[:(B + 1) * BLOCKS].reshape(B + 1, BLOCKS)
        kv = ops.PagedKV((B + 1) * BLOCKS + 2, 2, 2, PAGE, 128, dtype=torch.int8 if int8 else torch.bfloat16)
        kv.pool.fill_(100)
        whole = i32(pages)
        for b in range(B):
            kv.pool[whole[b].long()] = b + 1
            if int8:
                kv.scales[whole[b].long()] = b + 1.0
        before = kv.pool.clone(), kv.scales.clone() if int8 else None
        step = 1 + seed % 3
        parents = np.maximum(np.arange(T) - step, 0)
        tokens = rng.integers(0, 2, T)
        free = torch.full((2000,), -1, dtype=torch.int32, device="cuda")
        a = ops.tree_accept(i32(parents), i32(tokens), i32(rng.integers(0, 2, T) if seed % 2 else tokens), i32(offsets), i32(lens), kv, whole[:B], free, i32([0]))
        assert int(a.status) == 0
        torch.cuda.synchronize()
        assert torch.equal(kv.pool, before[0]) and (not int8 or torch.equal(kv.scales, before[1]))
        given = free[:int(a.free_count)].tolist()
        assert set(given) <= set(pages[:B].ravel().tolist()) and bool((free[int(a.free_count):] == -1).all())
