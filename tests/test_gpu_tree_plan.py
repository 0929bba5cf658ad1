"""Masks and positions of trees of drafts, and the acceptance of a path, against a walk on the host."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
D = 128


@pytest.fixture(autouse=True)
def used_memory():
    """what is allocated next has been written before, so that an entry that a kernel leaves out shows"""
    if torch.cuda.is_available():
        kept = [torch.full((n // 4,), float("nan"), device="cuda") for n in [1 << 28] + [1 << 19] * 64]
        del kept


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def forest(rng, nodes, reach=8):
    """parents of sequences with so many drafts each"""
    return np.concatenate([[-1 if i == 0 or rng.random() < 0.02 else int(rng.integers(max(0, i - reach), i)) for i in range(n)] for n in nodes] + [[]]).astype(np.int32)


def plan_by_hand(parents, offsets, lens, max_nodes, T):
    w = -(-max_nodes // 64)
    mask, pos = np.zeros((T, w), np.uint64), np.zeros(T, np.int32)
    for b in range(len(lens)):
        n = offsets[b + 1] - offsets[b]
        for i in range(n):
            t = offsets[b] + i
            if n > max_nodes:
                pos[t] = -1
                continue
            u = parents[t]
            if 0 <= u < i:
                mask[t], pos[t] = mask[offsets[b] + u], pos[offsets[b] + u] + 1
            else:
                pos[t] = lens[b]
            mask[t, i // 64] |= np.uint64(1 << (i % 64))
    return mask.view(np.int64), pos


@pytest.mark.parametrize("max_nodes", [1, 7, 64, 65, 128, 129, 200, 256])
@pytest.mark.parametrize("reach", [1, 3, 300])
def test_masks_and_positions(max_nodes, reach):
    """chains, bushes, trees that hang from the first draft alone; sequences without drafts; rows behind the last one"""
    from wf_bitnet import ops
    rng = np.random.default_rng(max_nodes + reach)
    nodes = [max_nodes, 1, 0, max(1, max_nodes - 1), max_nodes // 2 + 1, 0, max_nodes]
    offsets = np.concatenate([[0], np.cumsum(nodes)])
    T = int(offsets[-1]) + 5
    parents = np.concatenate([forest(rng, nodes, reach), rng.integers(-5, 5, 5).astype(np.int32)])
    lens = rng.integers(0, 5000, len(nodes)).astype(np.int32)
    p = ops.tree_plan(i32(parents), i32(offsets), i32(lens), max_nodes)
    mask, pos = plan_by_hand(parents, offsets, lens, max_nodes, T)
    np.testing.assert_array_equal(p.mask.cpu().numpy(), mask)
    np.testing.assert_array_equal(p.positions.cpu().numpy(), pos)


def test_parents_that_are_none_and_trees_that_are_too_large():
    from wf_bitnet import ops
    parents, offsets, lens = i32([5, 0, 2, -7, 1, 0, 0]), i32([0, 3, 7]), i32([10, 20])
    p = ops.tree_plan(parents, offsets, lens, 4)
    assert p.mask[:, 0].tolist() == [1, 3, 4, 1, 2, 5, 9] and p.positions.tolist() == [10, 11, 10, 20, 20, 21, 21]
    p = ops.tree_plan(parents, offsets, lens, 3)
    assert p.mask[:, 0].tolist() == [1, 3, 4, 0, 0, 0, 0] and p.positions.tolist() == [10, 11, 10, -1, -1, -1, -1]
    p = ops.tree_plan(parents, offsets, i32([-1, 2**31 - 1]), 4)
    assert not p.mask.any() and p.positions.tolist() == [-1] * 7
    for off in ([0, 9, 12], [5, 3, 1], [-4, 2, 2]):       # offsets that do not fit their rows: nothing outside them is touched
        ops.tree_plan(parents, i32(off), lens, 4)
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    p = ops.tree_plan(parents, i32([0]), e, 4)
    assert not p.mask.any() and not p.positions.any()
    assert ops.tree_plan(e, i32([0, 0]), i32([4]), 4).mask.shape == (0, 1)


def test_many_sequences():
    from wf_bitnet import ops
    rng = np.random.default_rng(0)
    nodes = rng.integers(0, 20, 3000)
    offsets = np.concatenate([[0], np.cumsum(nodes)])
    parents, lens = forest(rng, nodes), rng.integers(0, 100, 3000).astype(np.int32)
    p = ops.tree_plan(i32(parents), i32(offsets), i32(lens), 20)
    mask, pos = plan_by_hand(parents, offsets, lens, 20, len(parents))
    np.testing.assert_array_equal(p.mask.cpu().numpy(), mask)
    np.testing.assert_array_equal(p.positions.cpu().numpy(), pos)


def test_plan_refusals():
    from wf_bitnet import ops
    ok = dict(parents=i32([-1, 0]), offsets=i32([0, 2]), seq_lens=i32([3]), max_nodes=64)
    for key, bad in (("parents", i32([[0]])), ("parents", ok["parents"].long()), ("offsets", i32([0])), ("seq_lens", i32([3]).cpu()), ("max_nodes", 0), ("max_nodes", -1)):
        with pytest.raises(ValueError):
            ops.tree_plan(**{**ok, key: bad})
    with pytest.raises(NotImplementedError):
        ops.tree_plan(**{**ok, "max_nodes": 257})


# ---- acceptance
def accept_by_hand(parents, tokens, targets, offsets, lens, pool, scales, table, free, count, page):
    pool, free = pool.clone(), free.copy()
    scales = None if scales is None else scales.clone()
    path, kept, nxt, new = np.full(len(parents), -1, np.int32), [], [], []
    for b in range(len(lens)):
        a, n = offsets[b], offsets[b + 1] - offsets[b]
        if n == 0:
            kept.append(0), nxt.append(-1), new.append(lens[b])
            continue
        way = [0]
        while True:
            here = [j for j in range(way[-1] + 1, n) if parents[a + j] == way[-1] and tokens[a + j] == targets[a + way[-1]]]
            if not here:
                break
            way.append(here[0])
        path[a:a + len(way)] = way
        kept.append(len(way)), nxt.append(targets[a + way[-1]]), new.append(lens[b] + len(way))
        for k, j in enumerate(way):
            s, d = lens[b] + j, lens[b] + k
            pool[table[b, d // page], :, :, :, d % page] = pool[table[b, s // page], :, :, :, s % page]
            if scales is not None:
                scales[table[b, d // page], :, :, :, d % page] = scales[table[b, s // page], :, :, :, s % page]
        for j in range(-(-new[-1] // page), -(-(lens[b] + n) // page)):
            free[count] = table[b, j]
            count += 1
    return kept, path, nxt, new, count, pool, scales, free


def state(seed, ctx, nodes, page, layers=2, kv_heads=2, dtype=torch.bfloat16, spare=3, agree=0.8, pad=2, head_dim=D):
    from wf_bitnet import ops
    rng = np.random.default_rng(seed)
    B, T = len(ctx), sum(nodes) + pad
    blocks = max([-(-(c + n) // page) for c, n in zip(ctx, nodes)] + [1])
    order = rng.permutation(B * blocks + spare).astype(np.int32)
    table = order[spare:].reshape(B, blocks)
    kv = ops.PagedKV(len(order), layers, kv_heads, page, head_dim, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(seed)
    if dtype == torch.int8:
        kv.pool.copy_(torch.randint(0, 256, kv.pool.shape, generator=g, device="cuda", dtype=torch.uint8))
        kv.scales.copy_(torch.rand(kv.scales.shape, generator=g, device="cuda"))
    else:
        kv.pool.copy_(torch.randn(kv.pool.shape, generator=g, device="cuda"))
    offsets = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    parents = np.concatenate([forest(rng, nodes, 4), np.zeros(pad, np.int32)]).astype(np.int32)
    tokens, targets = rng.integers(0, 5, T).astype(np.int32), rng.integers(0, 5, T).astype(np.int32)
    for b in range(B):
        for j in range(1, nodes[b]):
            if parents[offsets[b] + j] >= 0 and rng.random() < agree:
                targets[offsets[b] + parents[offsets[b] + j]] = tokens[offsets[b] + j]
    free = np.full(len(order), -9, np.int32)
    free[:spare] = order[:spare]
    return kv, parents, tokens, targets, offsets, np.asarray(ctx, np.int32), table, free, spare


def run_accept(s, page):
    from wf_bitnet import ops
    kv, parents, tokens, targets, offsets, lens, table, free, count = s
    before = kv.pool.clone(), None if kv.dtype != torch.int8 else kv.scales.clone()
    fr = i32(free)
    a = ops.tree_accept(i32(parents), i32(tokens), i32(targets), i32(offsets), i32(lens), kv, i32(table), fr, i32([count]))
    return a, fr, before


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8, torch.float32])
@pytest.mark.parametrize("page", [1, 7, 16, 64])
@pytest.mark.parametrize("agree", [0.0, 0.8, 1.0])
def test_acceptance(agree, page, dtype):
    ctx, nodes = [5, 0, 33, 100, 16, 9, 64], [60, 1, 0, 256, 17, 2, 33]
    s = state(page, ctx, nodes, page, dtype=dtype, agree=agree)
    a, fr, before = run_accept(s, page)
    kept, path, nxt, new, count, pool, scales, free = accept_by_hand(*s[1:6], *before, s[6], s[7], s[8], page)
    assert a.accepted.tolist() == kept and a.next_tokens.tolist() == nxt and a.lens.tolist() == new and int(a.free_count) == count and int(a.status) == 0
    np.testing.assert_array_equal(a.path.cpu().numpy(), path)
    np.testing.assert_array_equal(fr.cpu().numpy(), free)
    assert torch.equal(s[0].pool, pool) and (scales is None or torch.equal(s[0].scales, scales))
    if agree == 1.0:
        assert max(kept) > 5


def test_a_chain_that_is_kept_whole_and_a_jump_at_its_end():
    """places that stay, and a last one that moves far"""
    n = 200
    s = state(3, [10], [n], 16, agree=0.0)
    kv, parents, tokens, targets, offsets, lens, table, free, count = s
    parents[:n] = np.arange(-1, n - 1)
    tokens[:n], targets[:n] = np.arange(n), np.arange(1, n + 1)
    a, fr, before = run_accept(s, 16)
    assert int(a.accepted) == n and int(a.next_tokens) == n and int(a.free_count) == count and torch.equal(kv.pool, before[0])
    parents[n - 1], targets[49], tokens[n - 1] = 49, 7777, 7777
    targets[n - 1] = -3
    a, fr, before = run_accept(s, 16)
    assert int(a.accepted) == 51 and a.path[:52].tolist() == [*range(50), n - 1, -1] and int(a.next_tokens) == -3
    want = accept_by_hand(*s[1:6], *before, table, free, count, 16)
    assert torch.equal(kv.pool, want[5]) and fr.tolist() == want[7].tolist() and int(a.free_count) == want[4]


def test_what_cannot_be_done_is_not_done():
    from wf_bitnet import ops
    page = 16
    s = state(1, [5, 100], [40, 40], page, spare=3)
    kv, parents, tokens, targets, offsets, lens, table, free, count = s
    want = accept_by_hand(*s[1:6], kv.pool.clone(), None, table, free, count, page)
    base = dict(parents=i32(parents), tokens=i32(tokens), targets=i32(targets), offsets=i32(offsets), seq_lens=i32(lens), kv=kv, block_table=i32(table))
    pool = kv.pool.clone()
    cases = [(dict(), i32(free[:count + 1]), count, 1), (dict(), i32(free), -1, 16), (dict(), i32(free), len(free) + 1, 16), (dict(block_table=i32(table[:, :6])), i32(free), count, 4),
             (dict(seq_lens=i32([5, -1])), i32(free), count, 8), (dict(seq_lens=i32([5, 2**31 - 5])), i32(free), count, 8)]
    for change, fr, cnt, status in cases:
        was = fr.clone()
        a = ops.tree_accept(**{**base, **change}, free_pages=fr, free_count=i32([cnt]))
        assert int(a.status) & status, (change.keys(), int(a.status))
        assert torch.equal(fr, was) and torch.equal(kv.pool, pool) and int(a.free_count) == cnt
        assert a.accepted.tolist() == want[0] and a.next_tokens.tolist() == want[2]
        if not change:
            assert a.lens.tolist() == [45, 140]
    big = state(2, [5], [257], page)
    a, fr, before = run_accept(big, page)
    assert int(a.status) == 8 and int(a.accepted) == 0 and int(a.next_tokens) == -1 and (a.path == -1).all() and torch.equal(big[0].pool, before[0])


def test_no_sequences_and_no_drafts():
    s = state(4, [5, 6], [0, 0], 16, pad=0)
    a, fr, before = run_accept(s, 16)
    assert a.accepted.tolist() == [0, 0] and a.next_tokens.tolist() == [-1, -1] and a.lens.tolist() == [5, 6] and int(a.free_count) == s[8] and int(a.status) == 0
    from wf_bitnet import ops
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    a = ops.tree_accept(e, e, e, i32([0]), e, s[0], e.view(0, 4), i32([1, 2]), i32([2]))
    assert int(a.free_count) == 2 and int(a.status) == 0 and a.accepted.numel() == 0


def test_many_sequences_hand_pages_back():
    rng = np.random.default_rng(9)
    B = 700
    s = state(5, rng.integers(0, 40, B).tolist(), rng.integers(0, 30, B).tolist(), 4, layers=1, kv_heads=1)
    a, fr, before = run_accept(s, 4)
    want = accept_by_hand(*s[1:6], before[0], None, s[6], s[7], s[8], 4)
    assert a.accepted.tolist() == want[0] and a.lens.tolist() == want[3] and int(a.free_count) == want[4]
    np.testing.assert_array_equal(fr.cpu().numpy(), want[7])
    assert torch.equal(s[0].pool, want[5])


def test_accept_refusals():
    from wf_bitnet import ops
    kv, parents, tokens, targets, offsets, lens, table, free, count = state(1, [5, 100], [4, 4], 16)
    ok = dict(parents=i32(parents), tokens=i32(tokens), targets=i32(targets), offsets=i32(offsets), seq_lens=i32(lens), kv=kv, block_table=i32(table), free_pages=i32(free), free_count=i32([count]))
    ops.tree_accept(**ok)
    for key, bad in (("parents", ok["parents"].long()), ("tokens", ok["tokens"][:-1]), ("targets", ok["targets"].cpu()), ("offsets", ok["offsets"][:-1]), ("seq_lens", ok["seq_lens"][:1]),
                     ("block_table", ok["block_table"][0]), ("free_pages", torch.stack([ok["free_pages"]] * 2, -1)[..., 0]), ("free_count", i32([1, 2]))):
        with pytest.raises(ValueError):
            ops.tree_accept(**{**ok, key: bad})
    with pytest.raises(NotImplementedError):
        ops.tree_accept(**{**ok, "kv": ops.PagedKV(4, 1, 1, 16, 12)})
