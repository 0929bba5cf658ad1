"""Block tables and slot maps planned on the GPU, and pages handed back, against the host's free list (sgl_kernel.kvcache.PageAllocator)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def plan_by_hand(lens, new, table, free, count, page, cap):
    """The same step with the host allocator's free list: (rows, positions, pages, slots, offsets, lens, count, table)."""
    from sgl_kernel.kvcache import PageAllocator
    pool = PageAllocator(1)
    pool._free = [int(x) for x in free[:count]]
    table = table.copy()
    rows, pos, pages, slots, offsets = [], [], [], [], [0]
    for b, (a, n) in enumerate(zip(lens, new)):
        old, after = -(-int(a) // page), -(-int(a + n) // page)
        table[b, old:after] = pool.allocate_pages(after - old).numpy() if after > old else []
        for p in range(a, a + n):
            rows.append(b), pos.append(p), pages.append(table[b, p // page]), slots.append(p % page)
        offsets.append(offsets[-1] + int(n))
    pad = cap - len(rows)
    i32 = lambda x, fill: np.array(list(x) + [fill] * pad, dtype=np.int32)  # noqa: E731
    return (i32(rows, -1), i32(pos, 0), i32(pages, -1), i32(slots, 0), np.array(offsets, np.int32), (lens + new).astype(np.int32), np.array([pool.num_free_pages()], np.int32), table)


def state(seed, rows, ctx, portion, page, blocks=None, spare=3):
    """lengths, new tokens, a table whose entries in use are distinct pages, and the free list of the others (junk beyond its end)"""
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, ctx + 1, rows).astype(np.int32)
    new = rng.integers(0, portion + 1, rows).astype(np.int32)
    have, after = -(-lens // page), -(-(lens + new) // page)
    blocks = blocks or int(max(1, after.max(initial=1)))
    order = rng.permutation(int(after.sum()) + spare).astype(np.int32)
    table = np.full((rows, blocks), -7, dtype=np.int32)
    at = 0
    for b in range(rows):
        table[b, :have[b]] = order[at:at + have[b]]
        at += have[b]
    free = np.full(len(order) + 2, -9, dtype=np.int32)
    free[:len(order) - at] = order[at:]
    return lens, new, table, free, len(order) - at


def run(lens, new, table, free, count, page, cap):
    from wf_bitnet import ops
    dev = [torch.from_numpy(x).cuda() for x in (lens, new, table, free)] + [torch.tensor([count], dtype=torch.int32, device="cuda")]
    before = [t.clone() for t in dev]
    p = ops.paged_plan(*dev, page, cap)
    for i in (0, 1, 3, 4):
        assert torch.equal(dev[i], before[i])            # lengths and the free list are only read
    return p, dev


SHAPES = [(1, 0, 1, 16), (1, 40, 1, 16), (3, 100, 1, 16), (32, 4096, 1, 16), (128, 50, 3, 1), (129, 300, 9, 7), (500, 1000, 60, 48), (513, 0, 33, 128), (2048, 200, 40, 16), (8192, 20, 2, 64)]


@pytest.mark.parametrize("rows, ctx, portion, page", SHAPES)
@pytest.mark.parametrize("pad", [0, 1, 515])
def test_plan_is_the_host_allocators(rows, ctx, portion, page, pad):
    s = state(rows + pad, rows, ctx, portion, page)
    cap = int(s[1].sum()) + pad
    want = plan_by_hand(*s, page, cap)
    p, dev = run(*s, page, cap)
    got = (p.rows, p.positions, p.pages, p.slots, p.offsets, p.lens, p.free_count, dev[2])
    for name, g, w in zip(("rows", "positions", "pages", "slots", "offsets", "lens", "free_count", "table"), got, want):
        np.testing.assert_array_equal(g.cpu().numpy(), w, err_msg=name)
    assert int(p.status) == 0


def test_no_requests_and_no_tokens():
    from wf_bitnet import ops
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    count = torch.tensor([2], dtype=torch.int32, device="cuda")
    p = ops.paged_plan(e, e, e.view(0, 4), torch.arange(2, dtype=torch.int32, device="cuda"), count, 16, 5)
    assert p.rows.tolist() == [-1] * 5 and p.pages.tolist() == [-1] * 5 and p.offsets.tolist() == [0] and p.lens.numel() == 0 and int(p.free_count) == 2 and int(p.status) == 0
    lens = torch.tensor([5, 0], dtype=torch.int32, device="cuda")
    p = ops.paged_plan(lens, torch.zeros_like(lens), torch.zeros(2, 1, dtype=torch.int32, device="cuda"), e, torch.zeros_like(count), 16, 0)
    assert p.rows.numel() == 0 and p.offsets.tolist() == [0, 0, 0] and p.lens.tolist() == [5, 0] and int(p.status) == 0


def test_long_positions_need_no_sum_beyond_31_bits():
    """A sequence that ends at 2^31 - 1 tokens, next to one that would pass it."""
    big = 2**31 - 1
    page = 2**20
    table = np.full((2, 2048), 5, dtype=np.int32)
    p, _ = run(np.array([big - 3, 0], np.int32), np.array([3, 1], np.int32), table, np.array([9, 8], np.int32), 2, page, 4)
    assert int(p.status) == 0 and p.positions.tolist() == [big - 3, big - 2, big - 1, 0] and p.pages.tolist() == [5, 5, 5, 8] and p.slots.tolist()[:3] == [page - 4, page - 3, page - 2]
    p, _ = run(np.array([big - 2, 0], np.int32), np.array([3, 1], np.int32), table, np.array([9, 8], np.int32), 2, page, 4)
    assert int(p.status) == 8


@pytest.mark.parametrize("why", ["pages", "tokens", "blocks", "negative", "negative length", "count", "count below zero", "two"])
def test_a_step_that_does_not_fit_is_not_planned(why):
    from wf_bitnet import ops
    lens, new, table, free, count = state(5, 200, 90, 8, 16, blocks=9)
    cap, status = int(new.sum()), None
    need = int((-(-(lens + new) // 16) - -(-lens // 16)).sum())
    if why == "pages":
        count, status = need - 1, ops.PLAN_PAGES
    elif why == "tokens":
        cap, status = cap - 1, ops.PLAN_TOKENS
    elif why == "blocks":
        lens[17], new[17], status = 140, 5, ops.PLAN_BLOCKS
        table[17] = 0
    elif why == "negative":
        new[3], status = -1, ops.PLAN_LENGTH
    elif why == "negative length":
        lens[199], status = -5, ops.PLAN_LENGTH
    elif why == "count":
        count, status = len(free) + 1, ops.PLAN_COUNT
    elif why == "count below zero":
        count, status = -1, ops.PLAN_COUNT | ops.PLAN_PAGES
    else:
        count, cap, status = 0, 3, ops.PLAN_PAGES | ops.PLAN_TOKENS
    p, dev = run(lens, new, table, free, count, 16, cap)
    assert int(p.status) == status
    assert (p.rows == -1).all() and (p.pages == -1).all() and not p.positions.any() and not p.slots.any() and not p.offsets.any()
    assert int(p.free_count) == count and np.array_equal(p.lens.cpu().numpy(), lens) and np.array_equal(dev[2].cpu().numpy(), table)


@pytest.mark.parametrize("rows, ctx, page", [(1, 0, 16), (1, 33, 16), (129, 300, 7), (512, 8192, 16), (4096, 60, 1)])
def test_release_puts_the_pages_on_top(rows, ctx, page):
    from sgl_kernel.kvcache import PageAllocator
    from wf_bitnet import ops
    lens, _, table, free, count = state(rows, rows, ctx, 0, page, blocks=-(-ctx // page) + 2)
    free = np.concatenate([free, np.full(int((-(-lens // page)).sum()), -3, np.int32)])
    done = np.random.default_rng(rows).random(rows) < 0.6
    pool = PageAllocator(len(free))
    pool._free = [int(x) for x in free[:count]]
    for b in np.flatnonzero(done):
        pool.free_pages(torch.from_numpy(table[b, :-(-int(lens[b]) // page)]))
    f, t = torch.from_numpy(free).cuda(), torch.from_numpy(table).cuda()
    new_lens, new_count = ops.paged_release(torch.from_numpy(done).cuda(), torch.from_numpy(lens).cuda(), t, f, torch.tensor([count], dtype=torch.int32, device="cuda"), page)
    assert int(new_count) == pool.num_free_pages() and new_lens.tolist() == np.where(done, 0, lens).tolist()
    want = free.copy()
    want[:len(pool._free)] = pool._free
    assert np.array_equal(f.cpu().numpy(), want) and np.array_equal(t.cpu().numpy(), table)


@pytest.mark.parametrize("why", ["full", "length", "blocks", "count"])
def test_release_that_does_not_fit_does_nothing(why):
    from wf_bitnet import ops
    lens, count = [40, 16, 3], 4
    f = torch.arange(8, dtype=torch.int32, device="cuda")
    if why == "length":
        lens[2] = -1
    elif why == "blocks":
        lens[1] = 65
    elif why == "count":
        count = 9
    before = f.clone()
    free = f if why != "full" else f[:7]
    args = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lens, [count])]
    new_lens, new_count = ops.paged_release(torch.tensor([True, True, why != "full"], device="cuda") if why != "full" else torch.ones(3, dtype=torch.bool, device="cuda"), args[0],
                                            torch.zeros(3, 4, dtype=torch.int32, device="cuda"), free, args[1], 16)
    assert torch.equal(f, before) and new_lens.tolist() == lens and int(new_count) == count


def test_wrong_arguments_are_refused():
    from wf_bitnet import ops
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    ok = dict(seq_lens=i(2), new_lens=i(2), block_table=i(2, 3), free_pages=i(4), free_count=i(1), page_size=16, max_tokens=4)
    ops.paged_plan(**ok)
    for key, bad in (("seq_lens", i(3)), ("new_lens", i(2).long()), ("new_lens", i(2, 1)), ("block_table", i(3, 2).T), ("free_count", i(2)), ("free_pages", i(4).cpu()), ("page_size", 0),
                     ("page_size", -16), ("max_tokens", -1), ("block_table", i(2, 3).float())):
        with pytest.raises(ValueError):
            ops.paged_plan(**{**ok, key: bad})
    with pytest.raises(NotImplementedError):
        ops.paged_plan(**{**ok, "seq_lens": i(8193), "new_lens": i(8193), "block_table": i(8193, 1)})
    ok = dict(done=i(2).bool(), seq_lens=i(2), block_table=i(2, 3), free_pages=i(4), free_count=i(1), page_size=16)
    ops.paged_release(**ok)
    for key, bad in (("done", i(2)), ("done", i(3).bool()), ("seq_lens", i(2).long()), ("free_pages", i(8)[::2]), ("page_size", 0), ("free_count", i(0))):
        with pytest.raises(ValueError):
            ops.paged_release(**{**ok, key: bad})


def test_strided_lengths_are_read_as_they_stand():
    from wf_bitnet import ops
    both = torch.tensor([[3, 2], [20, 1], [0, 4]], dtype=torch.int32, device="cuda")
    table = torch.tensor([[5, -1], [6, 7], [-1, -1]], dtype=torch.int32, device="cuda")
    p = ops.paged_plan(both[:, 0], both[:, 1], table, torch.arange(10, dtype=torch.int32, device="cuda")[::2], torch.tensor([5], dtype=torch.int32, device="cuda"), 16, 7)
    assert p.pages.tolist() == [5, 5, 7, 8, 8, 8, 8] and p.positions.tolist() == [3, 4, 20, 0, 1, 2, 3] and p.rows.tolist() == [0, 0, 1, 2, 2, 2, 2]
    assert table.tolist() == [[5, -1], [6, 7], [8, -1]] and int(p.free_count) == 4


def test_a_captured_step_goes_on_from_where_it_stopped():
    """Lengths and the count advance inside the graph: every replay plans the next token of every sequence, until the pages are gone."""
    from wf_bitnet import ops
    lens, count = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.tensor([5], dtype=torch.int32, device="cuda")
    new = torch.ones_like(lens)
    table, free = torch.full((3, 4), -1, dtype=torch.int32, device="cuda"), torch.arange(5, dtype=torch.int32, device="cuda")

    def step():
        p = ops.paged_plan(lens, new, table, free, count, 2, 4)
        lens.copy_(p.lens)
        count.copy_(p.free_count)
        return p

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    assert table[:, 0].tolist() == [4, 3, 2]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p = step()
    graph.replay()
    torch.cuda.synchronize()
    assert lens.tolist() == [2, 2, 2] and int(count) == 2 and p.slots.tolist() == [1, 1, 1, 0] and p.pages.tolist() == [4, 3, 2, -1]
    graph.replay()                                       # three pages wanted, two left
    torch.cuda.synchronize()
    assert int(p.status) == ops.PLAN_PAGES and lens.tolist() == [2, 2, 2] and int(count) == 2
    new.copy_(torch.tensor([1, 0, 1], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert int(p.status) == 0 and lens.tolist() == [3, 2, 3] and int(count) == 0 and p.pages.tolist() == [1, 0, -1, -1]
