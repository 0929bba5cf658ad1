"""Attention of drafted tokens over the paged cache against softmax in 64 bits over the same cache."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F64 = torch.float64
D = 128


@pytest.fixture(autouse=True)
def used_memory():
    """what is allocated next has been written before, so that an entry that a kernel leaves out shows"""
    if torch.cuda.is_available():
        kept = [torch.full((n // 4,), float("nan"), device="cuda") for n in [1 << 28] + [1 << 19] * 64]
        del kept


def words_of(bits):
    """bool [n, k] -> int64 [n, ceil(k / 64)]"""
    n, k = bits.shape
    w = -(-k // 64)
    x = torch.zeros(n, w * 64, dtype=torch.int64)
    x[:, :k] = bits.long()
    return (x.view(n, w, 64) << torch.arange(64)).sum(-1)


def tree_bits(n, gen):
    """a random tree of n drafts: which ones each has above it, itself too"""
    bits = torch.eye(n, dtype=torch.bool)
    for i in range(1, n):
        up = int(torch.randint(max(0, i - 6), i, (1,), generator=gen))
        bits[i] |= bits[up]
    return bits


def case(ctx, nodes, H, Hkv, page, int8=False, seed=0, layers=2, layer=1, pad=3, bits=None, words=None, blocks=None):
    """Queries, cache, tables in shuffled order, masks; whatever no sequence has is NaN (bf16) or has NaN scales (int8)."""
    from wf_bitnet import ops
    g = torch.Generator().manual_seed(seed)
    B, T = len(ctx), sum(nodes) + pad
    blocks = blocks or max([-(-(c + n) // page) for c, n in zip(ctx, nodes)] + [1])
    pages = B * blocks + 3
    kv = ops.PagedKV(pages, layers, Hkv, page, D, dtype=torch.int8 if int8 else torch.bfloat16)
    gg = torch.Generator(device="cuda").manual_seed(seed)
    if int8:
        kv.pool.copy_(torch.randint(1, 256, kv.pool.shape, generator=gg, device="cuda", dtype=torch.uint8))
        kv.scales.copy_(torch.rand(kv.scales.shape, generator=gg, device="cuda") * 0.01 + 0.015)
    else:
        kv.pool.copy_(torch.randn(kv.pool.shape, generator=gg, device="cuda", dtype=torch.bfloat16))
    table = torch.randperm(pages, generator=g)[:B * blocks].view(B, blocks).to(torch.int32)
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b in range(B):
        for j in range(-(-(ctx[b] + nodes[b]) // page)):
            used[table[b, j].long(), :min(page, ctx[b] + nodes[b] - j * page)] = True
    hole = ~used.cuda()[:, None, None, None].expand(pages, layers, 2, Hkv, page)
    target = kv.scales if int8 else kv.pool
    target[hole] = math.nan
    target[:, [i for i in range(layers) if i != layer]] = math.nan
    if bits is None:
        bits = [tree_bits(n, g) for n in nodes]
    words = words or -(-max([1] + list(nodes)) // 64)
    mask = torch.zeros(T, words, dtype=torch.int64)
    at, offsets = 0, [0]
    for n, x in zip(nodes, bits):
        if n:
            y = words_of(x)
            mask[at:at + n, :y.shape[1]] = y
        at += n
        offsets.append(at)
    q = torch.randn(T, H, D, generator=gg, device="cuda").to(torch.bfloat16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return dict(q=q, kv=kv, layer=layer, block_table=table.cuda(), seq_lens=i32(list(ctx)), offsets=i32(offsets), mask=mask.cuda()), bits


def keys_of(kv, pages, layer, which, head, n):
    x = kv.pool[pages.long(), layer, which, head].to(F64)
    if kv.dtype == torch.int8:
        x = (x - 128) * kv.scales[pages.long(), layer, which, head].to(F64)[..., None]
    return x.reshape(-1, D)[:n]


def check(a, bits, scale=None, out_dtype=torch.bfloat16):
    """Tolerance: weights enter the value product rounded to bf16 (half a step 2^-8 of each, so 2^-8 of sum p |v|), the result is rounded once (2^-8 of it in bf16, 2^-24 in
    float); scores are float sums of 128 products (130 half steps of sum |q k|, on p twice that), 2^x is off by 2^-22, or by 7.5e-5 < 2^-13 where a polynomial gives it
    (in the weights and in their sum: 2^-12), and up to n weights and n weighted values are added in float (2 n steps 2^-23)."""
    from wf_bitnet import ops
    out = ops.paged_tree_attn(**a, **({} if scale is None else {"scale": scale}), out_dtype=out_dtype)
    q, kv, layer = a["q"], a["kv"], a["layer"]
    assert out.dtype == out_dtype and out.shape == q.shape
    G, sc = q.shape[1] // kv.kv_heads, 1 / math.sqrt(D) if scale is None else scale
    off, lens = a["offsets"].tolist(), a["seq_lens"].tolist()
    for b, see in enumerate(bits):
        n, c = off[b + 1] - off[b], lens[b]
        if n == 0:
            continue
        hidden = torch.cat([torch.zeros(n, c, dtype=torch.bool), ~see[:n, :n]], 1).cuda()
        for h in range(kv.kv_heads):
            got = out[off[b]:off[b + 1], h * G:(h + 1) * G].to(F64)
            k, v = (keys_of(kv, a["block_table"][b], layer, w, h, c + n) for w in (0, 1))
            qh = q[off[b]:off[b + 1], h * G:(h + 1) * G].to(F64)
            s = (qh @ k.T * sc).masked_fill(hidden[:, None], -math.inf)
            p = torch.softmax(s, -1)
            p = torch.where(hidden.all(-1)[:, None, None], 0.0, p)
            want, mag = p @ v, p @ v.abs()
            wide = 2 * 130 * 2.0**-24 * float((qh.abs() @ k.abs().T).max()) * abs(sc) + 2.0**-12 + 2 * k.shape[0] * 2.0**-23
            tol = (2.0**-8 if out_dtype == torch.bfloat16 else 2.0**-24) * want.abs() + (2.0**-8 + wide) * mag
            assert bool(((got - want).abs() <= tol * 1.01).all()), (b, h, float(((got - want).abs() - tol).max()))
    assert not out[off[-1]:].any()                       # rows of no sequence
    return out


HEADS = [(1, 1), (4, 4), (20, 5), (32, 8), (8, 1), (6, 2)]


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("ctx", [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 191, 1000, 4097])
def test_lengths(ctx, int8):
    check(*case([ctx, max(0, ctx - 1), ctx // 2], [7, 20, 1], 20, 5, 16, int8, ctx))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 255, 256])
def test_drafts(n, int8):
    """trees that fill their words and rows' tiles, just and not quite; the last words at every place of a tile of keys"""
    check(*case([100, 321], [n, max(1, n - 3)], 8, 2, 16, int8, n))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("H, Hkv", HEADS)
@pytest.mark.parametrize("B", [1, 2, 33])
def test_heads_and_batches(B, H, Hkv, int8):
    check(*case([(37 * b) % 300 for b in range(B)], [(5 * b) % 13 for b in range(B)] if B > 1 else [9], H, Hkv, 32, int8, B + H))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("page", [16, 32, 48, 64, 80, 128, 144, 256, 272])
def test_page_sizes(page, int8):
    check(*case([777, 3, 290], [13, 60, 2], 4, 2, page, int8, page))


@pytest.mark.parametrize("int8", [False, True])
def test_long_and_short_together(int8):
    """one long sequence is cut over many blocks beside sequences with a block each"""
    check(*case([20000] + [(17 * b) % 90 for b in range(40)], [50] + [b % 4 for b in range(40)], 8, 2, 16, int8, 5))


@pytest.mark.parametrize("int8", [False, True])
def test_more_row_tiles_than_sms(int8):
    check(*case([60 + b for b in range(30)], [40 + 6 * (b % 37) for b in range(30)], 64, 8, 16, int8, 6))


@pytest.mark.parametrize("int8", [False, True])
def test_any_pattern_of_bits(int8):
    """rows that see drafts behind them, none at all, all; without a context a row that sees none has zeros"""
    g = torch.Generator().manual_seed(1)
    bits = [torch.rand(n, n, generator=g) < 0.3 for n in (70, 130, 5)]
    bits[0][3], bits[1][:64], bits[2][:] = False, False, False
    bits[0][4] = True
    out = check(*case([0, 50, 0], [70, 130, 5], 8, 2, 16, int8, 1, bits=bits))
    assert not out[3].any() and not out[200:205].any()


def test_bits_behind_the_last_draft_count_for_nothing():
    a, bits = case([40, 3], [10, 70], 8, 2, 16, seed=2, words=2)
    want = check(a, bits)
    from wf_bitnet import ops
    a["mask"][:10, 0] |= ~torch.tensor((1 << 10) - 1, device="cuda")
    a["mask"][:10, 1] = -1
    a["mask"][10:80, 1] |= ~torch.tensor((1 << 6) - 1, device="cuda")
    a["mask"][80:] = -1
    assert torch.equal(ops.paged_tree_attn(**a), want)
    a["mask"] = torch.cat([a["mask"], torch.full_like(a["mask"], -1)], 1)
    assert torch.equal(ops.paged_tree_attn(**a), want)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("ctx, n", [(70, 90), (0, 20), (3000, 33)])
def test_what_a_row_does_not_see_has_no_weight(ctx, n, value, int8):
    """values and keys that are not finite: of rows that do not see them the result is as without them, of the others it is not finite"""
    from wf_bitnet import ops
    a, bits = case([ctx, 5], [n, 3], 8, 2, 16, int8, 7)
    clean = ops.paged_tree_attn(**a, out_dtype=torch.float32)
    j = n // 2
    page, slot = a["block_table"][0, (ctx + j) // 16].long(), (ctx + j) % 16
    target = a["kv"].scales if int8 else a["kv"].pool
    for which in (1, 0):
        target[page, a["layer"], which, :, slot] = value
        out = ops.paged_tree_attn(**a, out_dtype=torch.float32)
        blind = ~bits[0][:, j]
        keep = torch.cat([blind, torch.ones(3 + 3, dtype=torch.bool)]).cuda()
        # the same weights in float instead of rounded to bf16 where a row was taken again
        assert bool(((out[keep] - clean[keep]).abs() <= 2.0**-7 * 4).all())
        assert out[~keep].isfinite().sum() < out[~keep].numel()
        if which == 1 and not math.isnan(value) and not int8:
            assert bool((out[~keep] == value).all())
        target[page, a["layer"], which, :, slot] = 0.02 if int8 else 1.0
        clean = ops.paged_tree_attn(**a, out_dtype=torch.float32)


def test_rows_taken_again_are_right():
    """against 64 bits, the hidden value left out of it"""
    from wf_bitnet import ops
    ctx, n = 200, 40
    a, bits = case([ctx], [n], 8, 2, 16, seed=8, pad=0)
    j = 20
    page, slot = a["block_table"][0, (ctx + j) // 16].long(), (ctx + j) % 16
    a["kv"].pool[page, a["layer"], 1, :, slot] = math.nan
    out = ops.paged_tree_attn(**a)
    blind = ~bits[0][:, j]
    assert bool(blind.any()) and out[~blind.cuda()].isnan().all()
    a["kv"].pool[page, a["layer"], 1, :, slot] = 0.0
    rows = blind.nonzero()[:, 0]
    G = 4
    for h in range(2):
        k, v = (keys_of(a["kv"], a["block_table"][0], a["layer"], w, h, ctx + n) for w in (0, 1))
        hidden = torch.cat([torch.zeros(n, ctx, dtype=torch.bool), ~bits[0]], 1).cuda()[rows.cuda()]
        p = torch.softmax((a["q"][rows.cuda(), h * G:(h + 1) * G].to(F64) @ k.T / math.sqrt(D)).masked_fill(hidden[:, None], -math.inf), -1)
        got = out[rows.cuda(), h * G:(h + 1) * G].to(F64)
        assert bool(((got - p @ v).abs() <= 2.0**-8 * (p @ v).abs() + (2.0**-8 + 2.0**-11) * (p @ v.abs())).all())


@pytest.mark.parametrize("int8", [False, True])
def test_hidden_values_behind_a_long_context(int8):
    """values of several drafts that are not finite, some in one column alone; every row has the numbers of the clean ones, or what is not finite, where the formula has them"""
    from wf_bitnet import ops
    ctx, n = 60000, 60
    a, bits = case([ctx, 100], [n, 9], 16, 2, 16, int8, 21)
    clean = ops.paged_tree_attn(**a, out_dtype=torch.float32)
    spoilt = torch.zeros(n, D, dtype=torch.bool)
    for j, columns, value in ((7, slice(None), math.nan), (23, slice(5, 6), math.inf), (59, slice(64, 130), -math.inf)):
        page, slot = a["block_table"][0, (ctx + j) // 16].long(), (ctx + j) % 16
        if int8:
            a["kv"].scales[page, a["layer"], 1, :, slot] = value
            columns = slice(None)
        else:
            a["kv"].pool[page, a["layer"], 1, :, slot, columns] = value
        spoilt[:, columns] |= bits[0][:, j, None]
    out = ops.paged_tree_attn(**a, out_dtype=torch.float32)
    s = spoilt[:, None].expand(n, 16, D).cuda()
    assert not out[:n][s].isfinite().any()
    # the clean result has the hidden value's own (a weight of one in 60000 of a value of at most 6) where this one has none
    assert bool(((out[:n] - clean[:n])[~s].abs() <= 2.0**-7 * 4).all())
    assert torch.equal(out[n:n + 9], clean[n:n + 9])


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("n", [20, 200])
def test_a_row_that_sees_nothing_beside_a_hidden_nan(n, int8):
    """with one block a tile and with several: zeros, whatever the hidden value is"""
    from wf_bitnet import ops
    empty = torch.arange(n) % 3 == 1
    bits = tree_bits(n, torch.Generator().manual_seed(4))
    bits[:, 0] = True
    bits[empty] = False
    a, _ = case([0], [n], 8, 2, 16, int8, 6, bits=[bits])
    target = a["kv"].scales if int8 else a["kv"].pool
    target[a["block_table"][0, 0].long(), a["layer"], 1, :, 0] = math.nan
    out = ops.paged_tree_attn(**a, out_dtype=torch.float32)[:n]
    assert bool((out[empty.cuda()] == 0).all()) and bool(out[~empty.cuda()].isnan().all())


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("wide", [False, True])
def test_many_short_sequences(wide, int8):
    """a block has many row tiles one after another, of one group's rows and (wide) of two groups', some sequences without any"""
    g = torch.Generator().manual_seed(11 + wide)
    nodes = torch.randint(0, 6, (300,), generator=g).tolist()
    ctx = torch.randint(0, 140, (300,), generator=g).tolist()
    if wide:
        for b in range(0, 300, 7):
            nodes[b] = int(torch.randint(33, 130, (1,), generator=g))
    check(*case(ctx, nodes, 8, 2, 16, int8, 12, pad=2000))


@pytest.mark.parametrize("int8", [False, True])
def test_a_long_sequence_among_short_ones(int8):
    check(*case([3, 0, 30011, 64, 7, 9000], [1, 9, 40, 0, 100, 2], 16, 2, 64, int8, 13))


@pytest.mark.parametrize("int8", [False, True])
def test_sequences_without_drafts_and_with_too_many(int8):
    from wf_bitnet import ops
    a, bits = case([50, 20, 30], [0, 70, 9], 8, 2, 16, int8, 3)
    check(a, bits)
    b, _ = case([50, 20, 30], [0, 70, 9], 8, 2, 16, int8, 3)
    b["mask"] = b["mask"][:, :1].contiguous()            # words for 64 drafts: the sequence of 70 is left out
    out = ops.paged_tree_attn(**b)
    assert not out[:70].any() and torch.equal(out[70:], ops.paged_tree_attn(**a)[70:])
    c, _ = case([50], [0], 8, 2, 16, int8, 3)
    assert not ops.paged_tree_attn(**c).any()
    a["seq_lens"][1] = -1
    assert not ops.paged_tree_attn(**a)[:70].any()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("scale", [0.0, 0.02, 1.0, -0.1])
def test_scales_and_float_output(scale, int8):
    check(*case([500, 3], [30, 70], 8, 2, 16, int8), scale=scale, out_dtype=torch.float32)
    check(*case([100 + b for b in range(80)], [3] * 80, 8, 8, 16, int8), scale=scale, out_dtype=torch.float32)


def test_scores_of_hundreds():
    a, bits = case([900, 0], [30, 70], 8, 2, 16)
    a["q"] = a["q"] * 30
    check(a, bits)


def test_keys_of_minus_infinity():
    """a score of -inf has no weight; a row with none but those has zeros"""
    a, bits = case([40], [3], 4, 1, 16, pad=0)
    from wf_bitnet import ops
    a["q"] = a["q"].abs() + 0.1
    a["kv"].pool[:, a["layer"], 0] = -math.inf
    assert not ops.paged_tree_attn(**a).any()


def test_one_draft_is_decode_attention():
    from wf_bitnet import ops
    a, bits = case([1, 100, 999, 2048, 16], [1] * 5, 32, 8, 16, pad=0)
    got = ops.paged_tree_attn(**a, out_dtype=torch.float32)
    want = ops.paged_decode_attn(a["q"], a["kv"], a["layer"], a["block_table"], a["seq_lens"] + 1, out_dtype=torch.float32)
    # weights rounded to bf16 here and there alike, sums in another order; values are below 6
    assert bool(((got - want).abs() <= 2 * 2.0**-8 * 6).all())


def test_queries_inside_a_wider_row_and_off_alignment():
    from wf_bitnet import ops
    a, bits = case([200, 31], [9, 30], 8, 2, 16)
    want = check(a, bits)
    q = a["q"]
    T = q.shape[0]
    wide = torch.randn(T, 14 * D, device="cuda").to(torch.bfloat16)
    wide[:, D:9 * D] = q.view(T, -1)
    assert torch.equal(ops.paged_tree_attn(**{**a, "q": wide[:, D:9 * D].view(T, 8, D)}), want)
    odd = torch.empty(q.numel() + 3, dtype=torch.bfloat16, device="cuda")[3:].view_as(q)
    odd.copy_(q)
    assert torch.equal(ops.paged_tree_attn(**{**a, "q": odd}), want)
    two = torch.stack([a["block_table"], a["block_table"].flip(0)], -1)[..., 0]
    assert torch.equal(ops.paged_tree_attn(**{**a, "block_table": two, "mask": torch.stack([a["mask"], a["mask"]], -1)[..., 0]}), want)


def test_the_same_page_twice():
    a, bits = case([96, 40], [10, 10], 4, 2, 16)
    a["block_table"][0, 3] = a["block_table"][0, 0]
    a["block_table"][1, 1] = a["block_table"][0, 1]
    check(a, bits)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("page", [-1, 40000, 2**29, 2**31 - 1, -2**31])
def test_what_is_no_page_reads_as_zeros(page, int8):
    """numbers beyond the pool, 2^29 among them, which times the 8 heads' rows of a page here is 0 in 32 bits"""
    from wf_bitnet import ops
    a, _ = case([96, 40], [10, 10], 8, 2, 16, int8)
    blank = int(a["block_table"][0, 3])
    a["kv"].pool[blank] = 128 if int8 else 0
    if int8:
        a["kv"].scales[blank] = 0.0
    want = ops.paged_tree_attn(**a)
    a["block_table"][0, 3] = page
    assert torch.equal(ops.paged_tree_attn(**a), want)


def test_a_table_that_ends_inside_the_drafts():
    """the keys end with the table's row: nothing behind it is read"""
    from wf_bitnet import ops
    a, bits = case([60], [10], 4, 2, 16, pad=0)
    a["block_table"] = a["block_table"][:, :4].contiguous()                # 64 tokens
    see = bits[0].clone()
    see[:, 4:] = False
    want, _ = case([60], [10], 4, 2, 16, pad=0)
    want["mask"] = words_of(see).cuda()
    assert torch.equal(ops.paged_tree_attn(**a), ops.paged_tree_attn(**want))


def test_offsets_beyond_31_bits():
    from wf_bitnet import ops
    pages = 70000                                        # 70000 x 2 x 8 x 16 x 128 = 2.3e9 entries
    kv = ops.PagedKV(pages, 1, 8, 16, D)
    g = torch.Generator(device="cuda").manual_seed(0)
    kv.pool[-50:] = torch.randn(50, 1, 2, 8, 16, D, generator=g, device="cuda").to(torch.bfloat16)
    table = torch.arange(pages - 30, pages, device="cuda", dtype=torch.int32).flip(0)[None].contiguous()
    bits = [tree_bits(20, torch.Generator().manual_seed(0))]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.randn(20, 8, D, generator=g, device="cuda").to(torch.bfloat16)
    check(dict(q=q, kv=kv, layer=0, block_table=table, seq_lens=i32([401]), offsets=i32([0, 20]), mask=words_of(bits[0]).cuda()), bits)


def test_wrong_arguments_are_refused():
    from wf_bitnet import ops
    a, _ = case([20, 3], [5, 6], 8, 2, 16)
    ops.paged_tree_attn(**a)
    for key, bad in (("q", a["q"].float()), ("q", a["q"][0]), ("q", a["q"][..., :64]), ("q", a["q"][:-1]), ("layer", 2), ("layer", -1), ("block_table", a["block_table"][:1]),
                     ("block_table", a["block_table"].long()), ("seq_lens", a["seq_lens"][:1]), ("seq_lens", a["seq_lens"].cpu()), ("offsets", a["offsets"][:2]), ("mask", a["mask"].int()),
                     ("mask", a["mask"][:, :0]), ("mask", a["mask"][:-1]), ("out_dtype", torch.float16)):
        with pytest.raises(ValueError):
            ops.paged_tree_attn(**{**a, key: bad})
    with pytest.raises(NotImplementedError):
        ops.paged_tree_attn(**{**a, "mask": torch.zeros(14, 5, dtype=torch.int64, device="cuda")})
    for other in (ops.PagedKV(4, 2, 3, 16, D), ops.PagedKV(4, 2, 2, 24, D), ops.PagedKV(4, 2, 2, 16, D, dtype=torch.float32)):
        with pytest.raises(NotImplementedError):
            ops.paged_tree_attn(**{**a, "kv": other})
    assert ops.paged_tree_attn(**{**a, "q": a["q"][:0], "mask": a["mask"][:0]}).shape == (0, 8, D)
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    assert not ops.paged_tree_attn(**{**a, "block_table": e.view(0, 3), "seq_lens": e, "offsets": torch.zeros(1, dtype=torch.int32, device="cuda")}).any()


@pytest.mark.parametrize("int8", [False, True])
def test_graphs_and_streams_side_by_side(int8):
    """two captured graphs of different sizes, replayed together on two streams over new queries"""
    from wf_bitnet import ops
    cases = [case([3000 + b for b in range(9)], [b + 1 for b in range(9)], 20, 5, 16, int8, 1)[0], case([100], [250], 32, 8, 32, int8, 2)[0]]
    streams, graphs, outs = [torch.cuda.Stream() for _ in cases], [], []
    for a in cases:
        ops.paged_tree_attn(**a)
    torch.cuda.synchronize()
    for a in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.paged_tree_attn(**a))
        graphs.append(g)
    for turn in range(3):
        for a in cases:
            a["q"].copy_(torch.randn(a["q"].shape, device="cuda"))
            a["seq_lens"] -= turn
        torch.cuda.synchronize()
        for _ in range(10):
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for a, o in zip(cases, outs):
            assert torch.equal(o, ops.paged_tree_attn(**a))


@pytest.mark.parametrize("int8", [False, True])
def test_tiles_of_one_group_and_of_two_in_turn(int8):
    """row tiles of up to 128 rows beside wider ones, in rings of an odd number of tiles: three streams at a time, the same bits every time"""
    from wf_bitnet import ops
    a, bits = case([115, 9035, 0, 2681, 5288, 1809, 0, 5982, 3300], [145, 252, 249, 86, 128, 52, 122, 173, 74], 64, 8, 32, int8, 31, pad=60)
    want = check(a, bits)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(40):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.paged_tree_attn(**a))
        torch.cuda.synchronize()
        assert all(torch.equal(x, want) for x in got)
