"""Decode attention behind a shared prefix against softmax in 64 bits over the same cache."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F64 = torch.float64
D = 128


def cache(pages, layers, kv_heads, page, int8, seed, q_scale=1.0):
    from wf_bitnet import ops
    g = torch.Generator(device="cuda").manual_seed(seed)
    kv = ops.PagedKV(pages, layers, kv_heads, page, D, dtype=torch.int8 if int8 else torch.bfloat16)
    if int8:
        kv.pool.copy_(torch.randint(1, 256, kv.pool.shape, generator=g, device="cuda", dtype=torch.uint8))
        kv.scales.copy_(torch.rand(kv.scales.shape, generator=g, device="cuda") * 0.01 + 0.015)
    else:
        kv.pool.copy_(torch.randn(kv.pool.shape, generator=g, device="cuda", dtype=torch.bfloat16) * q_scale)
    return kv


def rows_of(kv, pages, layer, which, head, n):
    x = kv.pool[pages.long(), layer, which, head].to(F64)
    if kv.dtype == torch.int8:
        x = (x - 128) * kv.scales[pages.long(), layer, which, head].to(F64)[..., None]
    return x.reshape(-1, D)[:n]


def check(q, kv, layer, ptable, prefix, table, lens, scale=None, out_dtype=torch.bfloat16):
    """Tolerance: weights enter the value product rounded to 16 bits (half a step 2^-8 of each, that of bf16, so 2^-8 of sum p |v|), the result is rounded once (2^-8 of it in
    bf16, 2^-24 in float); scores are float sums of 128 products (130 half steps of sum |q k|, on p twice that), 2^x is off by 2^-22, or by
    7.5e-5 < 2^-13 where a polynomial gives it (in the weights and in their sum: 2^-12), and up to n weights and n weighted values are added in float
    (2 n steps 2^-23)."""
    from wf_bitnet import ops
    out = ops.paged_prefix_attn(q, kv, layer, ptable, prefix, table, lens, scale, out_dtype)
    assert out.dtype == out_dtype and out.shape == q.shape
    B, H, _ = q.shape
    G = H // kv.kv_heads
    sc = 1 / math.sqrt(D) if scale is None else scale
    for b in range(B):
        n = int(lens[b])
        for h in range(kv.kv_heads):
            k = torch.cat([rows_of(kv, ptable, layer, 0, h, prefix), rows_of(kv, table[b], layer, 0, h, n)])
            v = torch.cat([rows_of(kv, ptable, layer, 1, h, prefix), rows_of(kv, table[b], layer, 1, h, n)])
            got = out[b, h * G:(h + 1) * G].to(F64)
            if k.shape[0] == 0:
                assert not got.any()
                continue
            qh = q[b, h * G:(h + 1) * G].to(F64)
            p = torch.softmax(qh @ k.T * sc, -1)
            want, mag = p @ v, p @ v.abs()
            off = 2 * 130 * 2.0**-24 * float((qh.abs() @ k.abs().T).max()) * abs(sc) + 2.0**-12 + 2 * k.shape[0] * 2.0**-23
            tol = (2.0**-8 if out_dtype == torch.bfloat16 else 2.0**-24) * want.abs() + (2.0**-8 + off) * mag
            assert bool(((got - want).abs() <= tol * 1.01).all()), (b, h, ((got - want).abs() - tol).max())


def case(B, H, Hkv, prefix, lens, page, int8, seed=0, layers=2, layer=1, spare=3):
    """queries, cache, tables in shuffled order; whatever no sequence reads is NaN (bf16) or has NaN scales (int8)"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    blocks, pb = max([-(-n // page) for n in lens] + [0]), -(-prefix // page)
    pages = B * blocks + pb + spare
    kv = cache(pages, layers, Hkv, page, int8, seed)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    ptable, table = order[:pb].clone(), order[pb:pb + B * blocks].view(B, blocks).clone()
    used = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    for t, n in [(ptable, prefix)] + [(table[b], lens[b]) for b in range(B)]:
        for j in range(-(-n // page)):
            used[t[j].long(), :min(page, n - j * page)] = True
    target = kv.scales if int8 else kv.pool
    hole = ~used[:, None, None, None].expand(pages, layers, 2, Hkv, page)
    target[hole] = math.nan
    target[:, [i for i in range(layers) if i != layer]] = math.nan
    q = torch.randn(B, H, D, generator=g, device="cuda").to(torch.bfloat16)
    return q, kv, layer, ptable, prefix, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


HEADS = [(1, 1), (4, 4), (20, 5), (32, 8), (8, 1)]


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 127, 128, 129, 255, 257, 1000, 4097])
def test_prefix_lengths(prefix, int8):
    check(*case(3, 20, 5, prefix, [1, 40, 17], 16, int8, prefix))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("H, Hkv", HEADS)
@pytest.mark.parametrize("B", [1, 2, 33])
def test_heads_and_batches(B, H, Hkv, int8):
    check(*case(B, H, Hkv, 300, [(7 * b) % 50 for b in range(B)], 32, int8, B + H))


@pytest.mark.parametrize("B, H, Hkv, prefix", [(64, 8, 1, 700), (65, 4, 1, 385), (127, 8, 2, 900), (130, 8, 1, 2050), (256, 2, 1, 130)])
def test_many_rows(B, H, Hkv, prefix):
    """row tiles that are full, just over, part full"""
    check(*case(B, H, Hkv, prefix, [b % 5 for b in range(B)], 16, False, B))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("page", [16, 32, 48, 64, 80, 128, 144, 256, 272])
def test_page_sizes(page, int8):
    """pages smaller and larger than a tile of keys, and ones that end inside it"""
    check(*case(3, 4, 2, 777, [3, 290, 0], page, int8, page))


@pytest.mark.parametrize("int8", [False, True])
def test_no_prefix_no_own_keys_no_keys(int8):
    check(*case(3, 8, 2, 0, [5, 0, 33], 16, int8))
    check(*case(3, 8, 2, 200, [0, 0, 0], 16, int8))
    check(*case(2, 8, 2, 0, [0, 0], 16, int8))
    q, kv, layer, pt, prefix, table, lens = case(2, 8, 2, 200, [0, 20], 16, int8)
    check(q, kv, layer, pt, prefix, table, torch.zeros_like(lens))


def test_without_prefix_as_paged_decode_attention():
    from wf_bitnet import ops
    q, kv, layer, pt, prefix, table, lens = case(5, 32, 8, 0, [1, 100, 999, 2048, 16], 16, False)
    got = ops.paged_prefix_attn(q, kv, layer, pt, 0, table, lens, out_dtype=torch.float32)
    want = ops.paged_decode_attn(q, kv, layer, table, lens, out_dtype=torch.float32)
    # the same partial sums joined in another order: float steps of the sums of up to 16 parts
    assert bool(((got - want).abs() <= 64 * 2.0**-23 * want.abs().amax()).all())


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("scale", [0.0, 0.02, 1.0, -0.1])
def test_scales_and_float_output(scale, int8):
    check(*case(4, 8, 2, 500, [3, 1, 0, 70], 16, int8), scale=scale, out_dtype=torch.float32)


def test_scores_of_hundreds():
    """the running maximum grows and the first keys' weights vanish"""
    q, kv, layer, pt, prefix, table, lens = case(4, 8, 2, 900, [3, 1, 0, 70], 16, False)
    q = q * 30
    check(q, kv, layer, pt, prefix, table, lens)


def test_infinite_keys_and_values():
    """a score of -inf has no weight, whatever splits and tiles its key falls in; one key of NaN makes its rows NaN and no others"""
    from wf_bitnet import ops
    q, kv, layer, pt, prefix, table, lens = case(2, 4, 2, 400, [5, 9], 16, False)
    q = q.abs()
    clean = ops.paged_prefix_attn(q, kv, layer, pt, prefix, table, lens)
    kv.pool[pt[10].long(), layer, 0, 1, 3] = math.nan
    out = ops.paged_prefix_attn(q, kv, layer, pt, prefix, table, lens)
    assert out[:, 2:].isnan().all() and torch.equal(out[:, :2], clean[:, :2])
    kv.pool[pt[10].long(), layer, 0, 1, 3] = -math.inf
    out = ops.paged_prefix_attn(q, kv, layer, pt, prefix, table, lens).to(F64)
    keep = [j for j in range(400) if j != 163]
    for b in range(2):
        k = torch.cat([rows_of(kv, pt, layer, 0, 1, 400)[keep], rows_of(kv, table[b], layer, 0, 1, int(lens[b]))])
        v = torch.cat([rows_of(kv, pt, layer, 1, 1, 400)[keep], rows_of(kv, table[b], layer, 1, 1, int(lens[b]))])
        p = torch.softmax(q[b, 2:].to(F64) @ k.T / math.sqrt(D), -1)
        assert bool(((out[b, 2:] - p @ v).abs() <= 2.0**-8 * (p @ v).abs() + (2.0**-8 + 2.0**-12) * (p @ v.abs())).all())
    assert torch.equal(out[:, :2], clean[:, :2].to(F64))


def test_first_keys_of_minus_infinity():
    """a whole tile of keys without weight before the first that has one"""
    q, kv, layer, pt, prefix, table, lens = case(2, 4, 1, 600, [5, 0], 16, False)
    q = q.abs() + 0.1
    for j in range(16):
        kv.pool[pt[j].long(), layer, 0, 0] = -math.inf
    from wf_bitnet import ops
    out = ops.paged_prefix_attn(q, kv, layer, pt, prefix, table, lens).to(F64)
    for b in range(2):
        k = torch.cat([rows_of(kv, pt, layer, 0, 0, 600)[256:], rows_of(kv, table[b], layer, 0, 0, int(lens[b]))])
        v = torch.cat([rows_of(kv, pt, layer, 1, 0, 600)[256:], rows_of(kv, table[b], layer, 1, 0, int(lens[b]))])
        p = torch.softmax(q[b].to(F64) @ k.T / math.sqrt(D), -1)
        assert bool(((out[b] - p @ v).abs() <= 2.0**-8 * (p @ v).abs() + (2.0**-8 + 2.0**-11) * (p @ v.abs())).all())


def test_queries_inside_a_wider_row_and_off_alignment():
    from wf_bitnet import ops
    q, kv, layer, pt, prefix, table, lens = case(3, 8, 2, 200, [3, 1, 30], 16, False)
    want = ops.paged_prefix_attn(q, kv, layer, pt, prefix, table, lens)
    wide = torch.randn(3, 14 * D, device="cuda").to(torch.bfloat16)
    wide[:, D:9 * D] = q.view(3, -1)
    assert torch.equal(ops.paged_prefix_attn(wide[:, D:9 * D].view(3, 8, D), kv, layer, pt, prefix, table, lens), want)
    odd = torch.empty(q.numel() + 3, dtype=torch.bfloat16, device="cuda")[3:].view_as(q)
    odd.copy_(q)
    assert torch.equal(ops.paged_prefix_attn(odd, kv, layer, pt, prefix, table, lens), want)
    two = torch.stack([table, table.flip(0)], -1)[..., 0]      # entries 8 bytes apart
    assert not two.is_contiguous() and torch.equal(ops.paged_prefix_attn(q, kv, layer, pt, prefix, two, lens), want)


def test_the_same_page_twice():
    q, kv, layer, pt, prefix, table, lens = case(2, 4, 2, 96, [20, 3], 16, False)
    pt[3] = pt[0]
    table[0, 0] = pt[0]
    check(q, kv, layer, pt, prefix, table, lens)


def test_offsets_beyond_31_bits():
    from wf_bitnet import ops
    pages = 70000                                        # 70000 x 2 x 8 x 16 x 128 = 2.3e9 entries
    kv = ops.PagedKV(pages, 1, 8, 16, D)
    g = torch.Generator(device="cuda").manual_seed(0)
    pt = torch.randint(pages - 30, pages, (20,), generator=g, device="cuda", dtype=torch.int32)
    table = torch.tensor([[pages - 1, pages - 40]], dtype=torch.int32, device="cuda")
    kv.pool[-50:] = torch.randn(50, 1, 2, 8, 16, D, generator=g, device="cuda").to(torch.bfloat16)
    q = torch.randn(1, 8, D, generator=g, device="cuda").to(torch.bfloat16)
    check(q, kv, 0, pt, 313, table, torch.tensor([25], dtype=torch.int32, device="cuda"))


def test_wrong_arguments_are_refused():
    from wf_bitnet import ops
    q, kv, layer, pt, prefix, table, lens = case(2, 8, 2, 100, [20, 3], 16, False)
    ok = dict(q=q, kv=kv, layer=layer, prefix_table=pt, prefix_len=prefix, block_table=table, seq_lens=lens)
    ops.paged_prefix_attn(**ok)
    for key, bad in (("q", q.float()), ("q", q[0]), ("q", q[..., :64]), ("layer", 2), ("layer", -1), ("prefix_table", pt.long()), ("prefix_len", 113), ("prefix_len", -1), ("block_table", table[:1]),
                     ("block_table", table[0]), ("seq_lens", lens[:1]), ("seq_lens", lens.cpu()), ("out_dtype", torch.float16)):
        with pytest.raises(ValueError):
            ops.paged_prefix_attn(**{**ok, key: bad})
    for other in (ops.PagedKV(4, 1, 3, 16, D), ops.PagedKV(4, 1, 2, 24, D), ops.PagedKV(4, 2, 2, 16, D, dtype=torch.float32)):
        with pytest.raises(NotImplementedError):
            ops.paged_prefix_attn(q, other, 0, pt, 0, table[:, :0], lens)
    with pytest.raises(NotImplementedError):
        ops.paged_prefix_attn(torch.zeros(1, 18, D, dtype=torch.bfloat16, device="cuda"), kv, 0, pt, 0, table[:1], lens[:1])
    empty = ops.paged_prefix_attn(q[:0], kv, layer, pt, prefix, table[:0], lens[:0])
    assert empty.shape == (0, 8, D)


@pytest.mark.parametrize("int8", [False, True])
def test_graphs_and_streams_side_by_side(int8):
    """two captured graphs of different sizes, replayed together on two streams"""
    from wf_bitnet import ops
    a = case(40, 20, 5, 3000, [b % 60 + 1 for b in range(40)], 16, int8, 1)
    b = case(9, 32, 8, 700, [300 + b for b in range(9)], 32, int8, 2)
    want = [ops.paged_prefix_attn(*c) for c in (a, b)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.paged_prefix_attn(*c))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for o in outs:
        o.zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(outs, want))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("B, H, Hkv, prefix, lens", [(3, 32, 8, 500, [6000, 300, 0]), (2, 8, 1, 3000, [20000, 16385]), (1, 4, 4, 40, [5121])])
def test_long_own_parts(B, H, Hkv, prefix, lens, int8):
    """sequences of many chunks: more of them than the merge asks for at once"""
    check(*case(B, H, Hkv, prefix, lens, 16, int8, 4))


@pytest.mark.parametrize("B, own", [(128, 120), (256, 300), (300, 40)])
def test_wide_merges(B, own):
    """many rows: the merge takes 8 or 16 columns a thread"""
    q, kv, layer, pt, prefix, table, lens = case(B, 32, 8, 700, [(7 * b) % own for b in range(B)], 16, False, 6, layers=1, layer=0)
    some = [0, 1, B // 2, B - 1]
    from wf_bitnet import ops
    out = ops.paged_prefix_attn(q, kv, layer, pt, prefix, table, lens)
    for b in some:                                       # a sequence by itself: held against 64 bits by check
        check(q[b:b + 1], kv, layer, pt, prefix, table[b:b + 1], lens[b:b + 1])
        alone = ops.paged_prefix_attn(q[b:b + 1], kv, layer, pt, prefix, table[b:b + 1], lens[b:b + 1])
        # both are within 2^-8 |result| + (2^-8 + small) of the weighted values, |v| < 6 here, of the same number
        assert float((out[b] - alone[0]).abs().max()) < 4 * 2.0**-8 * 6


@pytest.mark.parametrize("int8", [False, True])
def test_replays_see_what_the_step_before_them_wrote(int8):
    """queries, tables and lengths written by the kernels right before the call, others at each replay"""
    from wf_bitnet import ops
    q, kv, layer, pt, prefix, table, lens = case(24, 8, 2, 900, [16 * (b % 20 + 1) for b in range(24)], 16, int8, 8)
    order = [torch.randperm(24, device="cuda") for _ in range(6)]
    turned = [pt[torch.arange(pt.numel() - 1, device="cuda").roll(i)] for i in range(6)]     # (the last page is not full)
    src = [(q[o].contiguous(), torch.cat([t, pt[-1:]]), table[o].contiguous(), lens[o].contiguous()) for o, t in zip(order, turned)]
    want = [ops.paged_prefix_attn(a, kv, layer, b, prefix, c, d) for a, b, c, d in src]
    held = [t.clone() for t in src[0]]
    feed = [t.clone() for t in src[0]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for h, f in zip(held, feed):
            h.copy_(f)
        out = ops.paged_prefix_attn(held[0], kv, layer, held[1], prefix, held[2], held[3])
    for _ in range(3):
        for s, w in zip(src, want):
            for f, t in zip(feed, s):
                f.copy_(t)
            graph.replay()
            assert torch.equal(out, w)


def test_one_serving_step_after_another():
    """plan -> cache -> attention behind the prefix -> logits -> log probabilities, the same as with everything computed in 64 bits; pages go back at the end"""
    from wf_bitnet import ops
    g = torch.Generator(device="cuda").manual_seed(7)
    B, H, Hkv, page, prefix, V = 5, 8, 2, 16, 45, 515
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    kv = ops.PagedKV(40, 1, Hkv, page, D)
    kv.pool.fill_(math.nan)
    free, count = torch.arange(40, dtype=torch.int32, device="cuda"), i32([40])
    # the prefix is one sequence, planned and cached once
    ptable = torch.full((1, 3), -1, dtype=torch.int32, device="cuda")
    p = ops.paged_plan(i32([0]), i32([prefix]), ptable, free, count, page, prefix + 3)
    pk, pv = randn(prefix + 3, Hkv * D), randn(prefix + 3, Hkv * D)
    ops.kv_scatter(kv, pk, pv, p.pages, p.slots, 0)
    count = p.free_count
    table, lens = torch.full((B, 4), -1, dtype=torch.int32, device="cuda"), i32([0] * B)
    keys, vals = [pk[:prefix].view(prefix, Hkv, D)] * B, [pv[:prefix].view(prefix, Hkv, D)] * B
    E, E64 = randn(V, H * D), None
    for new in ([3, 20, 1, 17, 1], [1, 1, 1, 1, 0], [1, 1, 1, 1, 1]):
        p = ops.paged_plan(lens, i32(new), table, free, count, page, 50)
        assert int(p.status) == 0
        k, v = randn(50, Hkv * D), randn(50, Hkv * D)
        ops.kv_scatter(kv, k, v, p.pages, p.slots, 0)
        lens, count = p.lens, p.free_count
        off = p.offsets.tolist()
        for b in range(B):
            keys[b] = torch.cat([keys[b], k[off[b]:off[b + 1]].view(-1, Hkv, D)])
            vals[b] = torch.cat([vals[b], v[off[b]:off[b + 1]].view(-1, Hkv, D)])
        q = randn(B, H, D)
        out = ops.paged_prefix_attn(q, kv, 0, ptable[0], prefix, table, lens)
        for b in range(B):
            for h in range(H):
                w = torch.softmax(keys[b][:, h // 4].to(F64) @ q[b, h].to(F64) / math.sqrt(D), 0)
                want, mag = w @ vals[b][:, h // 4].to(F64), w @ vals[b][:, h // 4].to(F64).abs()
                assert bool(((out[b, h].to(F64) - want).abs() <= 2.0**-8 * want.abs() + (2.0**-8 + 2.0**-12) * mag).all())
        nxt, logits = ops.lm_head_argmax(out.view(B, -1), E)
        lp, ent, tlp, tid = ops.token_logprobs(logits, nxt, 3)
        ref = torch.log_softmax(logits.to(F64), -1)
        assert torch.equal(tid[:, 0], nxt) and bool(((lp.to(F64) - ref.amax(-1)).abs() < 1e-5).all()) and torch.equal(lp, tlp[:, 0])
        assert bool(((ent.to(F64) + (ref * ref.exp()).sum(-1)).abs() < 1e-5).all())
    held = int((-(-lens // page)).sum())
    lens, count2 = ops.paged_release(torch.ones(B, dtype=torch.bool, device="cuda"), lens, table, free, count, page)
    assert int(count2) == int(count) + held == 40 - 3 and not lens.any()
    assert sorted(free[:37].tolist() + ptable[0].tolist()) == list(range(40))


def test_the_same_through_ctypes(monkeypatch):
    from wf_bitnet import _native, ops
    c = case(3, 8, 2, 200, [3, 1, 30], 16, False)
    g = torch.Generator(device="cuda").manual_seed(3)
    x, tok = torch.randn(4, 999, generator=g, device="cuda")[:, 2:], torch.tensor([1, 2, 3, 4], dtype=torch.int32, device="cuda")
    lens, new, count = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([3, 30, 0], [1, 5, 2], [6]))
    done = torch.tensor([True, False, True], device="cuda")

    def results():
        table, free = torch.arange(9, dtype=torch.int32, device="cuda").view(3, 3), torch.arange(10, 20, dtype=torch.int32, device="cuda")
        return [ops.paged_prefix_attn(*c), *ops.token_logprobs(x, tok, 5, 0.5), *ops.paged_plan(lens, new, table, free, count, 16, 11), table,
                *ops.paged_release(done, lens, table, free, count, 16), free]
    a = results()
    monkeypatch.setattr(_native, "_ops", _native._Ctypes)
    b = results()
    assert len(a) == len(b) and all(u.dtype == v.dtype and torch.equal(u, v) for u, v in zip(a, b))
    for bad in (lambda: ops.token_logprobs(x, tok.long()), lambda: ops.paged_prefix_attn(c[0], c[1], 5, *c[3:]), lambda: ops.paged_plan(lens, new[:2], lens.view(3, 1), lens, count, 16, 4),
                lambda: ops.paged_release(lens, lens, lens.view(3, 1), lens, count, 16), lambda: ops.paged_plan(lens, new, lens.view(3, 1).cpu(), lens, count, 16, 4)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("int8", [False, True])
def test_tables_far_wider_than_the_sequences(int8):
    """sequences are cut by their own lengths, whatever the table has room for"""
    q, kv, layer, pt, prefix, table, lens = case(3, 8, 2, 300, [30, 0, 290], 16, int8)
    wide = torch.zeros(3, 5000, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    check(q, kv, layer, pt, prefix, wide, lens)
