"""Norm, rotation and append of a step's tokens against 64 bits, and against the cache's own scatter."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F64 = torch.float64


@pytest.fixture(autouse=True)
def used_memory():
    """what is allocated next has been written before, so that an entry that a kernel leaves out shows"""
    if torch.cuda.is_available():
        kept = [torch.full((n // 4,), float("nan"), device="cuda") for n in [1 << 28] + [1 << 19] * 64]
        del kept


def tables(max_pos, rot, dtype=torch.float32, base=10000.0):
    angle = torch.arange(max_pos, device="cuda", dtype=F64)[:, None] * base ** (-torch.arange(0, rot, 2, device="cuda", dtype=F64) / max(rot, 1))
    return torch.cos(angle).to(dtype), torch.sin(angle).to(dtype)


def case(T, H, Hkv, D, page, int8=False, rot=None, seed=0, layers=2, max_pos=500, table=torch.float32, gain=torch.bfloat16, norms=(True, True)):
    from wf_bitnet import ops
    g = torch.Generator(device="cuda").manual_seed(seed)
    blocks = -(-max(T, 1) // page)
    kv = ops.PagedKV(blocks + 2, layers, Hkv, page, D, dtype=torch.int8 if int8 else torch.bfloat16)
    if int8:
        kv.pool.copy_(torch.randint(0, 256, kv.pool.shape, generator=g, device="cuda", dtype=torch.uint8))
        kv.scales.fill_(0.5)
    else:
        kv.pool.copy_(torch.randn(kv.pool.shape, generator=g, device="cuda"))
    order = torch.randperm(blocks + 2, generator=g, device="cuda").to(torch.int32)
    k = torch.arange(T, device="cuda")
    cos, sin = tables(max_pos, D if rot is None else rot, table)
    gains = [(torch.rand(D, generator=g, device="cuda") + 0.5).to(gain) if n else None for n in norms]
    return dict(qkv=(torch.randn(T, (H + 2 * Hkv) * D, generator=g, device="cuda") * 2).to(torch.bfloat16), H=H, kv=kv, layer=1,
                positions=torch.randint(0, max_pos, (T,), generator=g, device="cuda", dtype=torch.int32), pages=order[k // page].contiguous(), slots=(k % page).to(torch.int32), cos_tab=cos,
                sin_tab=sin, q_norm=gains[0], k_norm=gains[1])


def want_of(a, eps=1e-6, interleaved=False):
    """(queries, keys, values) in 64 bits, and of each entry the largest number in its pair"""
    kv, H = a["kv"], a["H"]
    D, Hkv, R = kv.head_dim, kv.kv_heads, 2 * a["cos_tab"].shape[1]
    x = a["qkv"].to(F64).reshape(-1, H + 2 * Hkv, D).clone()
    for sl, gain in ((slice(0, H), a["q_norm"]), (slice(H, H + Hkv), a["k_norm"])):
        if gain is not None:
            x[:, sl] *= gain.to(F64) / torch.sqrt(x[:, sl].square().mean(-1, keepdim=True) + eps)
    mag = x.abs()
    if R:
        cos, sin = (a[k].to(F64)[a["positions"].long()][:, None] for k in ("cos_tab", "sin_tab"))
        one, two = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
        qk = x[:, :H + Hkv]
        p, q = qk[..., one].clone(), qk[..., two].clone()
        qk[..., one], qk[..., two] = p * cos - q * sin, p * sin + q * cos
        m = p.abs() + q.abs()
        mag[:, :H + Hkv][..., one] = mag[:, :H + Hkv][..., two] = m
    return [t for t in (x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:])], [t for t in (mag[:, :H], mag[:, H:H + Hkv], mag[:, H + Hkv:])]


def near(got, want, mag):
    """one rounding to bf16 (half a step, 2^-8 of the value), and in float: 128 to 256 squares added (a sum over lanes of 8 in a row: at most 14 half steps on the sum, half of that on
    its root), the root 2 steps, the products of gain and rotation 6 more: below 32 half steps 2^-24 of what the pair has"""
    return bool(((got.to(F64) - want).abs() <= 2.0**-8 * want.abs() * 1.001 + 32 * 2.0**-24 * mag * 1.01).all())


def held(kv, layer, pages, slots):
    """[T, 2, Hkv, D] as the cache has it, in float"""
    x = kv.pool[pages.long(), layer, :, :, slots.long()]
    if kv.dtype == torch.int8:
        return (x.float() - 128) * kv.scales[pages.long(), layer, :, :, slots.long()][..., None]
    return x


def check(a, interleaved=False):
    from wf_bitnet import ops
    kv = a["kv"]
    before, scales = kv.pool.clone(), kv.scales.clone() if kv.dtype == torch.int8 else None
    q = ops.norm_rope_kv_append(**a, interleaved=interleaved)
    (wq, wk, wv), (mq, mk, _) = want_of(a, interleaved=interleaved)
    assert near(q, wq, mq)
    got = held(kv, a["layer"], a["pages"], a["slots"])
    if kv.dtype == torch.int8:
        # the codes are those that a scatter of the same bf16 rows writes
        for which, w, m in ((0, wk, mk), (1, wv, wv.abs())):
            top = (w.abs() + 2.0**-7 * m).amax(-1, keepdim=True)
            assert bool(((got[:, which].to(F64) - w).abs() <= top / 254 * 1.02 + 2.0**-7 * m).all())
        other = ops.PagedKV(kv.max_pages, kv.layers, kv.kv_heads, kv.page_size, kv.head_dim, dtype=torch.int8)
        other.pool.copy_(before)
        other.scales.copy_(scales)
        b = {**a, "kv": ops.PagedKV(kv.max_pages, kv.layers, kv.kv_heads, kv.page_size, kv.head_dim)}
        assert torch.equal(ops.norm_rope_kv_append(**b, interleaved=interleaved), q)
        rows = held(b["kv"], a["layer"], a["pages"], a["slots"])
        ops.kv_scatter(other, rows[:, 0].reshape(len(q), -1), rows[:, 1].reshape(len(q), -1), a["pages"], a["slots"], a["layer"])
        assert torch.equal(kv.pool, other.pool) and torch.equal(kv.scales, other.scales)
        return
    assert near(got[:, 0], wk, mk) and torch.equal(got[:, 1].to(F64), wv)
    before[a["pages"].long(), a["layer"], :, :, a["slots"].long()] = got
    assert torch.equal(before, kv.pool)                  # and nothing else is written


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("T", [1, 2, 31, 300, 5000])
@pytest.mark.parametrize("H, Hkv", [(1, 1), (20, 5), (32, 8), (7, 1)])
def test_tokens_and_heads(T, H, Hkv, int8):
    check(case(T, H, Hkv, 128, 16, int8, seed=T))


@pytest.mark.parametrize("D, rot", [(64, 64), (64, 16), (128, 128), (128, 96), (128, 64), (128, 8), (128, 0), (256, 256), (256, 80)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_sizes_of_head_and_rotation(D, rot, interleaved):
    check(case(77, 6, 3, D, 48, rot=rot, seed=rot), interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
def test_int8_interleaved(interleaved):
    check(case(77, 6, 3, 128, 48, True, rot=64), interleaved)


@pytest.mark.parametrize("table", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gain", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("norms", [(True, True), (True, False), (False, True), (False, False)])
def test_types_of_tables_and_gains(table, gain, norms):
    check(case(40, 4, 2, 128, 7, table=table, gain=gain, norms=norms))


def test_without_norms_as_rope_kv_append_up_to_its_roundings():
    from wf_bitnet import ops
    a = case(12, 8, 2, 128, 16, table=torch.bfloat16, norms=(False, False))
    q = ops.norm_rope_kv_append(**a)
    old = ops.PagedKV(a["kv"].max_pages, 2, 2, 16, 128)
    table = a["pages"][:, None].expand(-1, 500 // 16 + 1).contiguous()
    want = ops.rope_kv_append(a["qkv"], 8, old, 1, a["positions"], table, a["cos_tab"], a["sin_tab"])
    # there products and sum are rounded to bf16, too
    assert bool(((q.float() - want.float()).abs() <= 3 * 2.0**-8 * 12).all())


def test_tokens_without_a_place_and_positions_outside_the_table():
    from wf_bitnet import ops
    a = case(9, 4, 2, 128, 16)
    before = a["kv"].pool.clone()
    a["pages"][2], a["pages"][3], a["slots"][4], a["slots"][5] = -1, a["kv"].max_pages, 16, -1
    a["positions"][6], a["positions"][7] = -1, 500
    q = ops.norm_rope_kv_append(**a)
    live = [0, 1, 8]
    safe = {**a, "positions": a["positions"].clamp(0, 499)}
    (wq, wk, wv), (mq, mk, _) = want_of(safe)
    ok = torch.tensor([t not in (6, 7) for t in range(9)], device="cuda")
    assert near(q[ok], wq[ok], mq[ok]) and q[~ok].isnan().all()
    got = held(a["kv"], 1, a["pages"][live], a["slots"][live])
    assert near(got[:, 0], wk[live], mk[live])
    before[a["pages"][live].long(), 1, :, :, a["slots"][live].long()] = got
    assert torch.equal(before, a["kv"].pool)


def test_rows_of_zeros_and_of_nan():
    from wf_bitnet import ops
    a = case(6, 4, 2, 128, 16)
    a["qkv"][1] = 0
    a["qkv"][2, 130] = math.nan
    a["qkv"][3, 5 * 128 + 3] = math.inf
    q = ops.norm_rope_kv_append(**a)
    assert not q[1].any() and q[2, 1].isnan().all() and q[2, 0].isfinite().all() and q[2, 2:].isfinite().all() and q[3].isfinite().all()
    got = held(a["kv"], 1, a["pages"], a["slots"])
    assert got[2].isfinite().all() and not got[3, 0, 1].isfinite().all() and got[3, 1].isfinite().all()


def test_rows_of_a_wider_tensor_and_off_alignment():
    from wf_bitnet import ops
    a = case(20, 4, 2, 128, 16)
    want = ops.norm_rope_kv_append(**a)
    pool = a["kv"].pool.clone()
    wide = torch.randn(20, 1600, device="cuda").to(torch.bfloat16)
    wide[:, 64:64 + 1024] = a["qkv"]
    odd = torch.empty(20 * 1024 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(20, 1024)
    odd.copy_(a["qkv"])
    for x in (wide[:, 64:64 + 1024], odd, a["qkv"].T.contiguous().T, torch.stack([a["qkv"]] * 2, -1)[..., 0]):
        a["kv"].pool[a["pages"].long(), 1] = 0
        assert torch.equal(ops.norm_rope_kv_append(**{**a, "qkv": x}), want)
        assert torch.equal(held(a["kv"], 1, a["pages"], a["slots"]), pool[a["pages"].long(), 1, :, :, a["slots"].long()])


def test_pages_beyond_31_bits():
    from wf_bitnet import ops
    a = case(20, 8, 8, 128, 16)
    a["kv"] = ops.PagedKV(70000, 2, 8, 16, 128)          # 4.6e9 entries
    a["pages"] = a["pages"] + 69990
    q = ops.norm_rope_kv_append(**a)
    (wq, wk, wv), (mq, mk, _) = want_of(a)
    got = held(a["kv"], 1, a["pages"], a["slots"])
    assert near(q, wq, mq) and near(got[:, 0], wk, mk) and torch.equal(got[:, 1].to(F64), wv)


def test_refusals():
    from wf_bitnet import ops
    a = case(5, 4, 2, 128, 16)
    assert ops.norm_rope_kv_append(**{**a, "qkv": a["qkv"][:0], "positions": a["positions"][:0], "pages": a["pages"][:0], "slots": a["slots"][:0]}).shape == (0, 4, 128)
    for key, bad in (("qkv", a["qkv"].float()), ("qkv", a["qkv"][0]), ("qkv", a["qkv"][:, :-8]), ("H", 5), ("H", 0), ("layer", 2), ("layer", -1), ("positions", a["positions"].long()),
                     ("positions", a["positions"][:-1]), ("pages", a["pages"].cpu()), ("slots", a["slots"][None]), ("cos_tab", a["cos_tab"][:-1]), ("sin_tab", a["sin_tab"].bfloat16()),
                     ("cos_tab", a["cos_tab"][0]), ("q_norm", a["q_norm"][:-1]), ("k_norm", a["k_norm"].float()), ("eps", -1.0), ("eps", math.nan)):
        with pytest.raises(ValueError):
            ops.norm_rope_kv_append(**{**a, key: bad})
    with pytest.raises(ValueError):                      # float16 tables and gains
        ops.norm_rope_kv_append(**{**a, "cos_tab": a["cos_tab"].half(), "sin_tab": a["sin_tab"].half()})
    with pytest.raises(ValueError):
        ops.norm_rope_kv_append(**{**a, "q_norm": a["q_norm"].half(), "k_norm": a["k_norm"].half()})
    wide = torch.zeros(500, 70, device="cuda")
    with pytest.raises(ValueError):                      # more rotated dims than the head has
        ops.norm_rope_kv_append(**{**a, "cos_tab": wide, "sin_tab": wide})
    with pytest.raises(NotImplementedError):             # 12 rotated dims
        ops.norm_rope_kv_append(**{**a, "cos_tab": wide[:, :6].contiguous(), "sin_tab": wide[:, :6].contiguous()})
    with pytest.raises(NotImplementedError):
        b = case(5, 4, 2, 32, 16)
        ops.norm_rope_kv_append(**b)
    with pytest.raises(NotImplementedError):
        ops.norm_rope_kv_append(**{**a, "kv": ops.PagedKV(4, 2, 2, 16, 128, dtype=torch.float32)})


def test_a_captured_call():
    from wf_bitnet import ops
    a = case(64, 20, 5, 128, 16, True)
    ops.norm_rope_kv_append(**a)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q = ops.norm_rope_kv_append(**a)
    for seed in (1, 2):
        b = case(64, 20, 5, 128, 16, True, seed=seed)
        for k in ("qkv", "positions"):
            a[k].copy_(b[k])
        g.replay()
        torch.cuda.synchronize()
        pool = a["kv"].pool.clone()
        assert torch.equal(ops.norm_rope_kv_append(**a), q) and torch.equal(a["kv"].pool, pool)
