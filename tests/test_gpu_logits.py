"""Penalties, biases and grammar masks on logits against 64 bits, token by token."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F64 = torch.float64
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def used_memory():
    """what is allocated next has been written before, so that an entry that a kernel leaves out shows"""
    if torch.cuda.is_available():
        kept = [torch.full((n // 4,), float("nan"), device="cuda") for n in [1 << 28] + [1 << 19] * 64]
        del kept


def pack(ok):
    """bool [n, V] -> int32 words"""
    n, V = ok.shape
    x = np.zeros((n, -(-V // 32) * 32), np.uint8)
    x[:, :V] = ok
    return torch.from_numpy(np.packbits(x, axis=1, bitorder="little").view(np.int32).copy())


def case(rows, V, dtype, L=50, bias=5, masked=0.5, seed=0, nodes=False, tail=0, hot=None):
    """rows: how many each sequence has; tokens of the history often the same"""
    rng = np.random.default_rng(seed)
    B, N = len(rows), sum(rows) + tail
    hot = hot or max(1, min(V, 12))
    some = lambda *s: np.where(rng.random(s) < 0.7, rng.integers(0, hot, s), rng.integers(0, V, s)).astype(np.int32)  # noqa: E731
    a = {"logits": torch.from_numpy(rng.standard_normal((N, V)).astype(np.float32) * 3).to(dtype).cuda()}
    i32 = lambda x: torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()  # noqa: E731
    f32 = lambda x: torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).cuda()  # noqa: E731
    if L:
        lens = rng.integers(0, L + 1, B)
        a.update(history=i32(some(B, L)), history_lens=i32(lens), prompt_lens=i32((lens * rng.random(B)).astype(int)))
    a.update(repetition=f32(1 + rng.random(B)), frequency=f32(rng.random(B)), presence=f32(rng.random(B) - 0.3))
    if bias:
        a.update(bias_ids=i32(some(B, bias)), bias_values=f32(rng.standard_normal((B, bias)) * 5))
    if masked:
        a["allowed"] = pack((rng.random((N, 1)) > masked) | (rng.random((N, V)) < 0.1)).cuda()
    if nodes or any(r != 1 for r in rows) or tail:
        a["offsets"] = i32(np.concatenate([[0], np.cumsum(rows)]))
    if nodes:
        w = -(-max(rows) // 64)
        bits = rng.random((N, w * 64)) < 0.3
        for b in range(B):
            o = int(a["offsets"][b])
            bits[o:o + rows[b], rows[b]:] = False
        a["node_mask"] = torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int64).copy()).cuda()
        a["node_tokens"] = i32(some(N))
    return a


def want_of(a):
    """(result, the largest number on the way) in 64 bits"""
    x = a["logits"].to(F64).cpu().numpy().copy()
    N, V = x.shape
    off = a["offsets"].tolist() if "offsets" in a else list(range(N + 1))
    B = len(off) - 1
    get = lambda k: a[k].cpu().numpy() if a.get(k) is not None else None  # noqa: E731
    hist, hl, pl, rep, freq, pres = (get(k) for k in ("history", "history_lens", "prompt_lens", "repetition", "frequency", "presence"))
    bi, bv, ok, nt, nm = (get(k) for k in ("bias_ids", "bias_values", "allowed", "node_tokens", "node_mask"))
    big = np.abs(x)
    for b in range(B):
        h = hist[b, :hl[b] if hl is not None else None] if hist is not None else np.zeros(0, np.int32)
        p = pl[b] if pl is not None else 0
        for n in range(off[b], off[b + 1]):
            drawn = list(h[max(p, 0):])
            if nm is not None:
                bits = np.unpackbits(nm[n].view(np.uint8), bitorder="little")
                drawn += [nt[off[b] + j] for j in np.flatnonzero(bits) if off[b] + j < N]
            count = {}
            for t in drawn:
                count[int(t)] = count.get(int(t), 0) + 1
            with np.errstate(over="ignore", invalid="ignore"):
                for t in set(int(t) for t in h) | set(count):
                    if not 0 <= t < V:
                        continue
                    r = float(rep[b]) if rep is not None else 1.0
                    x[n, t] = x[n, t] / r if x[n, t] > 0 else x[n, t] * r
                    big[n, t] = np.fmax(big[n, t], np.abs(x[n, t]))
                    if t in count:
                        off_by = (float(freq[b]) if freq is not None else 0.0) * count[t] + (float(pres[b]) if pres is not None else 0.0)
                        x[n, t] -= off_by
                        big[n, t] += abs(off_by) + (float(freq[b]) * count[t] if freq is not None else 0.0)
                if bi is not None:
                    for t, v in dict(zip(bi[b].tolist(), bv[b].tolist())).items():
                        if 0 <= t < V:
                            x[n, t] += v
                            big[n, t] += abs(v)
            if ok is not None:
                allowed = np.unpackbits(ok[n].view(np.uint8), bitorder="little")[:V].astype(bool)
                x[n, ~allowed] = -math.inf
    return torch.from_numpy(x).cuda(), torch.from_numpy(big).cuda()


def agree(out, a):
    """a rounding to the type at the end (half a step), and a quotient or product, a product, two sums and a bias in float: six half steps 2^-24 of the largest number on the way"""
    want, big = want_of(a)
    half = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}[out.dtype]
    got = out.to(F64)
    most = torch.finfo(out.dtype).max
    tiny = torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps / 2
    same = (got == want) | (got.isnan() & want.isnan()) | ((want.abs() > most) & (got == want.sign() * math.inf))
    with_tol = (got - want).abs() <= half * want.abs() * 1.001 + 8 * 2.0**-24 * big + tiny
    return bool((same | with_tol).all())


def check(a, **more):
    from wf_bitnet import ops
    before = a["logits"].clone()
    out = ops.process_logits(**a, **more)
    assert out.dtype == a["logits"].dtype and agree(out, a)
    assert torch.equal(a["logits"].view(torch.int16 if before.dtype != torch.float32 else torch.int32), before.view(torch.int16 if before.dtype != torch.float32 else torch.int32))
    mine = a["logits"].clone()
    res = ops.process_logits(**{**a, "logits": mine}, out=mine)
    assert res is mine and torch.equal(mine.nan_to_num(7.0), out.nan_to_num(7.0))
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 2, 31, 32, 33, 100, 511, 512, 513, 4095, 4096, 4099, 32003, 128256])
def test_vocabularies(V, dtype):
    check(case([1] * 3, V, dtype, seed=V))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [[1], [2, 0, 3], [5] * 4, [9, 70, 1], [64] * 3, [256, 200]])
@pytest.mark.parametrize("nodes", [False, True])
def test_rows_of_sequences(rows, nodes, dtype):
    a = case(rows, 1003, dtype, nodes=nodes, tail=2, seed=sum(rows))
    out = check(a)
    end = sum(rows)
    assert torch.equal(out[end:], a["logits"][end:])


@pytest.mark.parametrize("dtype", TYPES)
def test_each_part_alone(dtype):
    from wf_bitnet import ops
    a = case([1] * 4, 777, dtype)
    keep = lambda *k: {x: a[x] for x in ("logits",) + k}  # noqa: E731
    assert torch.equal(ops.process_logits(a["logits"]), a["logits"])
    for part in (("history", "repetition"), ("history", "history_lens", "repetition"), ("history", "frequency"), ("history", "history_lens", "prompt_lens", "presence"),
                 ("bias_ids", "bias_values"), ("allowed",), ("repetition", "frequency", "presence"), ("history", "history_lens", "prompt_lens"), ("allowed", "bias_ids", "bias_values")):
        check(keep(*part))


@pytest.mark.parametrize("L", [1, 2, 255, 256, 257, 5000])
def test_histories(L):
    check(case([1, 1, 1], 3001, torch.float32, L=L, seed=L))


def test_a_token_drawn_thousands_of_times():
    a = case([1, 1], 50, torch.float32, L=20000, bias=0, masked=0)
    a["history"][:] = 7
    a["history_lens"][:] = 20000
    check(a)


def test_biases_of_the_same_token_the_last_one_counts():
    from wf_bitnet import ops
    a = {"logits": torch.zeros(1, 40, device="cuda"), "bias_ids": torch.tensor([[5, 7, 5, 50, -1, 5]], dtype=torch.int32, device="cuda"),
         "bias_values": torch.tensor([[1.0, 2, 3, 4, 5, 6]], device="cuda")}
    out = ops.process_logits(**a)
    assert out[0, 5] == 6 and out[0, 7] == 2 and out.count_nonzero() == 2
    check(case([1, 2], 33, torch.float32, bias=300))


def test_ids_outside_the_vocabulary_are_none():
    a = case([1, 1], 64, torch.float32, masked=0)
    a["history"][:, ::3] = -1
    a["history"][:, 1::7] = 64
    a["history"][:, 2::5] = 2**31 - 1
    a["bias_ids"][:, 0] = -2**31
    a["history_lens"][0] = 1000                          # beyond the width: the width
    a["prompt_lens"][1] = -5
    a["history_lens"] = a["history_lens"].clamp(max=50)
    check(a)


@pytest.mark.parametrize("dtype", TYPES)
def test_infinite_and_lowest_logits(dtype):
    """-inf stays -inf, the lowest number times a penalty becomes -inf, +inf and NaN stay; masked places are -inf whatever stood there"""
    a = case([1] * 3, 200, dtype, bias=3, seed=5, hot=40)
    low = torch.finfo(dtype).min
    a["logits"][:, 0:40:4], a["logits"][:, 1:40:4], a["logits"][:, 2:40:8], a["logits"][:, 6:40:8] = -math.inf, low, math.inf, math.nan
    out = check(a)
    assert out.isnan().any()
    a["allowed"][:] = 0
    assert (check(a) == -math.inf).all()


def test_rows_of_wider_tensors_and_off_alignment():
    from wf_bitnet import ops
    for dtype in TYPES:
        a = case([3, 2], 517, dtype, nodes=True)
        want = check(a)
        for lead in (1, 3, 4, 8):
            wide = torch.randn(5, 517 + 20, device="cuda").to(dtype)
            wide[:, lead:lead + 517] = a["logits"]
            side = torch.zeros(5, 517 + 31, device="cuda", dtype=dtype)
            x = wide[:, lead:lead + 517]
            assert torch.equal(ops.process_logits(**{**a, "logits": x}), want)
            y = side[:, 2:519]
            assert ops.process_logits(**{**a, "logits": x}, out=y) is y and torch.equal(y, want) and not side[:, :2].any() and not side[:, 519:].any()
            kept = wide.clone()
            ops.process_logits(**{**a, "logits": x}, out=x)
            kept[:, lead:lead + 517] = want
            assert torch.equal(wide, kept)
        assert torch.equal(ops.process_logits(**{**a, "logits": a["logits"].T.contiguous().T}), want)


def test_the_same_bits_every_time():
    from wf_bitnet import ops
    a = case([60] * 5, 32003, torch.bfloat16, L=3000, bias=40, nodes=True)
    want = ops.process_logits(**a)
    for _ in range(5):
        assert torch.equal(ops.process_logits(**a), want)


def test_a_captured_call():
    from wf_bitnet import ops
    a = case([4, 5], 2000, torch.bfloat16, nodes=True)
    ops.process_logits(**a)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.process_logits(**a)
    for seed in (3, 4):
        for k, v in case([4, 5], 2000, torch.bfloat16, nodes=True, seed=seed).items():
            a[k].copy_(v)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.process_logits(**a))


def test_refusals():
    from wf_bitnet import ops
    a = case([2, 3], 100, torch.float32, nodes=True)
    for key, bad in (("logits", a["logits"].double()), ("logits", a["logits"][0]), ("history", a["history"].long()), ("history", a["history"][:1]), ("history_lens", a["history_lens"].float()),
                     ("prompt_lens", a["prompt_lens"][:1]), ("repetition", a["repetition"].double()), ("frequency", a["frequency"].cpu()), ("presence", a["presence"][None]),
                     ("bias_values", a["bias_values"][:, :-1]), ("bias_values", None), ("allowed", a["allowed"][:, :-1]), ("allowed", a["allowed"][:-1]), ("offsets", a["offsets"][:0]),
                     ("offsets", a["offsets"].long()), ("offsets", None), ("node_tokens", None), ("node_tokens", a["node_tokens"][:-1]), ("node_mask", a["node_mask"].int()),
                     ("out", a["logits"].bfloat16()), ("out", a["logits"][:, :1].expand(-1, 100)), ("out", torch.empty(100, 5, device="cuda").T)):
        with pytest.raises(ValueError):
            ops.process_logits(**{**a, key: bad})
    with pytest.raises(NotImplementedError):
        ops.process_logits(**{**a, "node_mask": torch.zeros(5, 5, dtype=torch.int64, device="cuda")})
    assert ops.process_logits(a["logits"][:0]).shape == (0, 100)


def test_out_between_the_rows_and_over_them():
    from wf_bitnet import ops
    x = torch.randn(5, 2000, device="cuda")
    bias = dict(bias_ids=torch.full((5, 1), 7, dtype=torch.int32, device="cuda"), bias_values=torch.ones(5, 1, device="cuda"))
    want = ops.process_logits(x[:, :1000], **bias)
    ops.process_logits(x[:, :1000], out=x[:, 1000:], **bias)
    assert torch.equal(x[:, 1000:], want)
    for out in (x[:, 1:1001], x[:, 999:1999]):
        with pytest.raises(ValueError):
            ops.process_logits(x[:, :1000], out=out, **bias)
    y = x.view(10, 1000)
    with pytest.raises(ValueError):
        ops.process_logits(y[:9], out=y[1:], bias_ids=bias["bias_ids"].repeat(2, 1)[:9], bias_values=bias["bias_values"].repeat(2, 1)[:9])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [513, 1500, 9000, 32003, 32700, 70001])
@pytest.mark.parametrize("rows", [[60] * 5, [1] * 40, [200, 3, 90]])
def test_every_entry_is_written(rows, V, dtype):
    """vocabularies whose last chunk is short, with rows enough for the longer chunks"""
    from wf_bitnet import ops
    a = case(rows, V, dtype, L=300, bias=9, nodes=len(set(rows)) > 1, tail=1 if len(rows) == 3 else 0)
    mine = a["logits"].clone()
    ops.process_logits(**{**a, "logits": mine}, out=mine)
    out = ops.process_logits(**a, out=torch.full_like(mine, math.nan))
    assert torch.equal(out, mine)
