"""Log probabilities, entropy and alternatives against softmax in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F64 = torch.float64
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24                                           # half a step of float, relative


def reference(x, tokens, top, temperature=1.0):
    """(logprobs, entropy, top logprobs, top ids, the mean distance to the largest logit) in 64 bits; x on the GPU, NaN-free, no +inf"""
    z = x.to(F64) / temperature
    empty = torch.isneginf(z).all(-1)
    z0 = torch.where(empty[:, None], 0.0, z)
    logp = torch.where(empty[:, None], -math.inf, torch.log_softmax(z0, -1))
    p = torch.where(empty[:, None], 0.0, torch.softmax(z0, -1))
    entropy = -torch.xlogy(p, p).sum(-1)
    ids = torch.sort(x.to(F64) + 0.0, dim=-1, descending=True, stable=True).indices[:, :top]
    far = (p * torch.where(p > 0, z0.amax(-1, keepdim=True) - z0, 0.0)).sum(-1)
    return logp.gather(1, tokens.long()[:, None])[:, 0], entropy, logp.gather(1, ids), ids.to(torch.int32), far


def check(x, tokens, top, temperature=1.0):
    """Tolerances, each rounding half a step: a = (x - m) c has three; 2^a is off by |a| times that and by 2^-22 of its own (ex2.approx); a thread adds up to
    V / 512 + 32 of them and 9 + 4 + 3 joins follow, so log2 s is off by at most (V / 512 + 80) half steps and what the exponents' errors weigh, 4 half steps of
    the mean distance `far`; log p adds 4 half steps of |log p|; the entropy divides t, summed the same way, by s: (1 + far) times the above."""
    from wf_bitnet import ops
    lp, ent, tlp, tid = ops.token_logprobs(x, tokens, top, temperature)
    rlp, rent, rtlp, rtid, far = reference(x, tokens, top, temperature)
    assert tid.dtype == torch.int32 and torch.equal(tid, rtid)
    sums = (x.shape[1] / 512 + 80) * U + 4 * U * far
    for got, want, tol in ((lp, rlp, sums + 4 * U * rlp.abs()), (ent, rent, 2 * sums * (1 + far) + 4 * U * rent), (tlp, rtlp, sums[:, None] + 4 * U * rtlp.abs())):
        assert got.dtype == torch.float32 and got.shape == want.shape
        inf = torch.isinf(want)
        assert torch.equal(got.to(F64)[inf], want[inf])
        err = (got.to(F64) - want).abs()
        assert bool((err[~inf] <= tol.expand_as(want)[~inf]).all()), (err - tol)[~inf].max()


def rows(n, v, dtype, seed, scale=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(n, v, generator=g, device="cuda") * scale).to(dtype), torch.randint(0, v, (n,), generator=g, device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, v, top", [(1, 1, 1), (2, 3, 0), (5, 7, 7), (1, 64, 64), (3, 129, 33), (33, 1000, 20), (1, 32003, 5), (4, 32768, 64), (1, 128256, 20), (2, 128256, 0), (149, 50001, 32),
                                       (300, 8193, 1)])
def test_against_64_bits(dtype, n, v, top):
    check(*rows(n, v, dtype, n + v), top)


@pytest.mark.parametrize("n", [1, 18, 19, 36, 37, 73, 74, 75, 147, 148, 149, 300])
def test_every_number_of_blocks_a_row(n):
    check(*rows(n, 40000 + n, torch.float32, n), 3)


@pytest.mark.parametrize("temperature", [0.1, 0.7, 1.3, 50.0])
@pytest.mark.parametrize("dtype", TYPES)
def test_temperature(dtype, temperature):
    check(*rows(7, 5003, dtype, 9), 10, temperature)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [100, 32003, 128256])
def test_ties_go_to_the_lowest_index(dtype, v):
    x, tok = rows(6, v, dtype, 3)
    x = (x * 2).round().to(dtype)                        # few different numbers
    x[0] = 1.5                                           # one number
    x[1] = torch.where(torch.arange(v, device="cuda") % 2 == 0, 0.0, -0.0).to(dtype)   # the same number, twice written
    x[2, -3:] = 50.0
    x[3, :2] = 50.0
    check(x, tok, 64)
    check(x, tok, 5)


@pytest.mark.parametrize("order", ["up", "down", "up in steps"])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_sorted_rows(order, top):
    """Every entry belongs to the largest so far: the longest way."""
    v = 60001
    x = torch.arange(v, device="cuda", dtype=torch.float32) / v * 9
    if order == "down":
        x = x.flip(0)
    if order == "up in steps":
        x = (x * 50).floor()
    check(x.expand(3, v), torch.tensor([0, v - 1, 777], dtype=torch.int32, device="cuda"), top)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("allowed", [0, 1, 2, 40, 5000])
def test_masked_vocabulary(dtype, allowed):
    """-inf has no probability; rows with fewer allowed tokens than alternatives, and one with none"""
    x, tok = rows(5, 32003, dtype, allowed)
    g = torch.Generator(device="cuda").manual_seed(1)
    for r in range(5):
        keep = torch.randperm(32003, generator=g, device="cuda")[:allowed]
        y = torch.full_like(x[r], -math.inf)
        y[keep] = x[r, keep]
        x[r] = y
        if allowed and r % 2:
            tok[r] = keep[0]
    check(x, tok, 20)


@pytest.mark.parametrize("dtype", TYPES)
def test_masks_of_the_types_lowest_value(dtype):
    low = torch.finfo(dtype).min
    x, tok = rows(5, 4099, dtype, 1)
    x[0] = low                                           # all of it: even
    x[1, 7:] = low
    x[2] = torch.where(torch.arange(4099, device="cuda") % 3 == 0, low, -math.inf).to(dtype)
    x[3, 5] = torch.finfo(dtype).max
    tok[1] = 3
    tok[2] = 9
    lowest = reference(x, tok, 4)
    assert abs(float(lowest[0][0]) + math.log(4099)) < 1e-9
    check(x[:3], tok[:3], 4)
    x[3, 6] = low                                        # a difference beyond float: no probability
    from wf_bitnet import ops
    lp, ent, tlp, tid = ops.token_logprobs(x, torch.full_like(tok, 5), 4)
    assert float(lp[3]) == 0 and float(ent[3]) == 0 and int(tid[3, 0]) == 5 and float(tlp[3, 0]) == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("at", [0, 1, 1234, 40002])
def test_nan_and_infinity_stay_in_their_row(dtype, bad, at):
    from wf_bitnet import ops
    x, tok = rows(4, 40003, dtype, 2)
    keep = [0, 2, 3]
    good = ops.token_logprobs(x, tok, 6)
    y = x.clone()
    y[1, at] = bad
    lp, ent, tlp, tid = ops.token_logprobs(y, tok, 6)
    for a, b in zip((lp, ent, tlp, tid), good):
        assert torch.equal(a[keep], b[keep])
    assert lp[1].isnan() and ent[1].isnan() and tlp[1].isnan().all()
    want = torch.where(y[1].isnan(), -math.inf, y[1]).sort(descending=True, stable=True).indices[:6]
    assert torch.equal(tid[1], want.to(torch.int32))
    y[1] = math.nan
    assert ops.token_logprobs(y, tok, 6)[3][1].tolist() == [-1] * 6


def test_tokens_outside_the_vocabulary_have_none():
    from wf_bitnet import ops
    x, tok = rows(5, 1000, torch.float32, 4)
    good = ops.token_logprobs(x, tok, 2)
    tok[1], tok[3] = -1, 1000
    lp, ent, tlp, tid = ops.token_logprobs(x, tok, 2)
    assert lp[[1, 3]].isnan().all() and torch.equal(lp[[0, 2, 4]], good[0][[0, 2, 4]])
    assert torch.equal(ent, good[1]) and torch.equal(tlp, good[2]) and torch.equal(tid, good[3])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [9, 1001, 32003])
def test_rows_of_a_larger_buffer_at_every_alignment(dtype, v):
    buf, _ = rows(6, v + 13, dtype, v)
    tok = torch.randint(0, v, (6,), device="cuda", dtype=torch.int32)
    for off in range(9):
        check(buf[:, off:off + v], tok, 5)
    check(buf[::2, 3:3 + v], tok[::2], 5)
    check(buf[:, :v].T.contiguous().T, tok, 5)           # columns apart: laid out first


def test_no_rows():
    from wf_bitnet import ops
    lp, ent, tlp, tid = ops.token_logprobs(torch.empty(0, 50, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), 3)
    assert lp.shape == ent.shape == (0,) and tlp.shape == tid.shape == (0, 3)


def test_offsets_beyond_31_bits():
    v, n = 128256, 17000                                 # 2.2e9 entries
    x = torch.zeros(n, v, dtype=torch.bfloat16, device="cuda")
    x[n - 1, v - 2] = 20.0
    from wf_bitnet import ops
    lp, ent, tlp, tid = ops.token_logprobs(x, torch.full((n,), v - 2, dtype=torch.int32, device="cuda"), 2)
    assert tid[n - 1].tolist() == [v - 2, 0] and tid[n - 2].tolist() == [0, 1]
    want = 20.0 - math.log(math.exp(20.0) + v - 1)
    assert abs(float(lp[n - 1]) - want) < 1e-5 and abs(float(lp[0]) + math.log(v)) < 1e-5


def test_wrong_arguments_are_refused():
    from wf_bitnet import ops
    x, tok = rows(3, 100, torch.float32, 1)
    for a in ((x[0], tok, 0), (x, tok.long(), 0), (x, tok[:2], 0), (x, tok, -1), (x, tok, 101), (x.to(F64), tok, 0), (x, tok.cpu(), 0), (x, tok, 0, 0.0), (x, tok, 0, -1.0), (x, tok, 0, math.nan),
              (x, tok, 0, 1e-45), (torch.empty(2, 0, device="cuda"), tok[:2], 0)):
        with pytest.raises(ValueError):
            ops.token_logprobs(*a)
    with pytest.raises(NotImplementedError):
        ops.token_logprobs(x, tok, 65)


def test_another_stream_and_a_replayed_graph():
    from wf_bitnet import ops
    x, tok = rows(9, 70001, torch.bfloat16, 8)
    want = ops.token_logprobs(x, tok, 20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.token_logprobs(x, tok, 20)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    y, t = torch.zeros_like(x), torch.zeros_like(tok)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.token_logprobs(y, t, 20)
    y.copy_(x), t.copy_(tok)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
