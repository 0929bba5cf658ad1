"""Keys whose score is -inf have no weight in paged decode attention either: alone, as the own part behind a shared prefix, and whatever warp and chunk they fall in."""
import math

import pytest
import torch

from test_gpu_prefix_attn import D, F64, case, rows_of

pytestmark = pytest.mark.gpu


def without(kv, layer, pages, head, which, keep):
    return rows_of(kv, pages, layer, which, head, len(keep))[keep]


def sink(kv, layer, page, slots, head, int8):
    """keys of -inf scores for positive queries: -inf itself, or the lowest code with a scale of +inf"""
    if int8:
        kv.pool[page, layer, 0, head, slots] = 1
        kv.scales[page, layer, 0, head, slots] = math.inf
    else:
        kv.pool[page, layer, 0, head, slots] = -math.inf


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("prefix", [0, 300])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B, lens, dead", [(4, [1, 16, 40, 90], [range(1), range(16), range(16), range(16)]),          # all that a warp sees, or its first block
                                           (4, [33, 70, 200, 5], [range(32, 33), range(64), range(16, 128), [0, 2]]),   # a last block, whole rounds of all warps, single keys
                                           (2, [5000, 700], [range(1024), range(16, 700)])])                            # whole chunks
def test_keys_of_minus_infinity(B, lens, dead, out_dtype, prefix, int8):
    from wf_bitnet import ops
    q, kv, layer, pt, prefix, table, lens_t = case(B, 8, 2, prefix, lens, 16, int8, 3)
    q = q.abs() + 0.1
    for b in range(B):
        for j in dead[b]:
            sink(kv, layer, table[b][j // 16].long(), j % 16, 1, int8)
    out = ops.paged_prefix_attn(q, kv, layer, pt, prefix, table, lens_t, out_dtype=out_dtype)
    outs = [out] if prefix else [out, ops.paged_decode_attn(q, kv, layer, table, lens_t, out_dtype=out_dtype)]
    for b in range(B):
        keep = torch.ones(lens[b], dtype=torch.bool, device="cuda")
        keep[list(dead[b])] = False
        for h in range(2):
            live = keep if h == 1 else torch.ones_like(keep)
            k = torch.cat([rows_of(kv, pt, layer, 0, h, prefix), rows_of(kv, table[b], layer, 0, h, lens[b])[live]])
            v = torch.cat([rows_of(kv, pt, layer, 1, h, prefix), rows_of(kv, table[b], layer, 1, h, lens[b])[live]])
            for o in outs:
                got = o[b, h * 4:h * 4 + 4].to(F64)
                if k.shape[0] == 0:                       # no key with a weight: zeros, as with no key at all
                    assert not got.any()
                    continue
                qh = q[b, h * 4:h * 4 + 4].to(F64)
                p = torch.softmax(qh @ k.T / math.sqrt(D), -1)
                want, mag = p @ v, p @ v.abs()
                # the bound of test_gpu_prefix_attn.check: weights of 16 bits, 2^x off by 2^-13 in weight and sum, float sums, one rounding of the result
                off = 2 * 130 * 2.0**-24 * float((qh.abs() @ k.abs().T).max()) / math.sqrt(D) + 2.0**-12 + 2 * k.shape[0] * 2.0**-23
                tol = (2.0**-8 if out_dtype == torch.bfloat16 else 2.0**-24) * want.abs() + (2.0**-8 + off) * mag
                assert bool(((got - want).abs() <= tol * 1.01).all()), (b, h, ((got - want).abs() - tol).max())


@pytest.mark.parametrize("int8", [False, True])
def test_a_key_of_nan_still_shows(int8):
    """in the own part, behind a prefix: its rows are NaN, the others as they were"""
    from wf_bitnet import ops
    q, kv, layer, pt, prefix, table, lens = case(2, 4, 2, 400, [1, 60], 16, int8)
    clean = ops.paged_prefix_attn(q, kv, layer, pt, prefix, table, lens)
    for b, j in ((0, 0), (1, 37)):
        at = (table[b][j // 16].long(), layer, 0, 1, j % 16)
        if int8:
            kv.scales[at] = math.nan
        else:
            kv.pool[at] = math.nan
    out = ops.paged_prefix_attn(q, kv, layer, pt, prefix, table, lens)
    assert out[:, 2:].isnan().all() and torch.equal(out[:, :2], clean[:, :2])
