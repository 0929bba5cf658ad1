"""The merge of shared-prefix attention at batches where a thread takes 4, 8 and 16 columns, with more parts of the prefix and more chunks of own keys than it asks for at
once: sequences of the batch's own result against softmax in 64 bits."""
import math

import pytest
import torch

from test_gpu_prefix_attn import D, F64, case, rows_of

pytestmark = pytest.mark.gpu


def check_rows(out, some, q, kv, layer, ptable, prefix, table, lens):
    """the bound of test_gpu_prefix_attn.check, on some sequences of a result"""
    G = q.shape[1] // kv.kv_heads
    for b in some:
        n = int(lens[b])
        for h in range(kv.kv_heads):
            k = torch.cat([rows_of(kv, ptable, layer, 0, h, prefix), rows_of(kv, table[b], layer, 0, h, n)])
            v = torch.cat([rows_of(kv, ptable, layer, 1, h, prefix), rows_of(kv, table[b], layer, 1, h, n)])
            qh = q[b, h * G:(h + 1) * G].to(F64)
            p = torch.softmax(qh @ k.T / math.sqrt(D), -1)
            want, mag = p @ v, p @ v.abs()
            off = 2 * 130 * 2.0**-24 * float((qh.abs() @ k.abs().T).max()) / math.sqrt(D) + 2.0**-12 + 2 * k.shape[0] * 2.0**-23
            tol = (2.0**-8 if out.dtype == torch.bfloat16 else 2.0**-24) * want.abs() + (2.0**-8 + off) * mag
            err = (out[b, h * G:(h + 1) * G].to(F64) - want).abs()
            assert bool((err <= tol * 1.01).all()), (b, h, (err - tol).max())


# columns a thread, then the batch: with tables this wide (tokens) the own part has 4 to 8 chunks a sequence at most, and the prefix 16, 13 and 6 parts
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("columns, B, H, Hkv, prefix, wide", [(4, 40, 32, 8, 8192, 65536), (8, 128, 20, 5, 8192, 32768), (8, 600, 4, 1, 1000, 65536), (16, 152, 32, 8, 4096, 131072),
                                                              (16, 1200, 4, 1, 1000, 65536)])
def test_columns_parts_and_chunks(columns, B, H, Hkv, prefix, wide, int8):
    from wf_bitnet import ops
    long = {0: 1300, 1: 257, 2: 0, 3: 513, B // 2: 770, B - 2: 16, B - 1: 1029}
    lens = [long.get(b, b % 23) for b in range(B)]
    q, kv, layer, pt, prefix, table, lens = case(B, H, Hkv, prefix, lens, 16, int8, columns, layers=1, layer=0)
    w = torch.zeros(B, wide // 16, dtype=torch.int32, device="cuda")
    w[:, :table.shape[1]] = table
    # own keys that matter as much as the prefix's, so that a part that is left out shows
    if not int8:
        for b in long:
            kv.pool[table[b].long(), 0, 0] *= 1.5
    for dtype in (torch.bfloat16, torch.float32):
        out = ops.paged_prefix_attn(q, kv, layer, pt, prefix, w, lens, out_dtype=dtype)
        check_rows(out, list(long), q, kv, layer, pt, prefix, w, lens)


@pytest.mark.parametrize("B, own", [(128, 120), (256, 300), (300, 40)])
def test_every_sequence_of_a_wide_batch(B, own):
    from wf_bitnet import ops
    c = case(B, 32, 8, 700, [(7 * b) % own for b in range(B)], 16, False, 6, layers=1, layer=0)
    check_rows(ops.paged_prefix_attn(*c), [0, 1, 2, B // 3, B // 2, B - 2, B - 1], *c)


@pytest.mark.parametrize("int8", [False, True])
def test_the_same_call_twice(int8):
    """nothing depends on the order in which blocks end"""
    from wf_bitnet import ops
    c = case(64, 20, 5, 3000, [(37 * b) % 600 for b in range(64)], 16, int8, 9)
    first = ops.paged_prefix_attn(*c)
    assert all(torch.equal(ops.paged_prefix_attn(*c), first) for _ in range(5))
