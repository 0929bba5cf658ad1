"""Keys of the prefix whose score is -inf have no weight, however large their values are."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
D = 128


@pytest.mark.parametrize("prefix", [64, 200, 1000])
def test_the_largest_values_under_keys_without_weight(prefix):
    from wf_bitnet import ops
    g = torch.Generator(device="cuda").manual_seed(0)
    kv = ops.PagedKV(prefix // 16 + 2, 1, 1, 16, D)
    kv.pool.copy_(torch.randn(kv.pool.shape, generator=g, device="cuda"))
    table = torch.arange(prefix // 16 + 1, dtype=torch.int32, device="cuda")
    q = (torch.randn(3, 4, D, generator=g, device="cuda").abs() + 0.1).to(torch.bfloat16)
    own, lens = torch.zeros(3, 0, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    at = torch.arange(prefix, device="cuda")
    heard = at % 3 == 1
    k, v = (kv.pool[:, 0, w, 0].reshape(-1, D)[:prefix].clone() for w in (0, 1))
    k[~heard], v[~heard] = -math.inf, 3e38
    kv.pool[table.long()[at // 16], 0, 0, 0, at % 16], kv.pool[table.long()[at // 16], 0, 1, 0, at % 16] = k, v
    out = ops.paged_prefix_attn(q, kv, 0, table, prefix, own, lens).double()
    p = torch.softmax(q.double() @ k[heard].double().T / math.sqrt(D), -1)
    want, mag = p @ v[heard].double(), p @ v[heard].double().abs()
    # weights and result rounded to bf16 (half a step each), scores, exponentials and sums in float
    assert bool(((out - want).abs() <= 2.0**-8 * want.abs() + (2.0**-8 + 2.0**-11) * mag).all())
