"""Keys and values that are handed to the cache as parts of wider rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.int8])
def test_scatter_of_parts_of_rows(dtype):
    from wf_bitnet import ops
    g = torch.Generator(device="cuda").manual_seed(0)
    rows = torch.randn(9, 2, 256, generator=g, device="cuda").to(torch.bfloat16 if dtype == torch.int8 else dtype)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    pages, slots = i32([2, 0, 1, 1, 2, 0, 0, 2, 1]), i32(list(range(9)))
    a, b = (ops.PagedKV(3, 1, 2, 16, 128, dtype=dtype) for _ in range(2))
    ops.kv_scatter(a, rows[:, 0], rows[:, 1], pages, slots, 0)
    ops.kv_scatter(b, rows[:, 0].clone(), rows[:, 1].clone(), pages, slots, 0)
    assert torch.equal(a.pool, b.pool) and not torch.equal(a.pool[:, :, 0], a.pool[:, :, 1])
