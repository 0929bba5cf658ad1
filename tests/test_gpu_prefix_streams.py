"""Shared-prefix attention from several streams at a time: the same bits as alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("B, prefix", [(31, 16003), (64, 5000), (3, 700)])
def test_three_streams_at_a_time(B, prefix, int8):
    """up to 128 rows of a key/value head (two groups take every other tile) and more"""
    from test_gpu_prefix_attn import case

    from wf_bitnet import ops
    c = case(B, 32, 8, prefix, [(7 * b) % 90 for b in range(B)], 16, int8)
    want = ops.paged_prefix_attn(*c)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(60):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.paged_prefix_attn(*c))
        torch.cuda.synchronize()
        assert all(torch.equal(x, want) for x in got)
