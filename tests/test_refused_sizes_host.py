"""Workspace of shared-prefix attention: none for the sizes that the call refuses, right up to those that it takes."""
from wf_bitnet import _lib


def test_no_workspace_for_what_is_refused():
    need = _lib.lib().wf_prefix_attn_workspace_bytes
    assert need(2, 8, 2, 16, (1 << 30) + 1) == need(2, 8, 2, 0, (1 << 31) - 1) == 0
    assert need(1 << 22, 8, 2, 0, 40) == need((1 << 24) + 1, 1, 1, 16, 0) == 0
    assert need(65536, 1, 1, 16, 40) == 0 and need(65536, 1, 1, 0, 40) > 0 and need(65535, 1, 1, 16, 40) > 0
    assert need(2, 8, 2, 16, 1 << 30) > 0
