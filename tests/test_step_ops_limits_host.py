"""The largest sizes of the step operators, refused where an index of 32 bits would not hold what a loop adds to it; no GPU is reached."""
import ctypes as C

from wf_bitnet import _lib

BUF = (C.c_uint8 * 4096)()
P = (C.addressof(BUF) + 255) // 256 * 256                # never read: every call here ends at its checks


def test_more_pages_than_a_release_can_step_over():
    L = _lib.lib()

    def release(pool):
        return L.wf_paged_release(P, P, 8192, P, 262144, P, pool, P, 1, P, P, None)

    def plan(pool):
        return L.wf_paged_plan(P, P, 8192, P, 262144, P, pool, P, 1, 1 << 30, P, P, P, P, P, P, P, P, None)
    for call in (release, plan):
        for pool in ((1 << 30) + 1, (1 << 31) - 1):
            assert call(pool) == _lib.WF_ERR_UNSUPPORTED
            assert b"2^30" in L.wf_last_error()


def test_rows_of_a_block_table_end_where_a_page_can_be_asked_for_ahead():
    """a warp asks for pages up to 16 blocks of 16 tokens behind its own: such positions are below 2^31, too"""
    layout = _lib.KvLayout(P, 8, 1, 1, 16, 128, _lib.WF_BF16)

    def call(blocks):
        return _lib.lib().wf_paged_prefix_attn(P, C.byref(layout), 0, P, 40, P, blocks, P, 2, 8, 0.1, P, _lib.WF_BF16, P, 16, None)
    for blocks in ((1 << 27) - 1, (1 << 27) - 16, (1 << 27) - 255):
        assert call(blocks) == _lib.WF_ERR_UNSUPPORTED, blocks
    assert call((1 << 27) - 256) == _lib.WF_ERR_INVALID and b"workspace too small" in _lib.lib().wf_last_error()      # taken, up to its workspace
