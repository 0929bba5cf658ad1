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
