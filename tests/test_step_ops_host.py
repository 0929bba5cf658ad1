"""Refusals of the step operators (plans of pages and slots, shared-prefix attention, log probabilities) through the C ABI, their workspace size, and their torch ops'
registration: nothing here needs a GPU."""
import ctypes as C

import pytest
import torch

from wf_bitnet import _lib

BUF = (C.c_uint8 * 4096)()
P = (C.addressof(BUF) + 255) // 256 * 256                # 256-byte aligned host memory: never read, every call here ends at its checks


def test_plan_refusals():
    L = _lib.lib()

    def call(**k):
        a = dict(seq=P, new=P, rows=2, table=P, blocks=4, free=P, pool=8, count=P, page=16, cap=4, pos=P, tok=P, pages=P, slots=P, off=P, lens=P, cout=P, status=P)
        a.update(k)
        return L.wf_paged_plan(*a.values(), None)
    for bad in (dict(rows=-1), dict(blocks=-1), dict(pool=-1), dict(cap=-1), dict(page=0), dict(page=-16), dict(seq=None), dict(new=None), dict(table=None), dict(free=None), dict(count=None),
                dict(pos=None), dict(tok=None), dict(pages=None), dict(slots=None), dict(off=None), dict(lens=None), dict(cout=None), dict(status=None), dict(pos=P + 4), dict(slots=P + 8)):
        assert call(**bad) == _lib.WF_ERR_INVALID, bad
        assert b"wf_paged_plan" in L.wf_last_error()
    assert call(rows=8193) == call(cap=(1 << 30) + 1) == _lib.WF_ERR_UNSUPPORTED


def test_release_refusals():
    L = _lib.lib()

    def call(**k):
        a = dict(done=P, seq=P, rows=2, table=P, blocks=4, free=P, pool=8, count=P, page=16, lens=P, cout=P)
        a.update(k)
        return L.wf_paged_release(*a.values(), None)
    for bad in (dict(rows=-1), dict(blocks=-1), dict(pool=-1), dict(page=0), dict(done=None), dict(seq=None), dict(table=None), dict(free=None), dict(count=None), dict(lens=None), dict(cout=None)):
        assert call(**bad) == _lib.WF_ERR_INVALID, bad
        assert b"wf_paged_release" in L.wf_last_error()
    assert call(rows=8193) == _lib.WF_ERR_UNSUPPORTED


def test_prefix_attention_refusals():
    L = _lib.lib()

    def call(kv=(), **k):
        a = dict(q=P, kv=None, layer=0, pt=P, prefix=40, table=P, blocks=2, lens=P, B=2, H=8, scale=0.1, out=P, dt=_lib.WF_BF16, ws=P, ws_bytes=1 << 30)
        a.update(k)
        f = dict(pool=P, max_pages=8, layers=1, kv_heads=2, page_size=16, head_dim=128, dtype=_lib.WF_BF16)
        f.update(kv)
        layout = _lib.KvLayout(*f.values())
        a["kv"] = None if k.get("kv_null") else C.byref(layout)
        a.pop("kv_null", None)
        return L.wf_paged_prefix_attn(*a.values(), None)
    for bad in (dict(q=None), dict(pt=None), dict(table=None), dict(lens=None), dict(out=None), dict(ws=None), dict(ws_bytes=16), dict(prefix=-1), dict(blocks=-1), dict(B=-1), dict(H=0), dict(H=-2), dict(layer=1),
                dict(layer=-1), dict(dt=_lib.WF_F16), dict(q=P + 2), dict(out=P + 8), dict(ws=P + 8), dict(kv=dict(pool=None)), dict(kv=dict(pool=P + 2)), dict(kv=dict(kv_heads=0)), dict(kv_null=True)):
        assert call(**bad) == _lib.WF_ERR_INVALID, bad
        assert b"wf_paged_prefix_attn" in L.wf_last_error()
    for bad in (dict(kv=dict(head_dim=64)), dict(kv=dict(page_size=24)), dict(kv=dict(kv_heads=3)), dict(H=18), dict(kv=dict(dtype=_lib.WF_F32)), dict(prefix=(1 << 30) + 1),
                dict(blocks=1 << 27), dict(B=1 << 22)):
        assert call(**bad) == _lib.WF_ERR_UNSUPPORTED, bad
    assert call(B=0, q=None, out=None) == _lib.WF_OK


def test_more_sequences_than_a_grid_holds():
    layout = _lib.KvLayout(P, 8, 1, 1, 16, 128, _lib.WF_BF16)
    assert _lib.lib().wf_paged_prefix_attn(P, C.byref(layout), 0, P, 40, P, 2, P, 65536, 1, 0.1, P, _lib.WF_BF16, P, 1 << 60, None) == _lib.WF_ERR_UNSUPPORTED
    assert b"65535" in _lib.lib().wf_last_error()


def test_prefix_workspace_holds_both_parts():
    L = _lib.lib()
    assert L.wf_prefix_attn_workspace_bytes(0, 8, 2, 100, 100) == 0
    for B, H, Hkv in ((1, 1, 1), (33, 1, 1), (3, 20, 5), (128, 32, 8)):
        row = 130 * 4                                     # a row's partial result
        for seq in (16, 256, 257, 4096, 131072):
            own = L.wf_prefix_attn_workspace_bytes(B, H, Hkv, seq, 0)
            assert B * H * row * min(64, -(-seq // 256)) <= own <= L.wf_attn_workspace_bytes(B, H, 128, max(seq, 512))
        own = L.wf_prefix_attn_workspace_bytes(B, H, Hkv, 64, 0)
        for prefix in (1, 128, 5000, 1 << 20):
            both = L.wf_prefix_attn_workspace_bytes(B, H, Hkv, 64, prefix)
            assert both >= own + B * H * row and (both - own) % 256 == 0      # the own chunks start on a vector's boundary


def test_logprob_refusals():
    L = _lib.lib()

    def call(**k):
        a = dict(x=P, dt=_lib.WF_F32, rows=2, V=100, ld=100, tok=P, top=3, T=1.0, lp=P, ent=P, tlp=P, tid=P)
        a.update(k)
        return L.wf_token_logprobs(*a.values(), None)
    for bad in (dict(x=None), dict(tok=None), dict(lp=None), dict(ent=None), dict(tlp=None), dict(tid=None), dict(rows=-1), dict(V=0), dict(ld=99), dict(top=-1), dict(top=101), dict(T=0.0),
                dict(T=-1.0), dict(T=float("nan")), dict(T=float("inf")), dict(T=1e-45), dict(dt=_lib.WF_I8), dict(x=P + 2), dict(x=P + 1, dt=_lib.WF_BF16)):
        assert call(**bad) == _lib.WF_ERR_INVALID, bad
        assert b"wf_token_logprobs" in L.wf_last_error()
    assert call(top=65) == _lib.WF_ERR_UNSUPPORTED
    assert call(rows=0, x=None, tok=None, lp=None, ent=None, tlp=None, tid=None) == _lib.WF_OK


def test_logprobs_columns_beyond_their_index():
    # a block's indices run past the last column by a step: they are 32-bit
    rc = _lib.lib().wf_token_logprobs(P, _lib.WF_BF16, 1, (1 << 30) + 1, (1 << 30) + 1, P, 0, 1.0, P, P, None, None, None)
    assert rc == _lib.WF_ERR_UNSUPPORTED


def test_torch_ops_and_their_fakes():
    import sgl_kernel  # noqa: F401
    from wf_bitnet import _native
    if not _native.is_native():
        pytest.skip("no libwf_torch.so")
    ops = _native.ops()
    for name in ("paged_prefix_attn", "paged_plan", "paged_release", "token_logprobs"):
        assert "AutogradCUDA: fallthrough" in torch._C._dispatch_dump_table(f"wf_native::{name}")
        assert hasattr(_native._Ctypes, name)
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        i = lambda *s: torch.empty(*s, dtype=torch.int32, device="cuda")  # noqa: E731
        assert [tuple(t.shape) for t in ops.paged_plan(i(3), i(3), i(3, 2), i(9), i(1), 16, 7)] == [(7,)] * 4 + [(4,), (3,), (1,), (1,)]
        assert [tuple(t.shape) for t in ops.paged_release(i(3), i(3), i(3, 2), i(9), i(1), 16)] == [(3,), (1,)]
        lp, ent, tlp, tid = ops.token_logprobs(torch.empty(5, 40, device="cuda", dtype=torch.bfloat16), i(5), 4, 1.0)
        assert lp.dtype == ent.dtype == tlp.dtype == torch.float32 and tid.dtype == torch.int32 and tlp.shape == tid.shape == (5, 4)
        q = torch.empty(2, 8, 128, device="cuda", dtype=torch.bfloat16)
        assert ops.paged_prefix_attn(q, q, 4, 1, 2, 16, 128, 1, 0, i(3), 40, i(2, 2), i(2), 0.1, torch.float32).dtype == torch.float32
