"""Refusals of the operators on drafted tokens (masks, norm, rotation and append, attention, acceptance, logits) through the C ABI, their workspace size and their torch ops'
registration: nothing here needs a GPU."""
import ctypes as C

import pytest
import torch

from wf_bitnet import _lib

BUF = (C.c_uint8 * 4096)()
P = (C.addressof(BUF) + 255) // 256 * 256                # 256-byte aligned host memory: never read, every call here ends at its checks
BAD, NO = _lib.WF_ERR_INVALID, _lib.WF_ERR_UNSUPPORTED


def layout(**f):
    a = dict(pool=P, max_pages=8, layers=2, kv_heads=2, page_size=16, head_dim=128, dtype=_lib.WF_BF16)
    a.update(f)
    return C.byref(_lib.KvLayout(*a.values()))


def test_tree_plan():
    L = _lib.lib()

    def call(**k):
        a = dict(parents=P, offsets=P, lens=P, rows=2, tokens=9, nodes=64, mask=P, pos=P)
        a.update(k)
        return L.wf_tree_plan(*a.values(), None)
    for bad in (dict(rows=-1), dict(tokens=-1), dict(nodes=0), dict(nodes=-5), dict(parents=None), dict(offsets=None), dict(lens=None), dict(mask=None), dict(pos=None), dict(mask=P + 4)):
        assert call(**bad) == BAD, bad
        assert b"wf_tree_plan" in L.wf_last_error()
    for bad in (dict(nodes=257), dict(tokens=(1 << 30) + 1), dict(rows=(1 << 20) + 1)):
        assert call(**bad) == NO, bad
    assert call(tokens=0, parents=None, mask=None, pos=None) == _lib.WF_OK


def test_append():
    L = _lib.lib()

    def call(kv=None, **k):
        a = dict(qkv=P, ld=1536, T=3, H=8, kv=layout(**(kv or {})), layer=1, pos=P, pages=P, slots=P, cos=P, sin=P, tab=_lib.WF_F32, rot=128, max_pos=10, qn=P, kn=P, nt=_lib.WF_BF16, eps=1e-6, pairs=0,
                 out=P)
        a.update(k)
        return L.wf_norm_rope_kv_append(*a.values(), None)
    for bad in (dict(T=-1), dict(H=0), dict(layer=2), dict(layer=-1), dict(rot=-8), dict(rot=136), dict(max_pos=-1), dict(tab=_lib.WF_F16), dict(nt=_lib.WF_F16), dict(eps=-1.0), dict(eps=float("nan")),
                dict(eps=float("inf")), dict(ld=1535), dict(ld=1538), dict(qkv=None), dict(pos=None), dict(pages=None), dict(slots=None), dict(cos=None), dict(sin=None), dict(out=None), dict(qkv=P + 2),
                dict(out=P + 8), dict(qn=P + 4), dict(cos=P + 8), dict(kv=dict(pool=None)), dict(kv=dict(kv_heads=0)), dict(kv=dict(pool=P + 4))):
        assert call(**bad) == BAD, bad
        assert b"wf_norm_rope_kv_append" in L.wf_last_error()
    for bad in (dict(rot=12), dict(kv=dict(head_dim=96)), dict(rot=64, ld=768, kv=dict(head_dim=64, dtype=_lib.WF_I8)), dict(ld=8192, kv=dict(head_dim=256, dtype=_lib.WF_I8)), dict(kv=dict(dtype=_lib.WF_F32)), dict(H=1 << 21, ld=1 << 40), dict(T=(1 << 30) + 1)):
        assert call(**bad) == NO, bad
    assert call(T=0, qkv=None, out=None) == _lib.WF_OK


def test_tree_attention():
    L = _lib.lib()

    def call(kv=None, **k):
        a = dict(q=P, kv=layout(**(kv or {})), layer=1, table=P, blocks=4, lens=P, offsets=P, mask=P, words=1, B=2, T=9, H=8, scale=0.1, out=P, dt=_lib.WF_BF16, ws=P, ws_bytes=1 << 40)
        a.update(k)
        return L.wf_paged_tree_attn(*a.values(), None)
    for bad in (dict(q=None), dict(table=None), dict(lens=None), dict(offsets=None), dict(mask=None), dict(out=None), dict(ws=None), dict(ws_bytes=16), dict(blocks=-1), dict(B=-1), dict(T=-1), dict(H=0),
                dict(words=0), dict(layer=2), dict(layer=-1), dict(dt=_lib.WF_F16), dict(q=P + 2), dict(out=P + 8), dict(ws=P + 8), dict(mask=P + 4), dict(kv=dict(pool=None)), dict(kv=dict(pool=P + 2)),
                dict(kv=dict(kv_heads=0))):
        assert call(**bad) == BAD, bad
        assert b"wf_paged_tree_attn" in L.wf_last_error()
    for bad in (dict(kv=dict(head_dim=64)), dict(kv=dict(page_size=24)), dict(kv=dict(kv_heads=3)), dict(H=18), dict(kv=dict(dtype=_lib.WF_F32)), dict(words=5), dict(blocks=1 << 27), dict(T=1 << 22),
                dict(B=65537)):
        assert call(**bad) == NO, bad
    assert call(T=0, q=None, out=None) == _lib.WF_OK


def test_tree_attention_workspace():
    L = _lib.lib()
    assert L.wf_tree_attn_workspace_bytes(0, 9, 8, 2, 1) == L.wf_tree_attn_workspace_bytes(2, 9, 8, 2, 5) == 0
    sms = L.wf_sm_count()
    for B, T, H, Hkv, words in ((1, 1, 1, 1, 1), (8, 480, 20, 5, 1), (64, 9000, 64, 8, 4)):
        n = L.wf_tree_attn_workspace_bytes(B, T, H, Hkv, words)
        rows = min(256, -(-64 * words * H // Hkv // 32) * 32)
        assert 2 * sms * rows * 130 * 4 < n <= 2 * sms * (rows * 130 * 4 + 64) + 256


def test_accept():
    L = _lib.lib()

    def call(kv=None, **k):
        a = dict(parents=P, tokens=P, targets=P, offsets=P, lens=P, rows=2, n=9, kv=layout(**(kv or {})), table=P, blocks=4, free=P, pool=8, count=P, acc=P, path=P, nxt=P, out=P, cout=P, status=P)
        a.update(k)
        return L.wf_tree_accept(*a.values(), None)
    for bad in (dict(rows=-1), dict(n=-1), dict(blocks=-1), dict(pool=-1), dict(parents=None), dict(tokens=None), dict(targets=None), dict(offsets=None), dict(lens=None), dict(table=None), dict(free=None),
                dict(count=None), dict(acc=None), dict(path=None), dict(nxt=None), dict(out=None), dict(cout=None), dict(status=None), dict(kv=dict(pool=None)), dict(kv=dict(pool=P + 4)),
                dict(kv=dict(page_size=0))):
        assert call(**bad) == BAD, bad
        assert b"wf_tree_accept" in L.wf_last_error()
    for bad in (dict(rows=8193), dict(n=(1 << 30) + 1), dict(pool=(1 << 30) + 1), dict(kv=dict(head_dim=12)), dict(kv=dict(dtype=_lib.WF_F16)), dict(kv=dict(layers=1 << 26, kv_heads=1 << 4))):
        assert call(**bad) == NO, bad


def test_logits():
    L = _lib.lib()

    def call(**k):
        a = _lib.LogitsArgs(logits=P, out=P + 1024, dtype=_lib.WF_F32, rows=2, vocab=64, sequences=2, row_stride=64, out_stride=64, history=P, history_stride=5, history_width=5, bias_ids=P, bias_values=P,
                            bias_width=3, allowed=P, allowed_stride=2, node_tokens=P, node_mask=P, mask_words=1)
        for name, v in k.items():
            setattr(a, name, v)
        return L.wf_process_logits(C.byref(a), None)
    for bad in (dict(rows=-1), dict(vocab=0), dict(sequences=-1), dict(dtype=_lib.WF_I8), dict(row_stride=63), dict(out_stride=63), dict(sequences=3), dict(history_width=-1), dict(bias_width=-1),
                dict(mask_words=-1), dict(logits=None), dict(out=None), dict(bias_values=None), dict(node_tokens=None), dict(history_stride=4), dict(allowed_stride=1), dict(logits=P + 2), dict(out=P + 3),
                dict(node_mask=P + 4), dict(out=P, out_stride=128), dict(out=P + 4), dict(out=P + 256), dict(out=P - 252), dict(out=P + 256, out_stride=128),
                dict(out=P + 252, row_stride=128, out_stride=128), dict(out=P - 252, row_stride=128, out_stride=128)):
        assert call(**bad) == BAD, bad
        assert b"wf_process_logits" in L.wf_last_error()
    for bad in (dict(vocab=(1 << 30) + 1, row_stride=1 << 40, out_stride=1 << 40), dict(rows=(1 << 30) + 1, sequences=(1 << 30) + 1), dict(rows=65535, sequences=65535), dict(bias_width=65536),
                dict(mask_words=5)):
        assert call(**bad) == NO, bad
    assert call(rows=0, sequences=0, logits=None, out=None) == _lib.WF_OK
    assert L.wf_process_logits(None, None) == BAD


def test_torch_ops_and_their_fakes():
    from wf_bitnet import _native
    if not _native.is_native():
        pytest.skip("no libwf_torch.so")
    ops = _native.ops()
    for name in ("norm_rope_kv_append", "tree_plan", "paged_tree_attn", "tree_accept", "process_logits"):
        assert "AutogradCUDA: fallthrough" in torch._C._dispatch_dump_table(f"wf_native::{name}")
        assert hasattr(_native._Ctypes, name)
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        i = lambda *s: torch.empty(*s, dtype=torch.int32, device="cuda")  # noqa: E731
        mask, pos = ops.tree_plan(i(9), i(3), i(2), 65)
        assert mask.shape == (9, 2) and mask.dtype == torch.int64 and pos.shape == (9,) and pos.dtype == torch.int32
        q = torch.empty(9, 8, 128, device="cuda", dtype=torch.bfloat16)
        assert ops.paged_tree_attn(q, q, 4, 1, 2, 16, 128, 1, 0, i(2, 2), i(2), i(3), mask, 0.1, torch.float32).dtype == torch.float32
        assert [tuple(t.shape) for t in ops.tree_accept(i(9), i(9), i(9), i(3), i(2), q, 4, 1, 2, 16, 128, 1, i(2, 2), i(8), i(1))] == [(2,), (9,), (2,), (2,), (1,), (1,)]
        x = torch.empty(9, 1536, device="cuda", dtype=torch.bfloat16)
        t = torch.empty(10, 64, device="cuda")
        assert ops.norm_rope_kv_append(x, 8, q, 4, 1, 2, 16, 128, 1, 0, i(9), i(9), i(9), t, t, None, None, 1e-6, False).shape == (9, 8, 128)
        assert ops.process_logits(x, *(None,) * 13).shape == x.shape
