"""libwf_torch.so: the tensor-level calls as native torch ops (csrc/torch_ops.cpp).  Loading it registers the CUDA kernels of
torch.ops.sgl_kernel.bitnet_{gemv,gemm,quantize_activations}* and the torch.ops.wf_native ops.

It lies beside libwf_bitnet.so and is linked against the torch it was built with.  Where there is none (WF_BITNET_LIB names a library elsewhere) or it
does not load (another torch), the same calls go through ctypes: the same kernels, about 12 us more host time a call."""
from __future__ import annotations

import ctypes as C
import threading
import warnings

import torch

from . import _lib

TORCH_LIB_PATH = _lib.LIB_PATH.parent / "libwf_torch.so"
_ops = None
_loading = threading.Lock()


class _Ctypes:
    """The wf_native ops on the functions of wf_bitnet.ops."""

    @staticmethod
    def linear(x, w, tile, N, K, w_scale):
        from . import ops
        q, act_scale, rowsum = ops.quantize_activations(x, per_token=False)
        return ops.ternary_linear(w if tile else w.contiguous(), N, K, q, layout="tile" if tile else "i2s", mode="linear", rowsum=rowsum, act_scale=act_scale,
                                  w_scale=w_scale, out_dtype=torch.float32)

    @staticmethod
    def mlp(x, gate_up_tile, N2, down_w, gate_scale, up_scale, down_scale, norm, eps):
        from . import ops
        q, s, rs = ops.quantize_activations(x, per_token=True)
        ws = torch.tensor([gate_scale, up_scale], dtype=torch.float32, device=x.device)
        h = ops.ternary_linear(gate_up_tile, N2, x.shape[1], q, mode="linear", rowsum=rs, act_scale=s, w_scale=ws, relu2_mul=True, out_dtype=torch.bfloat16)
        q, s, rs, _ = ops.rmsnorm_quant(h, norm, eps)
        ws = torch.tensor([down_scale], dtype=torch.float32, device=x.device)
        return ops.ternary_linear(down_w.contiguous(), down_w.shape[0], down_w.shape[1] * 4, q, layout="i2s", mode="linear", rowsum=rs, act_scale=s, w_scale=ws,
                                  out_dtype=torch.bfloat16)

    @staticmethod
    def paged_decode_attn(q, pool, max_pages, layers, kv_heads, page_size, head_dim, kv_dtype, layer, block_table, seq_lens, scale, out_dtype):
        from . import ops
        return ops.paged_decode_attn_ctypes(q, _lib.KvLayout(pool.data_ptr(), max_pages, layers, kv_heads, page_size, head_dim, kv_dtype), layer, block_table, seq_lens, scale,
                                            out_dtype)

    @staticmethod
    def paged_prefix_attn(q, pool, max_pages, layers, kv_heads, page_size, head_dim, kv_dtype, layer, prefix_table, prefix_len, block_table, seq_lens, scale, out_dtype):
        from . import ops
        _need(q, pool, prefix_table, block_table, seq_lens)
        if q.dim() != 3 or q.dtype != torch.bfloat16:
            raise ValueError("q must be bf16 [B, H, D]")
        B, H, D = q.shape
        if D != head_dim:
            raise ValueError(f"q has heads of {D}, the cache of {head_dim}")
        if pool.device != q.device:
            raise ValueError(f"the cache must be on {q.device}")
        pt, bt, sl = _i32(prefix_table, 1, q, "prefix_table"), _i32(block_table, 2, q, "block_table"), _i32(seq_lens, 1, q, "seq_lens")
        if bt.shape[0] != B or sl.shape[0] != B:
            raise ValueError(f"block_table and seq_lens must have a row for each of {B} sequences")
        if not 0 <= prefix_len <= pt.shape[0] * page_size:
            raise ValueError(f"prefix_len ({prefix_len}) beyond the {pt.shape[0]} pages of prefix_table")
        if bt.shape[1] * page_size > 0x7fffffff or prefix_len > 0x7fffffff:
            raise ValueError("block_table out of range")
        with torch.cuda.device(q.device):
            qc = q.contiguous()
            qc = qc.clone() if qc.data_ptr() % 16 else qc
            nbytes = int(_lib.lib().wf_prefix_attn_workspace_bytes(B, H, kv_heads, bt.shape[1] * page_size, prefix_len))       # 0 for sizes that the call refuses: no memory for them
            out = torch.empty(B if nbytes or not (bt.shape[1] or prefix_len) else 0, H, D, dtype=out_dtype, device=q.device)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
            layout = _lib.KvLayout(pool.data_ptr(), max_pages, layers, kv_heads, page_size, head_dim, kv_dtype)
            _lib.check(_lib.lib().wf_paged_prefix_attn(qc.data_ptr(), C.byref(layout), layer, pt.data_ptr(), prefix_len, bt.data_ptr(), bt.shape[1], sl.data_ptr(), B, H, float(scale),
                                                       out.data_ptr(), ops._DT[out_dtype], ws.data_ptr(), ws.numel(), ops._stream()))
        return out

    @staticmethod
    def paged_plan(seq_lens, new_lens, block_table, free_pages, free_count, page_size, max_tokens):
        from . import ops
        _need(seq_lens, new_lens, block_table, free_pages, free_count)
        _i32(block_table, 2, block_table, "block_table")
        sl, nl = _i32(seq_lens, 1, block_table, "seq_lens"), _i32(new_lens, 1, block_table, "new_lens")
        fp, fc = _i32(free_pages, 1, block_table, "free_pages"), _i32(free_count, 1, block_table, "free_count")
        B = block_table.shape[0]
        if sl.shape[0] != B or nl.shape[0] != B:
            raise ValueError(f"seq_lens and new_lens must have an entry for each of the {B} rows of block_table")
        if fc.shape[0] != 1:
            raise ValueError("free_count must have one entry")
        if not block_table.is_contiguous():
            raise ValueError("block_table must be contiguous (it is written in place)")
        if not (0 <= max_tokens <= 0x7fffffff and 0 <= page_size <= 0x7fffffff):
            raise ValueError("max_tokens or page_size out of range")
        with torch.cuda.device(block_table.device):
            cap4 = 0 if max_tokens > 1 << 30 else (max_tokens + 3) // 4 * 4          # (the call refuses more)
            buf = torch.empty(4 * cap4 + 2 * B + 3, dtype=torch.int32, device=block_table.device)
            at = (0, cap4, 2 * cap4, 3 * cap4, 4 * cap4, 4 * cap4 + B + 1, 4 * cap4 + 2 * B + 1, 4 * cap4 + 2 * B + 2)
            out = [buf[a:a + n] for a, n in zip(at, (max_tokens,) * 4 + (B + 1, B, 1, 1))]
            ptr = [buf.data_ptr() + 4 * a for a in at]
            _lib.check(_lib.lib().wf_paged_plan(sl.data_ptr(), nl.data_ptr(), B, block_table.data_ptr(), block_table.shape[1], fp.data_ptr(), fp.shape[0], fc.data_ptr(), page_size,
                                                max_tokens, ptr[1], ptr[0], *ptr[2:], ops._stream()))
        return out

    @staticmethod
    def paged_release(done, seq_lens, block_table, free_pages, free_count, page_size):
        from . import ops
        _need(done, seq_lens, block_table, free_pages, free_count)
        bt, sl = _i32(block_table, 2, block_table, "block_table"), _i32(seq_lens, 1, block_table, "seq_lens")
        _i32(free_pages, 1, block_table, "free_pages")
        fc = _i32(free_count, 1, block_table, "free_count")
        B = bt.shape[0]
        if done.dtype != torch.bool or done.dim() != 1 or done.device != bt.device:
            raise ValueError(f"done must be bool [B] on {bt.device}")
        if done.shape[0] != B or sl.shape[0] != B:
            raise ValueError(f"done and seq_lens must have an entry for each of the {B} rows of block_table")
        if fc.shape[0] != 1:
            raise ValueError("free_count must have one entry")
        if not free_pages.is_contiguous():
            raise ValueError("free_pages must be contiguous (it is written in place)")
        if not 0 <= page_size <= 0x7fffffff:
            raise ValueError("page_size out of range")
        with torch.cuda.device(bt.device):
            dn, lens, count = done.contiguous(), torch.empty_like(sl), torch.empty_like(fc)
            _lib.check(_lib.lib().wf_paged_release(dn.data_ptr(), sl.data_ptr(), B, bt.data_ptr(), bt.shape[1], free_pages.data_ptr(), free_pages.shape[0], fc.data_ptr(), page_size,
                                                   lens.data_ptr(), count.data_ptr(), ops._stream()))
        return lens, count

    @staticmethod
    def token_logprobs(logits, tokens, top, temperature):
        from . import ops
        _need(logits, tokens)
        if logits.dim() != 2:
            raise ValueError("logits must be [rows, vocab]")
        tk = _i32(tokens, 1, logits, "tokens")
        if tk.shape[0] != logits.shape[0]:
            raise ValueError(f"tokens must have an entry for each of the {logits.shape[0]} rows of logits")
        dt = ops._dt(logits)
        n, V = logits.shape
        if not 0 <= top <= 0x7fffffff:
            raise ValueError("top out of range")
        with torch.cuda.device(logits.device):
            x = logits if (V <= 1 or logits.stride(1) == 1) and (n <= 1 or logits.stride(0) >= V) else logits.contiguous()
            lp, ent = (torch.empty(n, dtype=torch.float32, device=x.device) for _ in range(2))
            k = top if top <= min(64, V) else 0                                       # (the call refuses more)
            tlp, tid = (torch.empty(n, k, dtype=t, device=x.device) for t in (torch.float32, torch.int32))
            _lib.check(_lib.lib().wf_token_logprobs(x.data_ptr(), dt, n, V, x.stride(0) if n > 1 else V, tk.data_ptr(), top, float(temperature), lp.data_ptr(), ent.data_ptr(),
                                                    tlp.data_ptr(), tid.data_ptr(), ops._stream()))
        return lp, ent, tlp, tid

    @staticmethod
    def norm_rope_kv_append(qkv, H, pool, max_pages, layers, kv_heads, page_size, head_dim, kv_dtype, layer, positions, pages, slots, cos_tab, sin_tab, q_norm, k_norm, eps, interleaved):
        from . import ops
        _need(qkv, pool, positions, pages, slots, cos_tab, sin_tab)
        if qkv.dim() != 2 or qkv.dtype != torch.bfloat16:
            raise ValueError("qkv must be bf16 [tokens, (H + 2 Hkv) * D]")
        T, row = qkv.shape
        if not 0 < H < 1 << 24 or row != (H + 2 * kv_heads) * head_dim:
            raise ValueError(f"qkv has rows of {row}, {H} and 2 x {kv_heads} heads of {head_dim} make another")
        if pool.device != qkv.device:
            raise ValueError(f"the cache must be on {qkv.device}")
        ps, pg, sl = _i32(positions, 1, qkv, "positions"), _i32(pages, 1, qkv, "pages"), _i32(slots, 1, qkv, "slots")
        if not ps.shape[0] == pg.shape[0] == sl.shape[0] == T:
            raise ValueError(f"positions, pages and slots must have an entry for each of {T} tokens")
        if cos_tab.dim() != 2 or sin_tab.shape != cos_tab.shape or cos_tab.dtype != sin_tab.dtype or cos_tab.device != qkv.device or sin_tab.device != qkv.device:
            raise ValueError(f"cos_tab and sin_tab must be alike, [max_pos, R / 2] on {qkv.device}")
        gains = [g for g in (q_norm, k_norm) if g is not None]
        for g in gains:
            if g.dim() != 1 or g.shape[0] != head_dim or g.device != qkv.device:
                raise ValueError(f"q_norm and k_norm must be [{head_dim}] on {qkv.device}")
        if len(gains) == 2 and gains[0].dtype != gains[1].dtype:
            raise ValueError("q_norm and k_norm must have the same type")
        with torch.cuda.device(qkv.device):
            x = qkv if qkv.stride(1) == 1 and (T <= 1 or (qkv.stride(0) >= row and qkv.stride(0) % 4 == 0)) and qkv.data_ptr() % 16 == 0 else _on16(qkv)
            c, s = _on16(cos_tab), _on16(sin_tab)
            gq, gk = (None if g is None else _on16(g) for g in (q_norm, k_norm))
            out = torch.empty(T, H, head_dim, dtype=torch.bfloat16, device=qkv.device)
            layout = _lib.KvLayout(pool.data_ptr(), max_pages, layers, kv_heads, page_size, head_dim, kv_dtype)
            _lib.check(_lib.lib().wf_norm_rope_kv_append(x.data_ptr(), x.stride(0) if T > 1 else row, T, H, C.byref(layout), layer, ps.data_ptr(), pg.data_ptr(), sl.data_ptr(), c.data_ptr(),
                                                         s.data_ptr(), ops._dt(c), 2 * c.shape[1], c.shape[0], _ptr(gq), _ptr(gk), ops._dt(gains[0]) if gains else 0, float(eps),
                                                         1 if interleaved else 0, out.data_ptr(), ops._stream()))
        return out

    @staticmethod
    def tree_plan(parents, offsets, seq_lens, max_nodes):
        from . import ops
        _need(parents, offsets, seq_lens)
        pa, of, sl = _i32(parents, 1, parents, "parents"), _i32(offsets, 1, parents, "offsets"), _i32(seq_lens, 1, parents, "seq_lens")
        if of.shape[0] != sl.shape[0] + 1:
            raise ValueError("offsets must have one entry more than seq_lens")
        if not 0 <= max_nodes <= 0x7fffffff:
            raise ValueError("max_nodes out of range")
        T = pa.shape[0]
        with torch.cuda.device(pa.device):
            mask = torch.empty(T, (max_nodes + 63) // 64 if max_nodes <= 256 else 0, dtype=torch.int64, device=pa.device)
            pos = torch.empty(T, dtype=torch.int32, device=pa.device)
            _lib.check(_lib.lib().wf_tree_plan(pa.data_ptr(), of.data_ptr(), sl.data_ptr(), sl.shape[0], T, max_nodes, mask.data_ptr(), pos.data_ptr(), ops._stream()))
        return mask, pos

    @staticmethod
    def paged_tree_attn(q, pool, max_pages, layers, kv_heads, page_size, head_dim, kv_dtype, layer, block_table, seq_lens, offsets, mask, scale, out_dtype):
        from . import ops
        _need(q, pool, block_table, seq_lens, offsets, mask)
        if q.dim() != 3 or q.dtype != torch.bfloat16:
            raise ValueError("q must be bf16 [tokens, H, D]")
        T, H, D = q.shape
        if D != head_dim:
            raise ValueError(f"q has heads of {D}, the cache of {head_dim}")
        if pool.device != q.device:
            raise ValueError(f"the cache must be on {q.device}")
        bt, sl, of = _i32(block_table, 2, q, "block_table"), _i32(seq_lens, 1, q, "seq_lens"), _i32(offsets, 1, q, "offsets")
        B = bt.shape[0]
        if sl.shape[0] != B or of.shape[0] != B + 1:
            raise ValueError(f"seq_lens must have an entry for each of the {B} rows of block_table, offsets one more")
        if mask.dtype != torch.int64 or mask.dim() != 2 or mask.shape[0] != T or mask.shape[1] == 0 or mask.device != q.device:
            raise ValueError(f"mask must be int64 [{T}, words] on {q.device}")
        if bt.shape[1] * page_size > 0x7fffffff:
            raise ValueError("block_table out of range")
        with torch.cuda.device(q.device):
            qc, mk = _on16(q), mask.contiguous()
            nbytes = int(_lib.lib().wf_tree_attn_workspace_bytes(B, T, H, kv_heads, mk.shape[1]))       # 0 for sizes that the call refuses: no memory for them
            out = torch.empty(T if nbytes or B == 0 else 0, H, D, dtype=out_dtype, device=q.device)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
            layout = _lib.KvLayout(pool.data_ptr(), max_pages, layers, kv_heads, page_size, head_dim, kv_dtype)
            _lib.check(_lib.lib().wf_paged_tree_attn(qc.data_ptr(), C.byref(layout), layer, bt.data_ptr(), bt.shape[1], sl.data_ptr(), of.data_ptr(), mk.data_ptr(), mk.shape[1], B, T, H,
                                                     float(scale), out.data_ptr(), ops._DT[out_dtype], ws.data_ptr(), ws.numel(), ops._stream()))
        return out

    @staticmethod
    def tree_accept(parents, tokens, targets, offsets, seq_lens, pool, max_pages, layers, kv_heads, page_size, head_dim, kv_dtype, block_table, free_pages, free_count):
        from . import ops
        _need(parents, tokens, targets, offsets, seq_lens, pool, block_table, free_pages, free_count)
        bt = _i32(block_table, 2, block_table, "block_table")
        pa, tk, tg, of, sl = (_i32(t, 1, bt, n) for t, n in ((parents, "parents"), (tokens, "tokens"), (targets, "targets"), (offsets, "offsets"), (seq_lens, "seq_lens")))
        _i32(free_pages, 1, bt, "free_pages")
        fc = _i32(free_count, 1, bt, "free_count")
        B, T = bt.shape[0], pa.shape[0]
        if pool.device != bt.device:
            raise ValueError(f"the cache must be on {bt.device}")
        if sl.shape[0] != B or of.shape[0] != B + 1:
            raise ValueError(f"seq_lens must have an entry for each of the {B} rows of block_table, offsets one more")
        if tk.shape[0] != T or tg.shape[0] != T:
            raise ValueError(f"tokens and targets must have an entry for each of {T} parents")
        if fc.shape[0] != 1:
            raise ValueError("free_count must have one entry")
        if not free_pages.is_contiguous():
            raise ValueError("free_pages must be contiguous (it is written in place)")
        with torch.cuda.device(bt.device):
            new = lambda n: torch.empty(n, dtype=torch.int32, device=bt.device)  # noqa: E731
            out = [new(B), new(T), new(B), new(B), new(1), new(1)]
            layout = _lib.KvLayout(pool.data_ptr(), max_pages, layers, kv_heads, page_size, head_dim, kv_dtype)
            _lib.check(_lib.lib().wf_tree_accept(pa.data_ptr(), tk.data_ptr(), tg.data_ptr(), of.data_ptr(), sl.data_ptr(), B, T, C.byref(layout), bt.data_ptr(), bt.shape[1],
                                                 free_pages.data_ptr(), free_pages.shape[0], fc.data_ptr(), *(t.data_ptr() for t in out), ops._stream()))
        return out

    @staticmethod
    def process_logits(logits, history, history_lens, prompt_lens, repetition, frequency, presence, bias_ids, bias_values, allowed, offsets, node_tokens, node_mask, out):
        from . import ops
        _need(logits)
        if logits.dim() != 2:
            raise ValueError("logits must be [rows, vocab]")
        N, V = logits.shape

        def take(t, dtype, dim, name):
            if t is None:
                return None
            if t.dtype != dtype:
                raise ValueError(f"{name} must be {dtype}")
            if t.dim() != dim:
                raise ValueError(f"{name} must have {dim} dimension{'' if dim == 1 else 's'}")
            if t.device != logits.device:
                raise ValueError(f"{name} must be on {logits.device}")
            return t.contiguous()
        off = take(offsets, torch.int32, 1, "offsets")
        if off is not None and off.shape[0] == 0:
            raise ValueError("offsets must have an entry more than there are sequences")
        B = N if off is None else off.shape[0] - 1
        hist = take(history, torch.int32, 2, "history")
        if hist is not None and hist.shape[0] != B:
            raise ValueError(f"history must have a row for each of {B} sequences")
        each = []
        for t, dtype, name in ((history_lens, torch.int32, "history_lens"), (prompt_lens, torch.int32, "prompt_lens"), (repetition, torch.float32, "repetition"),
                               (frequency, torch.float32, "frequency"), (presence, torch.float32, "presence")):
            x = take(t, dtype, 1, name)
            if x is not None and x.shape[0] != B:
                raise ValueError(f"{name} must have an entry for each of {B} sequences")
            each.append(x)
        bi, bv = take(bias_ids, torch.int32, 2, "bias_ids"), None
        if bi is not None:
            bv = take(bias_values, torch.float32, 2, "bias_values")
            if bv is None or bv.shape != bi.shape or bi.shape[0] != B:
                raise ValueError(f"bias_ids and bias_values must be alike, with a row for each of {B} sequences")
        ok = take(allowed, torch.int32, 2, "allowed")
        if ok is not None and ok.shape != (N, (V + 31) // 32):
            raise ValueError(f"allowed must be [{N}, {(V + 31) // 32}]")
        nm, nt = take(node_mask, torch.int64, 2, "node_mask"), None
        if nm is not None:
            nt = take(node_tokens, torch.int32, 1, "node_tokens")
            if nt is None or nt.shape[0] != N or nm.shape[0] != N:
                raise ValueError(f"node_mask and node_tokens must have an entry for each of {N} rows")
        fits = lambda t: (V <= 1 or t.stride(1) == 1) and (N <= 1 or t.stride(0) >= V)  # noqa: E731
        dt = ops._dt(logits)
        if out is not None:
            if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
                raise ValueError("out must be as logits is")
            if not fits(out):
                raise ValueError("out must have its rows' entries side by side (it is written in place)")
        with torch.cuda.device(logits.device):
            x = logits if fits(logits) else logits.contiguous()
            y = torch.empty(N, V, dtype=logits.dtype, device=logits.device) if out is None else out
            a = _lib.LogitsArgs(x.data_ptr(), y.data_ptr(), dt, N, V, B, x.stride(0) if N > 1 else V, y.stride(0) if N > 1 else V, _ptr(off), _ptr(hist), 0 if hist is None else hist.shape[1],
                                *(_ptr(t) for t in each), _ptr(bi), _ptr(bv), _ptr(ok), 0 if ok is None else ok.shape[1], _ptr(nt), _ptr(nm), 0 if hist is None else hist.shape[1],
                                0 if bi is None else bi.shape[1], 0 if nm is None else nm.shape[1])
            _lib.check(_lib.lib().wf_process_logits(C.byref(a), ops._stream()))
        return y if out is None else logits.new_empty(0)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _on16(t):
    """contiguous, from a 16-byte boundary"""
    c = t.contiguous()
    return c.clone() if c.data_ptr() % 16 else c


def _need(*ts):
    from . import ops
    ops._need_cuda(*ts)


def _i32(t, dim, like, name):
    """an int32 tensor of `dim` dimensions on the device of `like`, contiguous"""
    if t.dtype != torch.int32:
        raise ValueError(f"{name} must be int32")
    if t.dim() != dim:
        raise ValueError(f"{name} must have {dim} dimension{'' if dim == 1 else 's'}")
    if t.device != like.device:
        raise ValueError(f"{name} must be on {like.device}")
    return t.contiguous()


def _fake_linear(x, w, tile, N, K, w_scale):
    return x.new_empty(x.shape[0], N, dtype=torch.float32)


def _fake_mlp(x, gate_up_tile, N2, down_w, gate_scale, up_scale, down_scale, norm, eps):
    return x.new_empty(x.shape[0], down_w.shape[0], dtype=torch.bfloat16)


def _fake_attn(q, pool, max_pages, layers, kv_heads, page_size, head_dim, kv_dtype, layer, block_table, seq_lens, scale, out_dtype):
    return q.new_empty(q.shape, dtype=out_dtype)


def _fake_prefix_attn(q, pool, max_pages, layers, kv_heads, page_size, head_dim, kv_dtype, layer, prefix_table, prefix_len, block_table, seq_lens, scale, out_dtype):
    return q.new_empty(q.shape, dtype=out_dtype)


def _fake_plan(seq_lens, new_lens, block_table, free_pages, free_count, page_size, max_tokens):
    B = block_table.shape[0]
    return [block_table.new_empty(n) for n in (max_tokens,) * 4 + (B + 1, B, 1, 1)]


def _fake_release(done, seq_lens, block_table, free_pages, free_count, page_size):
    return seq_lens.new_empty(seq_lens.shape), free_count.new_empty(1)


def _fake_logprobs(logits, tokens, top, temperature):
    n = logits.shape[0]
    f = lambda *s: logits.new_empty(s, dtype=torch.float32)  # noqa: E731
    return f(n), f(n), f(n, top), logits.new_empty((n, top), dtype=torch.int32)


def _fake_append(qkv, H, pool, max_pages, layers, kv_heads, page_size, head_dim, kv_dtype, layer, positions, pages, slots, cos_tab, sin_tab, q_norm, k_norm, eps, interleaved):
    return qkv.new_empty(qkv.shape[0], H, head_dim)


def _fake_tree_plan(parents, offsets, seq_lens, max_nodes):
    return parents.new_empty((parents.shape[0], (max_nodes + 63) // 64), dtype=torch.int64), parents.new_empty(parents.shape)


def _fake_tree_attn(q, pool, max_pages, layers, kv_heads, page_size, head_dim, kv_dtype, layer, block_table, seq_lens, offsets, mask, scale, out_dtype):
    return q.new_empty(q.shape, dtype=out_dtype)


def _fake_accept(parents, tokens, targets, offsets, seq_lens, pool, max_pages, layers, kv_heads, page_size, head_dim, kv_dtype, block_table, free_pages, free_count):
    B = block_table.shape[0]
    return [block_table.new_empty(n) for n in (B, parents.shape[0], B, B, 1, 1)]


def _fake_logits(logits, history, history_lens, prompt_lens, repetition, frequency, presence, bias_ids, bias_values, allowed, offsets, node_tokens, node_mask, out):
    return logits.new_empty(logits.shape if out is None else 0)


_FAKES = {"linear": _fake_linear, "mlp": _fake_mlp, "paged_decode_attn": _fake_attn, "paged_prefix_attn": _fake_prefix_attn, "paged_plan": _fake_plan,
          "paged_release": _fake_release, "token_logprobs": _fake_logprobs, "norm_rope_kv_append": _fake_append, "tree_plan": _fake_tree_plan,
          "paged_tree_attn": _fake_tree_attn, "tree_accept": _fake_accept, "process_logits": _fake_logits}


def _load():
    if not TORCH_LIB_PATH.exists():
        _lib.lib()                       # raises where there is no library at all
        why = f"{TORCH_LIB_PATH} not found (`make -C {_lib._PKG_ROOT / 'csrc'}` builds it)"
    else:
        try:
            torch.ops.load_library(str(TORCH_LIB_PATH))
        except OSError as e:
            why = f"{TORCH_LIB_PATH} does not load: {e}"
        else:
            for name, fake in _FAKES.items():
                torch.library.register_fake(f"wf_native::{name}", fake)
            return torch.ops.wf_native
    warnings.warn(f"{why}; the BitNet ops call their kernels through ctypes")
    return _Ctypes


def ops():
    """torch.ops.wf_native, or the same functions through ctypes; raises when libwf_bitnet.so has not been built."""
    global _ops
    if _ops is None:
        with _loading:
            if _ops is None:
                _ops = _load()
    return _ops


def is_native() -> bool:
    return ops() is not _Ctypes
