"""Operators of a serving step over the paged cache, as cases that can be timed and compared: block tables and slot maps planned on the GPU
from request lengths (and pages handed back), decode attention of a batch that shares a long prefix, and log probabilities of given tokens
with entropy and top alternatives.

`run` computes them in elementary torch operations, or with `own` through the framework's entry points; `exact` states the results in
64 bits, or as whole numbers, from their definitions."""
from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_PKG = str(Path(__file__).resolve().parents[1] / "wrinklefree-inference-engine_b200")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

F64 = torch.float64
DIM = 128                                              # size of a head
HEADS = ((20, 5), (32, 8), (64, 8))                    # (query heads, key/value heads)
VOCABS = (32000, 32768, 128256)
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # the plan of a decode step: 32 sequences, one token each (the smallest call, latency alone)
        {"name": "plan_decode_32", "kind": "plan", "rows": 32, "portion": 1, "share": 1.0, "ctx": 4096, "page": 16, "capacity": 32},
        # a step that mixes 256 sequences, an eighth of them with a portion of a prompt, buffers padded to the step's budget
        {"name": "plan_mixed_256", "kind": "plan", "rows": 256, "portion": 700, "share": 0.125, "ctx": 8192, "page": 16, "capacity": 24576},
        # prompts of a large batch planned at once, pages of 48 tokens
        {"name": "plan_prompts_2048", "kind": "plan", "rows": 2048, "portion": 250, "share": 1.0, "ctx": 1500, "page": 48, "capacity": 524288},
        # half of 512 sequences have ended and hand their pages back
        {"name": "release_512", "kind": "release", "rows": 512, "share": 0.5, "ctx": 8192, "page": 16},
        # four sequences behind a system prompt of odd length, 2B heads
        {"name": "prefix_4_2k", "kind": "prefix", "b": 4, "heads": 20, "kv_heads": 5, "prefix": 1987, "ctx": 60, "page": 16, "cache": "bf16"},
        # a batch of 64 behind a long instruction, 2B heads
        {"name": "prefix_64_8k", "kind": "prefix", "b": 64, "heads": 20, "kv_heads": 5, "prefix": 8192, "ctx": 300, "page": 16, "cache": "bf16"},
        # 128 questions about one long document, 8B heads (the largest)
        {"name": "prefix_128_32k", "kind": "prefix", "b": 128, "heads": 32, "kv_heads": 8, "prefix": 32768, "ctx": 512, "page": 64, "cache": "bf16"},
        # 70B heads and the 8-bit cache, the document's last page part full
        {"name": "prefix_31_16k_int8", "kind": "prefix", "b": 31, "heads": 64, "kv_heads": 8, "prefix": 16003, "ctx": 1000, "page": 32, "cache": "int8"},
        # the token just drawn, with the alternatives that an API returns
        {"name": "logprobs_1", "kind": "logprobs", "n": 1, "vocab": 128256, "type": "f32", "top": 20, "masked": 0.0, "temperature": 1.0},
        # a decode batch whose logits come in bf16
        {"name": "logprobs_64_bf16", "kind": "logprobs", "n": 64, "vocab": 128256, "type": "bf16", "top": 5, "masked": 0.0, "temperature": 0.7},
        # decoding under a grammar: in a third of the rows few tokens are allowed; odd vocabulary
        {"name": "logprobs_33_grammar", "kind": "logprobs", "n": 33, "vocab": 32003, "type": "f16", "top": 64, "masked": 0.33, "temperature": 1.0},
        # a prompt is scored, every position of it
        {"name": "logprobs_score_2000", "kind": "logprobs", "n": 2000, "vocab": 128256, "type": "f32", "top": 0, "masked": 0.0, "temperature": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("plan", "release", "prefix", "prefix", "logprobs", "logprobs"))
    if kind == "plan":
        rows, share = _log(rng, 1, 2048), rng.choice((1.0, 0.5, 0.125))
        portion = _log(rng, 1, max(1, min(4000, 262144 // rows)))
        capacity = min(524288, rows + int(rows * share * portion * rng.uniform(1.0, 1.5)) + 1)
        return {"kind": kind, "rows": rows, "portion": portion, "share": share, "ctx": _log(rng, 1, 8192 if rows <= 512 else 1500), "page": rng.choice((1, 16, 16, 32, 48, 64, 7)),
                "capacity": capacity}
    if kind == "release":
        rows = _log(rng, 1, 512)
        return {"kind": kind, "rows": rows, "share": rng.uniform(0.0, 1.0), "ctx": _log(rng, 1, 8192), "page": rng.choice((1, 16, 16, 32, 48, 64, 7))}
    if kind == "prefix":
        heads, kv_heads = rng.choice(HEADS)
        b = _log(rng, 1, 128)
        prefix = _log(rng, 1, 32768)
        if heads == 64:
            prefix = max(1, prefix // 2)
        return {"kind": kind, "b": b, "heads": heads, "kv_heads": kv_heads, "prefix": prefix, "ctx": _log(rng, 1, 512 if b > 32 else 2048), "page": rng.choice((16, 16, 32, 48, 64, 128)),
                "cache": rng.choice(("bf16", "bf16", "int8"))}
    vocab = rng.choice(VOCABS + (_log(rng, 100, 128256) | 1,))
    return {"kind": kind, "n": _log(rng, 1, max(1, min(2000, 128256 * 2000 // vocab))), "vocab": vocab, "type": rng.choice(("f32", "bf16", "f16")), "top": rng.choice((0, 1, 5, 20, 64)),
            "masked": rng.choice((0.0, 0.0, 0.33)), "temperature": rng.choice((1.0, 1.0, 0.7, 1.3))}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _lengths(g, n, hi):
    """n lengths from a half of `hi` to `hi`"""
    return torch.randint(max(1, hi // 2), hi + 1, (n,), generator=g, device="cuda", dtype=torch.int32)


def _tables(g, held, page, blocks, pages):
    """rows of pages in the order of a shuffled pool, and the pages that are left"""
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    have = (held + page - 1) // page
    first = torch.cumsum(have, 0) - have
    j = torch.arange(blocks, device="cuda")
    at = first[:, None] + j
    table = torch.where(j < have[:, None], order[at.clamp(max=pages - 1).long()], -1).to(torch.int32)
    return table.contiguous(), order, int(have.sum())


def _inputs(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    if kind in ("plan", "release"):
        rows, page = case["rows"], case["page"]
        lens = _lengths(g, rows, case["ctx"])
        new = torch.zeros_like(lens)
        if kind == "plan":
            new = torch.where(torch.rand(rows, generator=g, device="cuda") < case["share"], _lengths(g, rows, case["portion"]), 1).to(torch.int32)
            fits = torch.cumsum(new, 0) <= case["capacity"]
            new = torch.where(fits, new, 0).to(torch.int32)
        blocks = (case["ctx"] + case.get("portion", 0) + page - 1) // page + 1
        pages = rows * blocks
        table, order, used = _tables(g, lens, page, blocks, pages)
        free = torch.empty(pages, dtype=torch.int32, device="cuda")
        free.fill_(-1)
        free[:pages - used] = order[used:]
        s = {"case": case, "lens": lens, "new": new, "table": table, "free": free, "count": torch.tensor([pages - used], dtype=torch.int32, device="cuda")}
        if kind == "release":
            s["done"] = torch.rand(rows, generator=g, device="cuda") < case["share"]
        return s
    if kind == "prefix":
        b, heads, kvh, page, layers = case["b"], case["heads"], case["kv_heads"], case["page"], 2
        lens = _lengths(g, b, case["ctx"])
        blocks, pblocks = (case["ctx"] + page - 1) // page, (case["prefix"] + page - 1) // page
        pages = b * blocks + pblocks
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        q = torch.randn(b, heads, DIM, generator=g, device="cuda").to(torch.bfloat16)
        shape = (pages, layers, 2, kvh, page, DIM)
        s = {"case": case, "q": q, "lens": lens, "table": order[pblocks:].view(b, blocks).contiguous(), "prefix_table": order[:pblocks].contiguous(), "layer": 1}
        if case["cache"] == "int8":                    # codes are kept as code + 128
            s["pool"] = torch.randint(1, 256, shape, generator=g, device="cuda", dtype=torch.uint8)
            s["scales"] = (torch.rand(shape[:-1], generator=g, device="cuda") * 0.01 + 0.015)
        else:
            s["pool"] = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)
        return s
    n, v = case["n"], case["vocab"]
    x = torch.randn(n, v, generator=g, device="cuda") * 2.5
    if case["masked"]:
        rows = torch.rand(n, 1, generator=g, device="cuda") < case["masked"]
        x = torch.where(rows & (torch.rand(n, v, generator=g, device="cuda") > 100.0 / v), -math.inf, x)
    return {"case": case, "logits": x.to(TYPES[case["type"]]), "tokens": torch.randint(0, v, (n,), generator=g, device="cuda", dtype=torch.int32)}


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["kind"] == "prefix":               # the handle on the cache that a program keeps
        from wf_bitnet import ops
        pool, scales = s.pop("pool"), s.pop("scales", None)
        s["kv"] = ops.PagedKV(pool.shape[0], pool.shape[1], pool.shape[3], pool.shape[4], DIM, dtype=torch.bfloat16 if scales is None else torch.int8)
        s["kv"].pool.copy_(pool)
        if scales is not None:
            s["kv"].scales.copy_(scales)
    return s


# ---- the plain forms
def _plan(s):
    c = s["case"]
    page, cap = c["page"], c["capacity"]
    lens, new, table, free, count = s["lens"].long(), s["new"].long(), s["table"], s["free"], s["count"].long()
    total = lens + new
    old = (lens + page - 1) // page
    need = (total + page - 1) // page - old
    tok_end, page_end = torch.cumsum(new, 0), torch.cumsum(need, 0)
    status = ((page_end[-1:] > count) * 1 + (tok_end[-1:] > cap) * 2 + (((total + page - 1) // page).amax(0, keepdim=True) > table.shape[1]) * 4).to(torch.int32)
    ok = status == 0
    j = torch.arange(table.shape[1], device="cuda")
    k = (page_end - need)[:, None] + j - old[:, None]
    fresh = (k >= (page_end - need)[:, None]) & (k < page_end[:, None]) & ok
    table = torch.where(fresh, free[(count - 1 - k).clamp(0, free.shape[0] - 1)], table)
    t = torch.arange(cap, device="cuda")
    row = torch.searchsorted(tok_end, t, right=True)
    live = (row < lens.shape[0]) & ok
    r = row.clamp(max=lens.shape[0] - 1)
    pos = lens[r] + t - (tok_end - new)[r]
    block = (pos // page).clamp(0, table.shape[1] - 1)
    i32 = lambda x, other: torch.where(live, x, other).to(torch.int32)  # noqa: E731
    offsets = torch.cat([torch.zeros_like(tok_end[:1]), tok_end])
    return {"positions": i32(pos, 0), "rows": i32(row, -1), "pages": i32(table[r, block].long(), -1), "slots": i32(pos % page, 0), "offsets": torch.where(ok, offsets, 0).to(torch.int32),
            "lens": torch.where(ok, total, lens).to(torch.int32), "count": torch.where(ok, count - page_end[-1:], count).to(torch.int32), "status": status, "table": table}


def _release(s):
    page = s["case"]["page"]
    lens, table, free, count, done = s["lens"].long(), s["table"], s["free"], s["count"].long(), s["done"]
    have = torch.where(done, (lens + page - 1) // page, 0)
    end = torch.cumsum(have, 0)
    k = torch.arange(free.shape[0], device="cuda") - count
    row = torch.searchsorted(end, k, right=True).clamp(max=lens.shape[0] - 1)
    j = (k - (end - have)[row]).clamp(0, table.shape[1] - 1)
    back = (k >= 0) & (k < end[-1:])
    return {"free": torch.where(back, table[row, j], free), "lens": torch.where(done, 0, lens).to(torch.int32), "count": (count + end[-1:]).to(torch.int32)}


def _rows_of(s, table, kv):
    """[..., kv heads, tokens, DIM] in float of the pages that `table` names"""
    x = s["pool"][table.long(), s["layer"], kv].float()
    if "scales" in s:
        x = (x - 128.0) * s["scales"][table.long(), s["layer"], kv][..., None]
    x = x.transpose(-4, -3)                            # [..., kv heads, blocks, page, DIM]
    return x.reshape(*x.shape[:-3], x.shape[-3] * x.shape[-2], DIM)


def _prefix(s):
    c = s["case"]
    b, h, kvh = c["b"], c["heads"], c["kv_heads"]
    q = s["q"].float().view(b, kvh, h // kvh, DIM) / math.sqrt(DIM)
    kp, vp = _rows_of(s, s["prefix_table"], 0)[:, :c["prefix"]], _rows_of(s, s["prefix_table"], 1)[:, :c["prefix"]]
    ko, vo = _rows_of(s, s["table"], 0), _rows_of(s, s["table"], 1)
    sp = torch.matmul(q.transpose(0, 1).reshape(kvh, -1, DIM), kp.transpose(1, 2))               # [kv heads, b * group, prefix]
    so = torch.matmul(q, ko.transpose(2, 3))                                                     # [b, kv heads, group, own]
    so = torch.where(torch.arange(ko.shape[2], device="cuda") < s["lens"][:, None, None, None], so, -math.inf)
    sp = sp.view(kvh, b, h // kvh, -1)
    top = torch.maximum(sp.amax(-1).transpose(0, 1), so.amax(-1))                                # [b, kv heads, group]
    ep, eo = torch.exp(sp - top.transpose(0, 1)[..., None]), torch.exp(so - top[..., None])
    o = torch.matmul(ep.view(kvh, -1, c["prefix"]), vp).view(kvh, b, -1, DIM).transpose(0, 1) + torch.matmul(eo, vo)
    return (o / (ep.sum(-1).transpose(0, 1) + eo.sum(-1))[..., None]).reshape(b, h, DIM).to(torch.bfloat16)


def _logprobs(s):
    c = s["case"]
    x = s["logits"].float()
    z = x / c["temperature"]
    top = z.amax(-1, keepdim=True)
    d = z - top
    e = torch.exp(d)
    total = e.sum(-1)
    lse = torch.log(total)
    entropy = lse - (e * torch.where(e > 0, d, 0.0)).sum(-1) / total
    out = {"logprobs": d.gather(1, s["tokens"].long()[:, None])[:, 0] - lse, "entropy": entropy}
    if c["top"]:
        bits = (x + 0.0).view(torch.int32)
        bits = bits ^ ((bits >> 31) & 0x7fffffff)      # orders as the numbers do; ties: the lowest index
        key = (bits.long() << 32) + (c["vocab"] - torch.arange(c["vocab"], device="cuda"))
        ids = c["vocab"] - (torch.topk(key, c["top"], sorted=True).values & 0xffffffff)
        out["top_logprobs"], out["top_ids"] = d.gather(1, ids) - lse[:, None], ids.to(torch.int32)
    return out


def run(s):
    c = s["case"]
    kind = c["kind"]
    if not own:
        return {"plan": _plan, "release": _release, "prefix": _prefix, "logprobs": _logprobs}[kind](s)
    from wf_bitnet import ops
    if kind == "plan":
        p = ops.paged_plan(s["lens"], s["new"], s["table"], s["free"], s["count"], c["page"], c["capacity"])
        return {"positions": p.positions, "rows": p.rows, "pages": p.pages, "slots": p.slots, "offsets": p.offsets, "lens": p.lens, "count": p.free_count, "status": p.status,
                "table": s["table"]}
    if kind == "release":
        lens, count = ops.paged_release(s["done"], s["lens"], s["table"], s["free"], s["count"], c["page"])
        return {"free": s["free"], "lens": lens, "count": count}
    if kind == "prefix":
        return ops.paged_prefix_attn(s["q"], s["kv"], s["layer"], s["prefix_table"], c["prefix"], s["table"], s["lens"])
    lp, entropy, top_lp, top_ids = ops.token_logprobs(s["logits"], s["tokens"], top=c["top"], temperature=c["temperature"])
    out = {"logprobs": lp, "entropy": entropy}
    if c["top"]:
        out["top_logprobs"], out["top_ids"] = top_lp, top_ids
    return out


def work(case):
    kind = case["kind"]
    if kind == "plan":
        rows, page = case["rows"], case["page"]
        tokens = rows * (1 - case["share"]) + rows * case["share"] * 0.75 * case["portion"]
        pages = tokens / page
        # lengths, pages and part-full pages in; table entries, four maps, offsets and lengths out
        return {"bytes": 4 * (2 * rows + pages + rows + pages + 4 * case["capacity"] + 2 * rows + 4), "flops": 8 * case["capacity"]}
    if kind == "release":
        rows, pages = case["rows"], case["rows"] * case["share"] * (0.75 * case["ctx"] / case["page"] + 0.5)
        return {"bytes": 9 * rows + 8 * pages + 8, "flops": 2 * pages}
    if kind == "prefix":
        b, h, kvh = case["b"], case["heads"], case["kv_heads"]
        per = 2 * kvh * (DIM + 4 if case["cache"] == "int8" else 2 * DIM)
        keys = case["prefix"] + b * 0.75 * case["ctx"]
        return {"bytes": keys * per + 4 * b * h * DIM, "flops": 4 * b * h * DIM * (case["prefix"] + 0.75 * case["ctx"])}
    n, v = case["n"], case["vocab"]
    return {"bytes": n * v * (4 if case["type"] == "f32" else 2) + n * (12 + 8 * case["top"]), "flops": 6 * n * v}


# ---- the definitions, in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "plan":
        return _exact_plan(case, s)
    if kind == "release":
        lens, table, free, done = (s[k].cpu().numpy() for k in ("lens", "table", "free", "done"))
        free, count = free.copy(), int(s["count"][0])
        for b in np.flatnonzero(done):
            for p in table[b, :-(-int(lens[b]) // case["page"])]:
                free[count] = p
                count += 1
        return {"free": free, "lens": np.where(done, 0, lens).astype(np.int32), "count": np.array([count], dtype=np.int32)}
    if kind == "prefix":
        return _exact_prefix(case, s)
    x = s["logits"].to(F64) / case["temperature"]
    p = torch.softmax(x, -1)
    logp = torch.log_softmax(x, -1)
    out = {"logprobs": logp[torch.arange(case["n"], device="cuda"), s["tokens"].long()], "entropy": -torch.xlogy(p, p).sum(-1)}
    if case["top"]:
        ids = torch.sort(s["logits"].to(F64), dim=-1, descending=True, stable=True).indices[:, :case["top"]]
        out["top_logprobs"], out["top_ids"] = torch.gather(logp, 1, ids), ids.to(torch.int32)
    return out


def _exact_plan(case, s):
    page, cap = case["page"], case["capacity"]
    lens, new, table, free = (s[k].cpu().numpy().copy() for k in ("lens", "new", "table", "free"))
    count = int(s["count"][0])
    pos, rows, pages, slots = np.zeros(cap, np.int32), np.full(cap, -1, np.int32), np.full(cap, -1, np.int32), np.zeros(cap, np.int32)
    offsets = [0]
    for b in range(len(lens)):
        a, n = int(lens[b]), int(new[b])
        for j in range(-(-a // page), -(-(a + n) // page)):
            count -= 1
            table[b, j] = free[count]
        p = np.arange(a, a + n)
        at = slice(offsets[-1], offsets[-1] + n)
        pos[at], rows[at], pages[at], slots[at] = p, b, table[b, p // page], p % page
        offsets.append(offsets[-1] + n)
    return {"positions": pos, "rows": rows, "pages": pages, "slots": slots, "offsets": np.array(offsets, np.int32), "lens": (lens + new).astype(np.int32),
            "count": np.array([count], np.int32), "status": np.zeros(1, np.int32), "table": table}


def _exact_prefix(case, s):
    b, h, kvh, page, pre = case["b"], case["heads"], case["kv_heads"], case["page"], case["prefix"]
    if 4.0 * b * h * DIM * pre > 8e10:
        return None
    lens, out = s["lens"].tolist(), torch.empty(b, h, DIM, dtype=F64, device="cuda")

    def keys(pages, kv, head, n):
        x = s["pool"][pages.long(), s["layer"], kv, head].to(F64)
        if "scales" in s:
            x = (x - 128) * s["scales"][pages.long(), s["layer"], kv, head].to(F64)[..., None]
        return x.reshape(-1, DIM)[:n]

    for head in range(kvh):
        kp, vp = keys(s["prefix_table"], 0, head, pre), keys(s["prefix_table"], 1, head, pre)
        for i in range(b):
            k, v = torch.cat([kp, keys(s["table"][i], 0, head, lens[i])]), torch.cat([vp, keys(s["table"][i], 1, head, lens[i])])
            g = slice(head * (h // kvh), (head + 1) * (h // kvh))
            out[i, g] = torch.softmax(s["q"][i, g].to(F64) @ k.T / math.sqrt(DIM), -1) @ v
    return out
