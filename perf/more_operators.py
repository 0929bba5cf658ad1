"""Operators of a step that verifies drafted tokens, as cases that can be timed and compared: masks and positions of a tree of drafts, queries and keys normed,
rotated and appended to the paged cache, attention of the tree's tokens over the cache, penalties, biases and grammar masks on their logits, and the acceptance of
a path with the cache closed up behind it.

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
EPS = 1e-6


def listed():
    return [
        # the trees of eight sequences, up to 60 drafts each (the smallest call, latency alone)
        {"name": "plan_8_trees", "kind": "plan", "b": 8, "nodes": 60, "ctx": 4096},
        # 256 wide trees, four words of mask a token
        {"name": "plan_256_trees", "kind": "plan", "b": 256, "nodes": 256, "ctx": 4096},
        # a decode batch into the 8-bit cache, 2B heads
        {"name": "append_64_int8", "kind": "append", "t": 64, "heads": 20, "kv_heads": 5, "page": 16, "cache": "int8", "rot": 128, "pairs": False, "norm": True},
        # prompts, 8B heads
        {"name": "append_prompts_16384", "kind": "append", "t": 16384, "heads": 32, "kv_heads": 8, "page": 16, "cache": "bf16", "rot": 128, "pairs": False, "norm": True},
        # one sequence verifies a tree over a context of up to 4096, 2B heads
        {"name": "attn_1_60", "kind": "attn", "b": 1, "nodes": 60, "heads": 20, "kv_heads": 5, "ctx": 4096, "page": 16, "cache": "bf16"},
        # a batch with small trees, 8B heads
        {"name": "attn_48_12", "kind": "attn", "b": 48, "nodes": 12, "heads": 32, "kv_heads": 8, "ctx": 4096, "page": 16, "cache": "bf16"},
        # wide trees over long contexts, 70B heads: as much arithmetic as a prompt (the largest)
        {"name": "attn_8_250", "kind": "attn", "b": 8, "nodes": 250, "heads": 64, "kv_heads": 8, "ctx": 16384, "page": 64, "cache": "bf16"},
        # odd sizes over the 8-bit cache
        {"name": "attn_31_25_int8", "kind": "attn", "b": 31, "nodes": 25, "heads": 32, "kv_heads": 8, "ctx": 8000, "page": 48, "cache": "int8"},
        # one sequence's next token: penalties over a long history, and biases
        {"name": "logits_1", "kind": "logits", "b": 1, "nodes": 1, "vocab": 128256, "type": "f32", "history": 4096, "bias": 20, "masked": 0.0},
        # the trees of 32 sequences, each token's own past penalised, under a grammar
        {"name": "logits_32_trees", "kind": "logits", "b": 32, "nodes": 60, "vocab": 128256, "type": "bf16", "history": 2000, "bias": 20, "masked": 0.33},
        # eight sequences accept what they agree with, 2B cache of 30 layers
        {"name": "accept_8", "kind": "accept", "b": 8, "nodes": 60, "heads": 20, "kv_heads": 5, "layers": 30, "ctx": 256, "page": 16},
        # 64 sequences, 8B cache of 32 layers
        {"name": "accept_64", "kind": "accept", "b": 64, "nodes": 60, "heads": 32, "kv_heads": 8, "layers": 32, "ctx": 100, "page": 16},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("plan", "append", "attn", "attn", "logits", "accept"))
    if kind == "plan":
        return {"kind": kind, "b": _log(rng, 1, 256), "nodes": _log(rng, 1, 256), "ctx": _log(rng, 1, 16384)}
    heads, kv_heads = rng.choice(HEADS)
    if kind == "append":
        t = _log(rng, 1, 16384 * 48 // (heads + 2 * kv_heads))
        return {"kind": kind, "t": min(t, 16384), "heads": heads, "kv_heads": kv_heads, "page": rng.choice((16, 16, 32, 48, 64, 7)), "cache": rng.choice(("bf16", "bf16", "int8")),
                "rot": rng.choice((128, 128, 64, 32)), "pairs": rng.choice((False, False, True)), "norm": rng.choice((True, True, False))}
    if kind == "attn":
        nodes = _log(rng, 1, 256)
        b = _log(rng, 1, 64)
        ctx = _log(rng, 16, max(17, min(16384, 8 * 250 * 16384 * 64 // (b * nodes * heads))))
        return {"kind": kind, "b": b, "nodes": nodes, "heads": heads, "kv_heads": kv_heads, "ctx": min(ctx, 1200000 // b), "page": rng.choice((16, 16, 32, 48, 64, 128)),
                "cache": rng.choice(("bf16", "bf16", "int8"))}
    if kind == "logits":
        vocab = rng.choice(VOCABS + (_log(rng, 100, 128256) | 1,))
        nodes = rng.choice((1, 1, _log(rng, 2, 64)))
        return {"kind": kind, "b": _log(rng, 1, max(1, min(256, 32 * 60 * 128256 // (nodes * max(vocab, 8000))))), "nodes": nodes, "vocab": vocab,
                "type": rng.choice(("f32", "bf16", "f16")), "history": _log(rng, 1, 4096), "bias": rng.choice((0, 1, 20, 100)), "masked": rng.choice((0.0, 0.33))}
    heads, kv_heads = rng.choice(HEADS[:2])
    b, layers = _log(rng, 1, 64), rng.choice((2, 30, 32))
    return {"kind": kind, "b": b, "nodes": _log(rng, 1, 60), "heads": heads, "kv_heads": kv_heads, "layers": layers, "ctx": _log(rng, 1, 200), "page": rng.choice((16, 16, 32, 7))}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32)


def _lengths(g, n, hi):
    """n lengths from a half of `hi` to `hi`"""
    return _ints(g, max(1, hi // 2), hi + 1, n)


def _trees(g, b, nodes):
    """Drafts one sequence after another in buffers for b * nodes of them: how many each has, where they start, and of each the draft that it follows (-1: the
    first one, which is the token drawn last)."""
    n = _lengths(g, b, nodes)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int32, device="cuda"), torch.cumsum(n, 0).to(torch.int32)])
    i = torch.arange(nodes, device="cuda", dtype=torch.int32)
    up = torch.where(i > 0, (i - 1 - _ints(g, 0, 8, b, nodes)).clamp(min=0), -1)
    row, at, live = _places(offsets, b * nodes)
    return n, offsets, torch.where(live, up[row, at.clamp(max=nodes - 1)], -1).to(torch.int32)


def _places(offsets, t):
    """of each of t rows: its sequence, its place there, and whether it has one"""
    k = torch.arange(t, device="cuda")
    row = torch.searchsorted(offsets[1:].long(), k, right=True)
    live = row < offsets.shape[0] - 1
    row = row.clamp(max=offsets.shape[0] - 2)
    return row, torch.where(live, k - offsets[row], 0), live


def _padded(x, offsets, nodes, fill):
    """rows one after another -> [sequences, nodes, ...]"""
    i = torch.arange(nodes, device="cuda")
    y = x[(offsets[:-1, None] + i).clamp(max=x.shape[0] - 1).long()]
    keep = i < (offsets[1:] - offsets[:-1])[:, None]
    return torch.where(keep.view(*keep.shape, *(1,) * (y.dim() - 2)), y, fill)


def _reach(parents, offsets, nodes):
    """[sequences, nodes, nodes]: 1 where a draft is the other one or follows it, by doubling the steps looked over; drafts that are none reach themselves"""
    up = _padded(parents, offsets, nodes, -1)
    r = (up[:, :, None] == torch.arange(nodes, device="cuda")).float() + torch.eye(nodes, device="cuda")
    for _ in range(max(1, (nodes - 1).bit_length())):
        r = torch.matmul(r, r).clamp(max=1.0)
    return r


def _words(bits):
    """[..., n] of 0 and 1 -> int64 [..., ceil(n / 64)]"""
    w = -(-bits.shape[-1] // 64)
    bits = torch.nn.functional.pad(bits.long(), (0, 64 * w - bits.shape[-1])).view(*bits.shape[:-1], w, 64)
    return (bits << torch.arange(64, device="cuda")).sum(-1)


def _tree_masks(parents, offsets, nodes):
    r = _reach(parents, offsets, nodes)
    row, at, live = _places(offsets, parents.shape[0])
    return torch.where(live[:, None], _words(r)[row, at], 0), torch.where(live, r.sum(-1)[row, at] - 1, 0.0).long(), row, live


def _pages(g, b, tokens, page, spare):
    """tables for `tokens` tokens a sequence in the order of a shuffled pool, and the pages that are left"""
    blocks = -(-tokens // page)
    order = torch.randperm(b * blocks + spare, generator=g, device="cuda").to(torch.int32)
    return order[:b * blocks].view(b, blocks).contiguous(), order


def _pool(g, shape, cache):
    if cache == "int8":                                # codes are kept as code + 128
        return torch.randint(1, 256, shape, generator=g, device="cuda", dtype=torch.uint8), torch.rand(shape[:-1], generator=g, device="cuda") * 0.01 + 0.015
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16), None


def _inputs(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    s = {"case": case}
    if kind == "append":
        t, heads, kvh, page = case["t"], case["heads"], case["kv_heads"], case["page"]
        blocks = -(-t // page)
        order = torch.randperm(blocks + 3, generator=g, device="cuda").to(torch.int32)
        k = torch.arange(t, device="cuda")
        s["pool"], s["scales"] = _pool(g, (blocks + 3, 2, 2, kvh, page, DIM), case["cache"])
        s["pages"], s["slots"] = order[k // page].contiguous(), (k % page).to(torch.int32)
        s["qkv"] = (torch.randn(t, (heads + 2 * kvh) * DIM, generator=g, device="cuda") * 1.5).to(torch.bfloat16)
        s["positions"] = _ints(g, 0, 8192, t)
        angle = torch.arange(8192, device="cuda", dtype=F64)[:, None] * 500000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=F64) / case["rot"])
        s["cos"], s["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
        for name in ("q_norm", "k_norm"):
            s[name] = (torch.rand(DIM, generator=g, device="cuda") + 0.5).to(torch.bfloat16) if case["norm"] else None
        s["layer"] = 1
        return s
    b, nodes = case["b"], case["nodes"]
    t = b * nodes
    if kind == "logits":
        v = case["vocab"]
        n, s["offsets"], s["parents"] = _trees(g, b, nodes)
        x = torch.randn(t, v, generator=g, device="cuda") * 2.5
        s["logits"] = x.to(TYPES[case["type"]])
        often = lambda *shape: (torch.rand(shape, generator=g, device="cuda") ** 3 * v).to(torch.int32).clamp(max=v - 1)  # noqa: E731
        s["history"], s["history_lens"] = often(b, case["history"]), _lengths(g, b, case["history"])
        s["prompt_lens"] = (s["history_lens"] * torch.rand(b, generator=g, device="cuda")).to(torch.int32)
        s["repetition"] = 1 + 0.3 * torch.rand(b, generator=g, device="cuda")
        s["frequency"], s["presence"] = (0.5 * torch.rand(b, generator=g, device="cuda") for _ in range(2))
        s["bias_ids"] = often(b, case["bias"]) if case["bias"] else None
        s["bias_values"] = torch.randn(b, case["bias"], generator=g, device="cuda") * 4 if case["bias"] else None
        s["allowed"] = None
        if case["masked"]:
            rows = torch.rand(t, 1, generator=g, device="cuda") < case["masked"]
            pad = -(-v // 32) * 32 - v
            ok = torch.nn.functional.pad(~rows | (torch.rand(t, v, generator=g, device="cuda") < 100.0 / v), (0, pad)).view(t, -1, 32)
            s["allowed"] = (ok.int() << torch.arange(32, device="cuda", dtype=torch.int32)).sum(-1, dtype=torch.int32)
        s["node_tokens"] = s["mask"] = None
        if nodes > 1:
            s["node_tokens"] = often(t)
            s["mask"] = _tree_masks(s["parents"], s["offsets"], nodes)[0]
        return s
    s["lens"] = _lengths(g, b, case["ctx"])
    n, s["offsets"], s["parents"] = _trees(g, b, nodes)
    if kind == "plan":
        return s
    heads, kvh, page = case["heads"], case["kv_heads"], case["page"]
    layers = case.get("layers", 2)
    s["table"], order = _pages(g, b, case["ctx"] + nodes, page, 5)
    s["pool"], s["scales"] = _pool(g, (order.shape[0], layers, 2, kvh, page, DIM), case.get("cache", "bf16"))
    if kind == "attn":
        s["q"] = torch.randn(t, heads, DIM, generator=g, device="cuda").to(torch.bfloat16)
        s["mask"] = _tree_masks(s["parents"], s["offsets"], nodes)[0]
        s["layer"] = 1
        return s
    # what the model draws behind each draft: often one of the drafts that follow it
    s["tokens"], s["targets"] = _ints(g, 0, 32000, t), _ints(g, 0, 32000, t)
    row, at, live = _places(s["offsets"], t)
    under = torch.where(live & (s["parents"] >= 0), s["offsets"][row] + s["parents"], t).long()
    child = torch.full((t + 1,), -1, device="cuda").scatter_reduce(0, under, torch.arange(t, device="cuda"), "amax")[:t]
    follow = (child >= 0) & (torch.rand(t, generator=g, device="cuda") < 0.7)
    s["targets"] = torch.where(follow, s["tokens"][child.clamp(min=0)], s["targets"])
    s["free"] = torch.full((order.shape[0],), -1, dtype=torch.int32, device="cuda")
    s["free"][:5] = order[-5:]
    s["count"] = torch.tensor([5], dtype=torch.int32, device="cuda")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and "pool" in s:                            # the handle on the cache that a program keeps
        from wf_bitnet import ops
        pool, scales = s.pop("pool"), s.pop("scales")
        s["kv"] = ops.PagedKV(pool.shape[0], pool.shape[1], pool.shape[3], pool.shape[4], DIM, dtype=torch.bfloat16 if scales is None else torch.int8)
        s["kv"].pool.copy_(pool)
        if scales is not None:
            s["kv"].scales.copy_(scales)
    return s


# ---- the plain forms
def _plan(s):
    mask, depth, row, live = _tree_masks(s["parents"], s["offsets"], s["case"]["nodes"])
    return {"mask": mask, "positions": torch.where(live, s["lens"][row] + depth, 0).to(torch.int32)}


def _append(s):
    c = s["case"]
    t, h, kvh, rot = c["t"], c["heads"], c["kv_heads"], c["rot"]
    x = s["qkv"].float().view(t, h + 2 * kvh, DIM)
    q, k, v = x[:, :h], x[:, h:h + kvh], x[:, h + kvh:]
    if c["norm"]:
        norm = lambda y, gain: y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * gain.float()  # noqa: E731
        q, k = norm(q, s["q_norm"]), norm(k, s["k_norm"])
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]

    def turn(y):
        if c["pairs"]:
            a, b = y[..., 0:rot:2], y[..., 1:rot:2]
            return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), y[..., rot:]], -1)
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, y[..., rot:]], -1)

    q, k = turn(q).to(torch.bfloat16), turn(k).to(torch.bfloat16)
    pages, slots, layer = s["pages"].long(), s["slots"].long(), s["layer"]
    if c["cache"] == "bf16":
        s["pool"][pages, layer, 0, :, slots], s["pool"][pages, layer, 1, :, slots] = k, v.to(torch.bfloat16)
        return {"q": q, "pool": s["pool"]}
    out = {"q": q}
    for kv, y in enumerate((k.float(), v)):
        top = y.abs().amax(-1)
        top = torch.where(top < 1e-6, 1.0, top)
        codes = torch.round(y * (127.0 / top)[..., None]).clamp(-127, 127)
        s["pool"][pages, layer, kv, :, slots] = (codes + 128).to(torch.uint8)
        s["scales"][pages, layer, kv, :, slots] = top / 127.0
        held = s["pool"][pages, layer, kv, :, slots].float() - 128.0
        out["k" if kv == 0 else "v"] = (held * s["scales"][pages, layer, kv, :, slots][..., None]).to(torch.bfloat16).view(t, -1)
    return out


def _rows_of(s, kv):
    """[sequences, kv heads, tokens, DIM] in float of the pages that the tables name"""
    table = s["table"].long()
    x = s["pool"][table, s["layer"], kv].float()
    if s["scales"] is not None:
        x = (x - 128.0) * s["scales"][table, s["layer"], kv][..., None]
    x = x.transpose(1, 2)                              # [b, kv heads, blocks, page, DIM]
    return x.reshape(x.shape[0], x.shape[1], -1, DIM)


def _attn(s):
    c = s["case"]
    b, nodes, h, kvh = c["b"], c["nodes"], c["heads"], c["kv_heads"]
    offsets, lens = s["offsets"].long(), s["lens"].long()
    k, v = _rows_of(s, 0), _rows_of(s, 1)
    q = _padded(s["q"], offsets, nodes, 0).float().view(b, nodes, kvh, h // kvh, DIM).transpose(1, 2).reshape(b, kvh, -1, DIM) / math.sqrt(DIM)
    sc = torch.matmul(q, k.transpose(2, 3)).view(b, kvh, nodes, h // kvh, -1)
    rel = torch.arange(k.shape[2], device="cuda") - lens[:, None]                                # [b, keys]: place among the drafts
    words = _padded(s["mask"], offsets, nodes, 0)
    word = torch.gather(words, 2, (rel.clamp(0, 64 * words.shape[2] - 1) // 64)[:, None].expand(-1, nodes, -1))
    sees = (rel < 0)[:, None] | (((word >> (rel % 64)[:, None]) & 1).bool() & ((rel >= 0) & (rel < (offsets[1:] - offsets[:-1])[:, None]))[:, None])
    sc = torch.where(sees[:, None, :, None], sc, -math.inf)
    top = sc.amax(-1, keepdim=True)
    e = torch.exp(sc - torch.where(top == -math.inf, 0.0, top))
    o = torch.matmul(e.view(b, kvh, -1, k.shape[2]), v).view(b, kvh, nodes, -1, DIM) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    row, at, live = _places(offsets, s["q"].shape[0])
    return torch.where(live[:, None, None], o.transpose(1, 2)[row, at].reshape(-1, h, DIM), 0.0).to(torch.bfloat16)


def _counts(ids, weights, vocab):
    """[rows, vocab] of the weights summed over the ids; ids of -1 are none"""
    return torch.zeros(ids.shape[0], vocab + 1, device="cuda").scatter_add_(1, torch.where(ids >= 0, ids, vocab).long(), weights)[:, :vocab]


def _logits(s):
    c = s["case"]
    v, nodes = c["vocab"], c["nodes"]
    row, _, live = _places(s["offsets"], s["logits"].shape[0])
    k = torch.arange(s["history"].shape[1], device="cuda")
    there = k < s["history_lens"][:, None]
    ids = torch.where(there, s["history"], -1)
    seen, count = _counts(ids, there.float(), v)[row], _counts(ids, (there & (k >= s["prompt_lens"][:, None])).float(), v)[row]
    if nodes > 1:                                      # a draft's own past
        mine = ((s["mask"][:, :, None] >> torch.arange(64, device="cuda")) & 1).flatten(1)[:, :nodes].bool()
        ids = torch.where(mine, _padded(s["node_tokens"], s["offsets"], nodes, -1)[row], -1)
        past = _counts(ids, mine.float(), v)
        seen, count = seen + past, count + past
    x = s["logits"].float()
    per = lambda name: s[name][row][:, None]  # noqa: E731
    y = torch.where(seen > 0, torch.where(x > 0, x / per("repetition"), x * per("repetition")), x)
    y = y - (per("frequency") * count + per("presence") * (count > 0))
    if s["bias_ids"] is not None:                      # the last entry of an id counts
        n = s["bias_ids"].shape[1]
        last = torch.zeros(c["b"], v, device="cuda").scatter_reduce(1, s["bias_ids"].long(), torch.arange(1, n + 1, device="cuda").float().expand(c["b"], n), "amax").long()
        bias = torch.where(last > 0, torch.gather(s["bias_values"], 1, (last - 1).clamp(min=0)), 0.0)
        y = y + bias[row]
    if s["allowed"] is not None:
        at = torch.arange(v, device="cuda")
        y = torch.where(((s["allowed"][:, at // 32] >> (at % 32)) & 1).bool(), y, -math.inf)
    return torch.where(live[:, None], y, x).to(s["logits"].dtype)


def _accept(s):
    c = s["case"]
    b, nodes, page = c["b"], c["nodes"], c["page"]
    t = b * nodes
    offsets, lens, table = s["offsets"].long(), s["lens"].long(), s["table"]
    n = offsets[1:] - offsets[:-1]
    up, tok, want = (_padded(s[k], offsets, nodes, fill).long() for k, fill in (("parents", -1), ("tokens", -1), ("targets", -2)))
    i = torch.arange(nodes, device="cuda")
    # a draft fits where it is what was drawn behind its parent, and the first of its siblings that is; it is kept where all up to the first one fit
    key = torch.where((up >= 0) & (i < n[:, None]), up * (1 << 20) + tok, -1 - i)
    twin = ((key[:, :, None] == key[:, None]) & (i < i[:, None])).any(-1)
    fits = (i == 0) | ((up >= 0) & (tok == torch.gather(want, 1, up.clamp(min=0))) & ~twin)
    kept = (torch.matmul(_reach(s["parents"], offsets, nodes), (~fits).float()[..., None])[..., 0] == 0) & (i < n[:, None])
    rank = torch.cumsum(kept, 1)
    accepted = rank[:, -1]
    path = torch.full((b, nodes + 1), -1, device="cuda").scatter(1, torch.where(kept, rank - 1, nodes), i.expand(b, nodes))[:, :nodes]
    row, at, live = _places(offsets, t)
    last = torch.gather(path, 1, (accepted - 1)[:, None])
    # the kept tokens' keys and values move up behind the cached ones; entries that stay where they are (or are none) are written as they stand
    stay = torch.where(path >= 0, path, i)
    src, dst = lens[:, None] + stay, lens[:, None] + i
    live_dst = dst < (lens + n)[:, None]
    src, dst = torch.where(live_dst, src, lens[:, None]), torch.where(live_dst, dst, lens[:, None])
    where = lambda p: (torch.gather(table.long(), 1, p // page), p % page)  # noqa: E731
    moved = s["pool"][where(src)[0], :, :, :, where(src)[1]]
    s["pool"][where(dst)[0], :, :, :, where(dst)[1]] = moved
    # pages behind the last kept token go back on the list
    have, old = (lens + accepted + page - 1) // page, (lens + n + page - 1) // page
    end = torch.cumsum(old - have, 0)
    k = torch.arange(s["free"].shape[0], device="cuda") - s["count"]
    r = torch.searchsorted(end, k, right=True).clamp(max=b - 1)
    j = (have[r] + k - (end - (old - have))[r]).clamp(0, table.shape[1] - 1)
    free = torch.where((k >= 0) & (k < end[-1]), table[r, j], s["free"])
    i32 = lambda x: x.to(torch.int32)  # noqa: E731
    return {"accepted": i32(accepted), "path": i32(torch.where(live, path[row, at], -1)), "next": i32(torch.gather(want, 1, last)[:, 0]), "lens": i32(lens + accepted),
            "count": i32(s["count"] + end[-1]), "free": free, "status": torch.zeros(1, dtype=torch.int32, device="cuda"), "pool": s["pool"]}


def run(s):
    c = s["case"]
    kind = c["kind"]
    if not own:
        return {"plan": _plan, "append": _append, "attn": _attn, "logits": _logits, "accept": _accept}[kind](s)
    from wf_bitnet import ops
    if kind == "plan":
        p = ops.tree_plan(s["parents"], s["offsets"], s["lens"], max_nodes=c["nodes"])
        return {"mask": p.mask, "positions": p.positions}
    if kind == "append":
        q = ops.norm_rope_kv_append(s["qkv"], c["heads"], s["kv"], s["layer"], s["positions"], s["pages"], s["slots"], s["cos"], s["sin"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS,
                                    interleaved=c["pairs"])
        if c["cache"] == "bf16":
            return {"q": q, "pool": s["kv"].pool}
        k, v = (torch.empty(c["t"], c["kv_heads"] * DIM, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        ops.kv_gather(s["kv"], k, v, s["pages"], s["slots"], s["layer"])                         # what the cache now holds
        return {"q": q, "k": k, "v": v}
    if kind == "attn":
        return ops.paged_tree_attn(s["q"], s["kv"], s["layer"], s["table"], s["lens"], s["offsets"], s["mask"])
    if kind == "logits":
        return ops.process_logits(s["logits"], history=s["history"], history_lens=s["history_lens"], prompt_lens=s["prompt_lens"], repetition=s["repetition"], frequency=s["frequency"],
                                  presence=s["presence"], bias_ids=s["bias_ids"], bias_values=s["bias_values"], allowed=s["allowed"], offsets=s["offsets"], node_tokens=s["node_tokens"],
                                  node_mask=s["mask"])
    a = ops.tree_accept(s["parents"], s["tokens"], s["targets"], s["offsets"], s["lens"], s["kv"], s["table"], s["free"], s["count"])
    return {"accepted": a.accepted, "path": a.path, "next": a.next_tokens, "lens": a.lens, "count": a.free_count, "free": s["free"], "status": a.status, "pool": s["kv"].pool}


def work(case):
    kind = case["kind"]
    if kind == "append":
        t, h, kvh = case["t"], case["heads"], case["kv_heads"]
        held = kvh * 2 * (DIM + 4 if case["cache"] == "int8" else 2 * DIM)
        back = kvh * 8 * DIM if case["cache"] == "int8" else 0
        return {"bytes": t * (2 * DIM * (h + 2 * kvh) + 2 * DIM * h + held + back + 12) + min(t, 8192) * 4 * case["rot"], "flops": t * (h + kvh) * DIM * 7}
    b, nodes = case["b"], case["nodes"]
    t, n = b * nodes, b * 0.75 * nodes
    if kind == "plan":
        return {"bytes": 4 * t + 12 * b + t * (8 * -(-nodes // 64) + 4), "flops": 4 * t}
    if kind == "attn":
        h, kvh = case["heads"], case["kv_heads"]
        per = 2 * kvh * (DIM + 4 if case["cache"] == "int8" else 2 * DIM)
        keys = 0.75 * (case["ctx"] + nodes)
        return {"bytes": b * keys * per + n * h * DIM * 2 + t * h * DIM * 2 + n * 8 * -(-nodes // 64), "flops": 4 * n * h * DIM * 0.75 * (case["ctx"] + 0.1 * nodes)}
    if kind == "logits":
        v, size = case["vocab"], 4 if case["type"] == "f32" else 2
        return {"bytes": 2 * t * v * size + (t * v / 8 if case["masked"] else 0) + b * (3 * case["history"] + 8 * case["bias"] + 24) + (12 * t if nodes > 1 else 0), "flops": 4 * t * v}
    # of the drafts kept behind the first one about two a sequence move (a third of the sequences keep none)
    return {"bytes": 12 * t + 4 * t + 24 * b + 2 * 2.0 * b * case["layers"] * 2 * case["kv_heads"] * DIM * 2 * min(1.0, nodes / 12), "flops": 4 * t}


# ---- the definitions, in 64 bits
def _paths(s):
    """of every row: the places of the drafts up to it, itself last"""
    off, up = s["offsets"].tolist(), s["parents"].tolist()
    out = []
    for b in range(len(off) - 1):
        mine = []
        for i in range(off[b + 1] - off[b]):
            u = up[off[b] + i]
            mine.append((mine[u] if u >= 0 else []) + [i])
        out += mine
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    return {"plan": _exact_plan, "append": _exact_append, "attn": _exact_attn, "logits": _exact_logits, "accept": _exact_accept}[case["kind"]](case, s)


def _exact_plan(case, s):
    w = -(-case["nodes"] // 64)
    t = case["b"] * case["nodes"]
    mask, positions = np.zeros((t, w), np.uint64), np.zeros(t, np.int32)
    row = np.searchsorted(s["offsets"].cpu().numpy()[1:], np.arange(t), side="right")
    lens = s["lens"].cpu().numpy()
    for k, path in enumerate(_paths(s)):
        for i in path:
            mask[k, i // 64] |= np.uint64(1 << (i % 64))
        positions[k] = lens[row[k]] + len(path) - 1
    return {"mask": mask.view(np.int64), "positions": positions}


def _exact_append(case, s):
    t, h, kvh, rot = case["t"], case["heads"], case["kv_heads"], case["rot"]
    x = s["qkv"].to(F64).reshape(t, h + 2 * kvh, DIM)
    for part, gain in ((slice(0, h), s["q_norm"]), (slice(h, h + kvh), s["k_norm"])):
        if gain is not None:
            x[:, part] *= gain.to(F64) / torch.sqrt(x[:, part].square().mean(-1, keepdim=True) + EPS)
    z = torch.complex(s["cos"].to(F64), s["sin"].to(F64))[s["positions"].long()][:, None]
    y = x[:, :h + kvh]
    one, two = (slice(0, rot, 2), slice(1, rot, 2)) if case["pairs"] else (slice(0, rot // 2), slice(rot // 2, rot))
    turned = torch.complex(y[..., one], y[..., two]) * z
    y[..., one], y[..., two] = turned.real, turned.imag
    q, k, v = x[:, :h], x[:, h:h + kvh], x[:, h + kvh:]
    if case["cache"] == "int8":                        # the codes' borders are not those of 64 bits
        return {"q": q, "k": None, "v": None}
    pool = s["pool"].to(F64)
    for kv, y in ((0, k), (1, v)):
        pool[s["pages"].long(), s["layer"], kv, :, s["slots"].long()] = y
    return {"q": q, "pool": pool}


def _exact_attn(case, s):
    h, kvh = case["heads"], case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=F64, device="cuda")
    off, lens, paths = s["offsets"].tolist(), s["lens"].tolist(), _paths(s)
    for b in range(case["b"]):
        a, e, n = off[b], off[b + 1], lens[b] + off[b + 1] - off[b]
        hidden = torch.ones(e - a, n, dtype=torch.bool)
        hidden[:, :lens[b]] = False
        for i in range(e - a):
            hidden[i, [lens[b] + j for j in paths[a + i]]] = False
        hidden = hidden.cuda()
        for head in range(kvh):
            kv = []
            for which in (0, 1):
                x = s["pool"][s["table"][b].long(), s["layer"], which, head].to(F64)
                if s["scales"] is not None:
                    x = (x - 128) * s["scales"][s["table"][b].long(), s["layer"], which, head].to(F64)[..., None]
                kv.append(x.reshape(-1, DIM)[:n])
            g = slice(head * (h // kvh), (head + 1) * (h // kvh))
            p = torch.softmax((s["q"][a:e, g].to(F64) @ kv[0].T / math.sqrt(DIM)).masked_fill(hidden[:, None], -math.inf), -1)
            out[a:e, g] = p @ kv[1]
    return out


def _exact_logits(case, s):
    v = case["vocab"]
    out = s["logits"].to(F64)
    off, lens, prompts = (s[k].tolist() for k in ("offsets", "history_lens", "prompt_lens"))
    paths = _paths(s)
    for b in range(case["b"]):
        hist = s["history"][b, :lens[b]].long()
        for t in range(off[b], off[b + 1]):
            past = hist[:0] if case["nodes"] == 1 else s["node_tokens"][[off[b] + i for i in paths[t]]].long()
            ids, n = torch.unique(torch.cat([hist[prompts[b]:], past]), return_counts=True)
            every = torch.unique(torch.cat([hist, past]))
            x = out[t]
            r = s["repetition"][b].to(F64)
            x[every] = torch.where(x[every] > 0, x[every] / r, x[every] * r)
            x[ids] -= s["frequency"][b].to(F64) * n + s["presence"][b].to(F64)
        if s["bias_ids"] is not None:
            last = dict(zip(s["bias_ids"][b].tolist(), s["bias_values"][b].tolist()))
            out[off[b]:off[b + 1], list(last)] += torch.tensor(list(last.values()), dtype=F64, device="cuda")
    if s["allowed"] is not None:
        for t in range(off[-1]):
            bits = np.unpackbits(s["allowed"][t].cpu().numpy().view(np.uint8), bitorder="little")[:v].astype(bool)
            out[t].masked_fill_(~torch.from_numpy(bits).cuda(), -math.inf)
    return out


def _exact_accept(case, s):
    page = case["page"]
    off, lens, table = s["offsets"].tolist(), s["lens"].tolist(), s["table"].cpu().numpy()
    up, tok, want = (s[k].tolist() for k in ("parents", "tokens", "targets"))
    free, count = s["free"].cpu().numpy().copy(), int(s["count"][0])
    t = case["b"] * case["nodes"]
    path, accepted, nxt, new = np.full(t, -1, np.int32), [], [], []
    src, dst = [], []
    for b in range(case["b"]):
        a, n, cur, kept = off[b], off[b + 1] - off[b], 0, [0]
        while True:
            follows = [j for j in range(n) if up[a + j] == cur and tok[a + j] == want[a + cur]]
            if not follows:
                break
            cur = follows[0]
            kept.append(cur)
        path[a:a + len(kept)] = kept
        accepted.append(len(kept))
        nxt.append(want[a + cur])
        new.append(lens[b] + len(kept))
        for k, j in enumerate(kept):
            src.append((int(table[b, (lens[b] + j) // page]), (lens[b] + j) % page))
            dst.append((int(table[b, (lens[b] + k) // page]), (lens[b] + k) % page))
        for j in range(-(-new[-1] // page), -(-(lens[b] + n) // page)):
            free[count] = table[b, j]
            count += 1
    pool = s["pool"]
    at = lambda x: [torch.tensor(y, device="cuda") for y in zip(*x)]  # noqa: E731
    (sp, ss), (dp, ds) = at(src), at(dst)
    pool[dp, :, :, :, ds] = pool[sp, :, :, :, ss].clone()
    i32 = lambda x: np.array(x, np.int32)  # noqa: E731
    return {"accepted": i32(accepted), "path": path, "next": i32(nxt), "lens": i32(new), "count": i32([count]), "free": free, "status": i32([0]), "pool": pool.to(F64)}
