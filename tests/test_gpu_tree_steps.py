"""Steps of drafted tokens from end to end: plan, append, attention, logits, acceptance, and on with what was kept."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F64 = torch.float64
D, H, HKV, LAYERS, V = 128, 8, 2, 2, 24
G = H // HKV


@pytest.fixture(autouse=True)
def used_memory():
    """what is allocated next has been written before, so that an entry that a kernel leaves out shows"""
    if torch.cuda.is_available():
        kept = [torch.full((n // 4,), float("nan"), device="cuda") for n in [1 << 28] + [1 << 19] * 64]
        del kept


class Model:
    """Two layers of attention without anything between them; the second one's result, in float, gives the logits."""
    def __init__(self, seed, page, int8, B, room):
        from wf_bitnet import ops
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.emb, self.head = r(V, 256).to(torch.bfloat16), r(H * D, V).to(F64)
        self.qkv = [(r(256, (H + 2 * HKV) * D) / 16).to(torch.bfloat16) for _ in range(LAYERS)]
        self.back = (r(H * D, 256) / 32).to(torch.bfloat16)
        self.norms = [(torch.rand(D, generator=g, device="cuda") + 0.5).to(torch.bfloat16) for _ in range(2)]
        angle = torch.arange(room, device="cuda", dtype=F64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=F64) / D)
        self.cos, self.sin = torch.cos(angle).float(), torch.sin(angle).float()
        self.kv = ops.PagedKV(B * -(-room // page) + 5, LAYERS, HKV, page, D, dtype=torch.int8 if int8 else torch.bfloat16)
        if int8:
            self.kv.scales.fill_(math.nan)
        else:
            self.kv.pool.fill_(math.nan)

    def run(self, tokens, positions, plan, mask, table, lens):
        """(queries of the last layer, its result): every layer's keys and values are appended"""
        from wf_bitnet import ops
        x = self.emb[tokens.long()]
        for i in range(LAYERS):
            q = ops.norm_rope_kv_append(x @ self.qkv[i], H, self.kv, i, positions, plan.pages, plan.slots, self.cos, self.sin, q_norm=self.norms[0], k_norm=self.norms[1])
            o = ops.paged_tree_attn(q, self.kv, i, table, lens, plan.offsets, mask, out_dtype=torch.float32)
            x = x + o.reshape(-1, H * D).to(torch.bfloat16) @ self.back
        return q, o

    def cached(self, layer, table, n):
        """what the cache has of a sequence's first n tokens"""
        from wf_bitnet import ops
        page = self.kv.page_size
        at = torch.arange(n, device="cuda")
        k, v = (torch.empty(n, HKV, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        ops.kv_gather(self.kv, k, v, table[at // page].contiguous(), (at % page).to(torch.int32), layer)
        return k, v

    def exact(self, layer, table, n, which):
        page, at = self.kv.page_size, torch.arange(n, device="cuda")
        x = self.kv.pool[table[at // page].long(), layer, which, :, at % page].to(F64)
        if self.kv.dtype == torch.int8:
            x = (x - 128) * self.kv.scales[table[at // page].long(), layer, which, :, at % page].to(F64)[..., None]
        return x


def penalised(x, hist, prompt, drafts, rep, freq, pres):
    x = x.clone()
    for t in set(hist) | set(drafts):
        x[t] = x[t] / rep if x[t] > 0 else x[t] * rep
        drawn = (hist[prompt:] + drafts).count(t)
        if drawn:
            x[t] -= freq * drawn + pres
    return x


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("page, int8", [(16, False), (16, True), (64, False)])
def test_steps_of_drafts(page, int8, captured):
    """Every token kept is one that the model in 64 bits would have drawn behind those kept before it, or is nearer to it than the attention's roundings let tell; and after all steps
    the cache holds of every sequence what was appended for the tokens kept, in order, bit by bit."""
    from wf_bitnet import ops
    rng = torch.Generator().manual_seed(page + int8)
    prompts = [70, 1, 33, 16, 5]
    B, N, steps, room = len(prompts), 12, 7, 256
    m = Model(3, page, int8, B, room)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    lens, table = i32([0] * B), torch.full((B, room // page), -1, dtype=torch.int32, device="cuda")
    free, count = torch.randperm(m.kv.max_pages, generator=rng).to(torch.int32).cuda(), i32([m.kv.max_pages])
    rep, freq, pres = (torch.full((B,), x, device="cuda") for x in (1.2, 0.3, 0.2))
    hist = [torch.randint(0, V, (n,), generator=rng).tolist() for n in prompts]
    seen = [[([], []) for _ in range(LAYERS)] for _ in range(B)]      # keys and values kept so far

    # ---- the prompts: chains that are kept whole
    T = sum(prompts)
    plan = ops.paged_plan(lens, i32(prompts), table, free, count, page, T)
    tree = ops.tree_plan(i32([i - 1 for n in prompts for i in range(n)]), plan.offsets, lens, 128)
    assert int(plan.status) == 0 and torch.equal(tree.positions, plan.positions)
    _, o = m.run(i32(sum(hist, [])), tree.positions, plan, tree.mask, table, lens)
    last = (plan.offsets[1:] - 1).long()
    nxt = (o.reshape(T, -1).to(F64) @ m.head)[last].argmax(-1).to(torch.int32)
    lens, count = plan.lens.clone(), plan.free_count.clone()
    for b in range(B):
        for i in range(LAYERS):
            for kept, x in zip(seen[b][i], m.cached(i, table[b], prompts[b])):
                kept.append(x)

    # ---- the steps, on the same memory each time, so that one graph does for all
    T = B * N
    s = dict(lens=lens, count=count, nxt=nxt, tokens=i32([0] * T), parents=i32([0] * T), hist=torch.zeros(B, 256, dtype=torch.int32, device="cuda"), hl=i32([0] * B),
             allowed=torch.zeros(T, 1, dtype=torch.int32, device="cuda"))
    new, pl = i32([N] * B), i32(prompts)

    def step():
        plan = ops.paged_plan(s["lens"], new, table, free, s["count"], page, T)
        tree = ops.tree_plan(s["parents"], plan.offsets, s["lens"], 64)
        q, o = m.run(s["tokens"], tree.positions, plan, tree.mask, table, s["lens"])
        logits = (o.reshape(T, -1).to(F64) @ m.head).float()
        logits = ops.process_logits(logits, history=s["hist"], history_lens=s["hl"], prompt_lens=pl, repetition=rep, frequency=freq, presence=pres, allowed=s["allowed"], offsets=plan.offsets,
                                    node_tokens=s["tokens"], node_mask=tree.mask)
        targets = logits.argmax(-1).to(torch.int32)
        return plan, tree, q, logits, targets

    def accept(plan, targets):
        return ops.tree_accept(s["parents"], s["tokens"], targets, plan.offsets, s["lens"], m.kv, table, free, plan.free_count)

    graph, extra = None, 0
    for k in range(steps):
        parents = [[-1] + [int(torch.randint(max(0, i - 5), i, (1,), generator=rng)) for i in range(1, N)] for _ in range(B)]
        tokens = [[int(s["nxt"][b])] + torch.randint(0, V, (N - 1,), generator=rng).tolist() for b in range(B)]
        if k == 3:
            parents[2] = [i - 1 for i in range(N)]
        allowed = torch.randint(0, 1 << V, (T,), generator=rng) | torch.randint(0, 1 << V, (T,), generator=rng) | 1
        s["parents"].copy_(i32(sum(parents, [])))
        s["tokens"].copy_(i32(sum(tokens, [])))
        s["allowed"].copy_(allowed.to(torch.int32)[:, None])
        for b in range(B):
            s["hist"][b, :len(hist[b])] = i32(hist[b])
        s["hl"].copy_(i32([len(h) for h in hist]))
        before = s["lens"].tolist()
        if captured and graph is None:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                r = step()
            first = r
        if captured:
            graph.replay()
            r = first
        else:
            r = step()
        plan, tree, q, logits, targets = r
        assert int(plan.status) == 0 and plan.free_count.item() >= 0
        # against 64 bits, from the queries and the cache as they are
        for b in range(B):
            kk, vv = (m.exact(LAYERS - 1, table[b], before[b] + N, w) for w in (0, 1))
            qb = q[b * N:(b + 1) * N].to(F64)
            up = torch.zeros(N, N, dtype=torch.bool)
            for i in range(N):
                j = i
                while j >= 0:
                    up[i, j] = True
                    j = parents[b][j]
            hidden = torch.cat([torch.zeros(N, before[b], dtype=torch.bool), ~up], 1).cuda()
            kg, vg = (x.repeat_interleave(G, 1) for x in (kk, vv))
            sc = torch.einsum("nhd,shd->nhs", qb, kg) / math.sqrt(D)
            p = torch.softmax(sc.masked_fill(hidden[:, None], -math.inf), -1)
            want, mag = torch.einsum("nhs,shd->nhd", p, vg), torch.einsum("nhs,shd->nhd", p, vg.abs())
            # weights rounded to bf16; scores summed in float (130 half steps of sum |q k|, twice on a weight), 2^x to 2^-13 in weights and sum, sums of n weights and weighted values
            wide = 2 * 130 * 2.0**-24 * float(torch.einsum("nhd,shd->nhs", qb.abs(), kg.abs()).max()) / math.sqrt(D) + 2.0**-12 + 2 * kk.shape[0] * 2.0**-23
            off = ((2.0**-24 * want.abs() + (2.0**-8 + wide) * mag).reshape(N, -1) @ m.head.abs()) * 1.2
            raw = want.reshape(N, -1) @ m.head
            for i in range(N):
                here = [tokens[b][j] for j in range(N) if up[i, j]]
                x = penalised(raw[i], hist[b], prompts[b], here, 1.2, 0.3, 0.2)
                x[torch.tensor([not (int(allowed[b * N + i]) >> t & 1) for t in range(V)], device="cuda")] = -math.inf
                got = int(targets[b * N + i])
                # a logit in float: the product's own rounding and those of penalties, below 8 half steps of the parts
                slack = float(off[i].max()) + 8 * 2.0**-24 * (float(raw[i].abs().max()) * 1.2 + 8)
                assert float(x[got]) >= float(x.max()) - 2 * slack
        # what of the step's keys and values is to stay
        place = [[[x[before[b]:] for x in m.cached(i, table[b], before[b] + N)] for i in range(LAYERS)] for b in range(B)]
        a = accept(plan, targets)
        assert int(a.status) == 0
        for b in range(B):
            way = [0]
            while True:
                nexts = [j for j in range(N) if parents[b][j] == way[-1] and tokens[b][j] == int(targets[b * N + way[-1]])]
                if not nexts:
                    break
                way.append(nexts[0])
            assert int(a.accepted[b]) == len(way) and a.path[b * N:b * N + len(way)].tolist() == way and int(a.next_tokens[b]) == int(targets[b * N + way[-1]])
            hist[b] += [tokens[b][j] for j in way]
            extra += len(way) - 1
            for i in range(LAYERS):
                for kept, x in zip(seen[b][i], place[b][i]):
                    kept.append(x[way])
        for name, x in (("lens", a.lens), ("count", a.free_count), ("nxt", a.next_tokens)):
            s[name].copy_(x)
    assert extra > 0                                     # drafts were kept, not roots alone
    for b in range(B):
        n = int(s["lens"][b])
        assert n == len(hist[b])
        for i in range(LAYERS):
            for kept, x in zip(seen[b][i], m.cached(i, table[b], n)):
                assert torch.equal(torch.cat(kept), x)
    used = sum(-(-len(h) // page) for h in hist)
    assert int(s["count"]) == m.kv.max_pages - used
    pages = torch.cat([free[:int(s["count"])]] + [table[b, :-(-len(hist[b]) // page)] for b in range(B)])
    assert sorted(pages.tolist()) == list(range(m.kv.max_pages))      # none lost, none twice


def chain(seed, int8):
    """One step's calls over a state of its own, anew every time: all results, and the memory written in place"""
    from wf_bitnet import ops
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, N, page = 6, 20, 16
    T, blocks = B * N, 12
    kv = ops.PagedKV(B * blocks + 4, LAYERS, HKV, page, D, dtype=torch.int8 if int8 else torch.bfloat16)
    start = torch.randint(1, 255, kv.pool.shape, generator=g, device="cuda", dtype=torch.uint8) if int8 else torch.randn(kv.pool.shape, generator=g, device="cuda", dtype=torch.bfloat16)
    lens = torch.randint(1, 150, (B,), generator=g, device="cuda", dtype=torch.int32)
    table0 = torch.arange(B * blocks, dtype=torch.int32, device="cuda").view(B, blocks)
    new = torch.full((B,), N, dtype=torch.int32, device="cuda")
    parents = torch.cat([torch.tensor([-1] + [max(0, i - 3) for i in range(1, N)], dtype=torch.int32)] * B).cuda()
    tokens, targets = (torch.randint(0, 3, (T,), generator=g, device="cuda", dtype=torch.int32) for _ in range(2))
    qkv = torch.randn(T, (H + 2 * HKV) * D, generator=g, device="cuda").to(torch.bfloat16)
    angle = torch.rand(256, D // 2, generator=g, device="cuda")
    cos, sin = torch.cos(angle), torch.sin(angle)
    w = torch.randn(H * D, 1000, generator=g, device="cuda").to(torch.bfloat16)
    one = torch.full((B,), 1.25, device="cuda")
    hist = torch.randint(0, 1000, (B, 30), generator=g, device="cuda", dtype=torch.int32)
    table, free, count = table0.clone(), torch.empty(B * blocks, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")

    def run():
        kv.pool.copy_(start)
        if int8:
            kv.scales.fill_(0.02)
        table.copy_(table0)
        # (a plan of its own pages: as many as the drafts need are handed out first)
        need = (lens + N + page - 1) // page - (lens + page - 1) // page
        free.copy_(torch.arange(B * blocks - 1, -1, -1, dtype=torch.int32, device="cuda"))
        count.copy_(need.sum(dtype=torch.int32)[None])
        plan = ops.paged_plan(lens, new, table, free, count, page, T)
        tree = ops.tree_plan(parents, plan.offsets, lens, 64)
        q = ops.norm_rope_kv_append(qkv, H, kv, 1, tree.positions, plan.pages, plan.slots, cos, sin)
        o = ops.paged_tree_attn(q, kv, 1, table, lens, plan.offsets, tree.mask)
        x = ops.process_logits(o.reshape(T, -1) @ w, history=hist, repetition=one, frequency=one, presence=one, offsets=plan.offsets, node_tokens=tokens, node_mask=tree.mask)
        a = ops.tree_accept(parents, tokens, targets, plan.offsets, lens, kv, table, free, plan.free_count)
        kept = plan.offsets[-1:]
        return [*plan[:6], kept, *tree, q, o, x, a.accepted, a.next_tokens, a.lens, a.free_count, a.status, kv.pool, table, free]
    return run


def same(a, b):
    return len(a) == len(b) and all(u.dtype == v.dtype and torch.equal(u.nan_to_num() if u.is_floating_point() else u, v.nan_to_num() if v.is_floating_point() else v) for u, v in zip(a, b))


@pytest.mark.parametrize("int8", [False, True])
def test_the_same_through_ctypes(int8, monkeypatch):
    from wf_bitnet import _native
    run = chain(1, int8)
    want = [t.clone() for t in run()]
    monkeypatch.setattr(_native, "_ops", _native._Ctypes)
    assert same(want, run())


def test_calls_from_several_threads():
    """three threads with a stream each; the results are those of the calls one after another"""
    import threading
    runs = [chain(k, k == 1) for k in range(3)]
    want = [[t.clone() for t in r()] for r in runs]
    torch.cuda.synchronize()
    good, errors = [0] * 3, []

    def work(k):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(20):
                    got = runs[k]()
                    s.synchronize()
                    good[k] += same(want[k], got)
        except Exception as e:                           # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and good == [20] * 3


FIRST = """
import sys, torch
sys.path.insert(0, sys.argv[1])
from test_gpu_tree_steps import chain, same
run = chain(2, False)
x = torch.randn(8, 8, device="cuda", dtype=torch.bfloat16) @ torch.randn(8, 8, device="cuda", dtype=torch.bfloat16)       # (the matrix product's own set-up)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run()
for _ in range(2):
    graph.replay()
torch.cuda.synchronize()
have = [t.clone() for t in got]
assert same(have, run())
print("same")
"""


def test_first_calls_inside_a_capture(tmp_path):
    """a fresh process whose first calls of these are captured"""
    import os
    import subprocess
    import sys
    r = subprocess.run([sys.executable, "-c", FIRST, os.path.dirname(os.path.abspath(__file__))], capture_output=True, text=True, timeout=300, cwd=tmp_path,
                       env=dict(os.environ, PYTHONPATH=os.pathsep.join(sys.path)))
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]
