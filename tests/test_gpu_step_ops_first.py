"""The step operators in a fresh process: their first call inside a capture, and first calls of several threads at once."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]
PRELUDE = """
import sys, threading
import torch
from wf_bitnet import ops
D = 128

def state(seed, int8):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kv = ops.PagedKV(30, 1, 2, 16, D, dtype=torch.int8 if int8 else torch.bfloat16)
    if int8:
        kv.pool.copy_(torch.randint(1, 256, kv.pool.shape, generator=g, device="cuda", dtype=torch.uint8))
        kv.scales.fill_(0.02)
    else:
        kv.pool.copy_(torch.randn(kv.pool.shape, generator=g, device="cuda"))
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    q = torch.randn(3, 8, D, generator=g, device="cuda").to(torch.bfloat16)
    return dict(q=q, kv=kv, pt=torch.arange(20, dtype=torch.int32, device="cuda"), table=torch.arange(20, 29, dtype=torch.int32, device="cuda").view(3, 3), lens=i([5, 40, 17]),
                new=i([1, 2, 3]), free=torch.arange(9, dtype=torch.int32, device="cuda"), count=i([9]), done=torch.tensor([True, False, True], device="cuda"),
                x=torch.randn(4, 5001, generator=g, device="cuda"), tok=i([1, 2, 3, 4]))

def calls(s):
    p = ops.paged_plan(s["lens"], s["new"], s["table"].clone(), s["free"], s["count"], 16, 8)
    r = ops.paged_release(s["done"], s["lens"], s["table"], s["free"].repeat(3), s["count"], 16)
    return [*p, *r, ops.paged_prefix_attn(s["q"], s["kv"], 0, s["pt"], 300, s["table"], s["lens"]), *ops.token_logprobs(s["x"], s["tok"], 7)]
"""


def fresh(code):
    env = dict(os.environ, PYTHONPATH=str(ROOT / "wrinklefree-inference-engine_b200"))
    r = subprocess.run([sys.executable, "-c", PRELUDE + code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    assert "fine" in r.stdout


@pytest.mark.parametrize("int8", [False, True])
def test_first_calls_inside_a_capture(int8):
    fresh(f"""
s = state(1, {int8})
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = calls(s)
for _ in range(2):
    graph.replay()
torch.cuda.synchronize()
want = calls(s)
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("fine")
""")


def test_first_calls_of_several_threads():
    fresh("""
states = [state(k, k % 2 == 1) for k in range(6)]
torch.cuda.synchronize()
start, out, bad = threading.Barrier(6), [None] * 6, []

def work(k):
    try:
        stream = torch.cuda.Stream()
        start.wait()
        with torch.cuda.stream(stream):
            for _ in range(20):
                out[k] = calls(states[k])
        stream.synchronize()
    except Exception as e:
        bad.append(e)

threads = [threading.Thread(target=work, args=(k,)) for k in range(6)]
[t.start() for t in threads]
[t.join() for t in threads]
assert not bad, bad
torch.cuda.synchronize()
for k in range(6):
    assert all(torch.equal(a, b) for a, b in zip(out[k], calls(states[k]))), k
print("fine")
""")
