"""Attention as the very first call of several threads at once, in fresh processes: what a kernel needs once per device is made before any of them launches it."""
import pytest

from test_gpu_step_ops_first import fresh

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("again", range(2))
@pytest.mark.parametrize("form", ["int8 prefix", "bf16 prefix", "bf16 own"])
def test_attention_first(form, again):
    fresh(f"""
from wf_bitnet import _native
_native.ops()
torch.zeros(1, device="cuda").add_(1)
N = 12
states = [state(k, {form.startswith("int8")}) for k in range(N)]
streams = [torch.cuda.Stream() for _ in range(N)]

def call(s):
    return ops.paged_prefix_attn(s["q"], s["kv"], 0, s["pt"], {0 if form.endswith("own") else 300}, s["table"], s["lens"])

torch.cuda.synchronize()
start, out, bad = threading.Barrier(N), [None] * N, []

def work(k):
    try:
        with torch.cuda.stream(streams[k]):
            start.wait()
            out[k] = call(states[k])
        streams[k].synchronize()
    except Exception as e:
        bad.append(e)

threads = [threading.Thread(target=work, args=(k,)) for k in range(N)]
[t.start() for t in threads]
[t.join() for t in threads]
assert not bad, bad
for k in range(N):
    assert torch.equal(out[k], call(states[k])), k
print("fine")
""")
