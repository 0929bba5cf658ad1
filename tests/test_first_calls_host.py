"""First calls of attention from several threads, against a stand-in for the CUDA runtime that is slow to set a kernel's attributes and refuses launches without them: no
GPU is needed, and the order that a fast runtime rarely shows comes up every time."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CUDA = Path("/usr/local/cuda/include")
CODE = """
import ctypes as C, sys, threading
from wf_bitnet import _lib
L = _lib.lib()
buf = (C.c_uint8 * 4096)()
P = (C.addressof(buf) + 255) // 256 * 256
FORM, THREADS, CALLS = sys.argv[1], int(sys.argv[2]), int(sys.argv[3])
layout = _lib.KvLayout(P, 64, 1, 2, 16, 128, _lib.WF_I8 if "int8" in FORM else _lib.WF_BF16)

def call():
    if "decode" in FORM:
        return L.wf_paged_decode_attn(P, C.byref(layout), 0, P, 3, P, 3, 8, 0.1, P, _lib.WF_BF16, P, 1 << 30, None)
    return L.wf_paged_prefix_attn(P, C.byref(layout), 0, P, 0 if "own" in FORM else 300, P, 3, P, 3, 8, 0.1, P, _lib.WF_BF16, P, 1 << 30, None)

start, seen = threading.Barrier(THREADS), []

def work():
    start.wait()
    for _ in range(CALLS):
        rc = call()
        seen.append((rc, L.wf_last_error() if rc else b""))

threads = [threading.Thread(target=work) for _ in range(THREADS)]
[t.start() for t in threads]
[t.join() for t in threads]
print(len([1 for rc, _ in seen if rc == 0]), [e for rc, e in seen if rc])
"""


@pytest.fixture(scope="module")
def runtime(tmp_path_factory):
    if not CUDA.exists():
        pytest.skip("no CUDA headers")
    so = tmp_path_factory.mktemp("fake") / "libfakecudart.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-o", str(so), str(ROOT / "tests" / "fake_cudart.cpp"), f"-I{CUDA}"], check=True)
    return so


def run(runtime, form, threads, calls, fail=0):
    env = dict(os.environ, PYTHONPATH=str(ROOT / "wrinklefree-inference-engine_b200"), LD_PRELOAD=str(runtime), FAIL_ATTRIBUTES=str(fail))
    r = subprocess.run([sys.executable, "-c", CODE, form, str(threads), str(calls)], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    good, bad = r.stdout.split(" ", 1)
    return int(good), bad.strip()


FORMS = ["bf16 prefix", "int8 prefix", "bf16 own", "int8 own", "bf16 decode", "int8 decode"]


@pytest.mark.parametrize("form", FORMS)
def test_no_launch_comes_before_its_attributes(runtime, form):
    assert run(runtime, form, 6, 2) == (12, "[]")


@pytest.mark.parametrize("form", FORMS)
def test_attributes_that_failed_are_set_by_the_next_call(runtime, form):
    good, bad = run(runtime, form, 1, 3, fail=1)
    assert good == 2 and "CUDA error 2" in bad
