"""The first call of a process inside a graph capture, and calls from two threads at once: nothing that
the operators prepare once (limits, cluster counts) needs a call outside."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CAPTURED = """
import torch
from qextract_infer_b200 import _C
g = torch.Generator(device="cuda").manual_seed(1)
r = lambda *s: torch.randn(*s, generator=g, device="cuda").half()
x, y, A, B = r(3, 64), r(3, 64), r(2, 64, 16), r(2, 16, 64)
ids, scales = torch.tensor([1, -1, 0], device="cuda"), torch.ones(2, device="cuda")
xt, yt, W, u = r(3, 40, 64), r(3, 40, 64), r(64, 1000), torch.rand(3, generator=g, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    a = _C.multi_lora_add(y, x, A, B, ids, scales)
    b = _C.multi_lora_add(yt, xt, A, B, ids, scales)
    logits = _C.lm_head_logits(a, W)
    tok, lp = _C.sample_logits(logits, u, 0.8, 40, 0.9)
graph.replay()
torch.cuda.synchronize()
a2, b2 = _C.multi_lora_add(y, x, A, B, ids, scales), _C.multi_lora_add(yt, xt, A, B, ids, scales)
l2 = _C.lm_head_logits(a2, W)
t2, p2 = _C.sample_logits(l2, u, 0.8, 40, 0.9)
for v, w in ((a, a2), (b, b2), (logits, l2), (tok, t2), (lp, p2)):
    assert torch.equal(v, w)
_C.check_device_error()
print("ok")
"""

THREADS = """
import threading
import torch
from qextract_infer_b200 import _C
g = torch.Generator(device="cuda").manual_seed(1)
r = lambda *s: torch.randn(*s, generator=g, device="cuda").half()
x, y, A, B = r(3, 40, 64), r(3, 40, 64), r(2, 64, 16), r(2, 16, 64)
ids, scales = torch.tensor([1, -1, 0], device="cuda"), torch.ones(2, device="cuda")
W, u = r(64, 1000), torch.rand(3, generator=g, device="cuda")
torch.cuda.synchronize()
got, errors = {}, []

def work(i):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                a = _C.multi_lora_add(y, x, A, B, ids, scales)
                got[i] = (a, *_C.sample_logits(_C.lm_head_logits(a[:, 0].contiguous(), W), u, 0.8, 0, 0.9))
            torch.cuda.current_stream().synchronize()
    except Exception as e:
        errors.append(e)

ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
[t.start() for t in ts]
[t.join() for t in ts]
assert not errors, errors
for i in range(1, 4):
    assert all(torch.equal(v, w) for v, w in zip(got[0], got[i]))
print("ok")
"""


@pytest.mark.parametrize("script", [CAPTURED, THREADS], ids=["captured", "threads"])
def test_first_calls(script):
    r = subprocess.run([sys.executable, "-c", script], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.endswith("ok\n"), r.stdout[-1000:] + r.stderr[-2000:]
