"""A missing or unloadable Python binding costs the five operators that need it, not the package."""

import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCRIPT = """
import sys

class NoBinding:
    def find_spec(self, name, path=None, target=None):
        if name == "qextract_infer_b200._binding":
            raise ImportError("undefined symbol: of another torch")

sys.meta_path.insert(0, NoBinding())
import torch
import qextract_infer_b200 as q
from qextract_infer_b200 import _C
assert q._C_AVAILABLE and q.check_backend()
x = torch.zeros(1, 128, dtype=torch.float16)
for call in (lambda: q.fused_rmsnorm(x, x[0]), lambda: q.fused_swiglu(x, x)):
    try:
        call()
    except RuntimeError as e:
        assert "CUDA tensor" in str(e), e
    else:
        raise AssertionError("no refusal of a CPU tensor")
n = 0
for call in (lambda: q.qk_norm_rope(x, 1, 1, x, x, 1e-6, x, x), lambda: q.ring_append_q4(x, x, x, x, 0, 4, 60),
             lambda: q.ring_gather_q4(x, x, 0, 4, 60), lambda: q.decode_attention_q4(x, x, x, 0, 4, 60),
             lambda: q.prefill_attention_q4(x, x, x, x, x, 0, 4, 60)):
    try:
        call()
    except ImportError as e:
        assert "of another torch" in str(e) and "qextract_infer_b200.build" in str(e), e
        n += 1
assert n == 5, n
print("ok")
"""


def test_without_the_binding():
    r = subprocess.run([sys.executable, "-c", SCRIPT], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.endswith("ok\n"), r.stdout + r.stderr
