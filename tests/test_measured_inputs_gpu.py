"""The sampling cases of perf/more_operators.py: their inputs are the seed's alone (some of a row's 20
tokens that stand out coincide, in small vocabularies usually), so that the kernel, the plain form and the
64-bit one, each of them with inputs of its own making and in another process, answer the same question."""

import json
import random
import subprocess
import sys

import pytest
import torch

from perf import more_operators as mo

pytestmark = pytest.mark.gpu

SIZES = [(1, 100), (64, 100), (7, 137), (33, 200), (16, 411), (64, 700), (5, 1500)]


def _case(b, v, mixed):
    return mo._sample(f"{b}x{v}", b=b, v=v, temperature=0.9, top_k=0, top_p=0.95, min_p=0.01, mixed=mixed)


@pytest.mark.parametrize("b,v", SIZES)
def test_two_preparations_are_the_same(b, v):
    """and where tokens that stand out coincide, the largest of their logits counts"""
    for seed in (1, 2):
        case = _case(b, v, True)
        first, second = mo.prepare(case, seed), mo.prepare(case, seed)
        for name, t in first.items():
            if name != "case":
                assert torch.equal(t, second[name]), name
        g = torch.Generator(device="cuda").manual_seed(seed)
        heap = 2.5 * torch.randn(b, v, generator=g, device="cuda")
        at = torch.randint(0, v, (b, 20), generator=g, device="cuda").tolist()
        peaks = 9 + 3 * torch.randn(b, 20, generator=g, device="cuda")
        want, values = heap.tolist(), peaks.tolist()
        for i in range(b):
            for j in set(at[i]):
                want[i][j] = max(x for k, x in zip(at[i], values[i]) if k == j)
        assert torch.equal(first["logits"].cpu(), torch.tensor(want).half())


CHILD = """
import json, sys
from perf import more_operators as mo
mo.own = sys.argv[1] == "own"
out = []
for case, seed in json.loads(sys.stdin.read()):
    tokens, logprobs = mo.exact(case, seed) if sys.argv[1] == "exact" else mo.run(mo.prepare(case, seed))
    out.append([tokens.tolist(), logprobs.double().tolist()])
print(json.dumps(out))
"""


def test_kernel_plain_form_and_64_bits_in_processes_of_their_own():
    rng = random.Random(6)
    jobs = [(_case(b, v, mixed), 3) for b, v in SIZES for mixed in (False, True)]
    while len(jobs) < 40:
        case = mo.draw(rng)
        if case["kind"] == "sample" and case["v"] <= 700:
            jobs.append((case, len(jobs)))
    sides = []
    for side in ("plain", "own", "exact"):
        r = subprocess.run([sys.executable, "-c", CHILD, side], input=json.dumps(jobs), capture_output=True, text=True, timeout=600)
        assert r.returncode == 0, r.stderr[-2000:]
        sides.append(json.loads(r.stdout.splitlines()[-1]))
    for (case, _), plain, own, exact in zip(jobs, *sides):
        assert plain[0] == own[0] == exact[0], case
        want = torch.tensor(exact[1], dtype=torch.float64)
        # one rounding to 32 bits, and sums of weights that are a few 2^-53 (plain) or v 2^-44 (kernel) off
        for side in (plain, own):
            off = (torch.tensor(side[1], dtype=torch.float64) - want).abs()
            assert (off <= want.abs() * 2.0 ** -24 + 1e-9).all(), case
